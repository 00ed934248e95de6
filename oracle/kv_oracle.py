"""The operators of include/hbfsim/kv_v1.h in 64 bits, one value at a time
where that is clearest (numpy; not the product path).  Caches
are dicts of numpy arrays: data (uint8 e4m3 codes [P, H, 2, T, D]), scale
(float64 [P, H, 2]), bounds (int8 [P, H, 2, D])."""
from __future__ import annotations

import numpy as np


def _decode_table() -> np.ndarray:
    """Value of every e4m3 code: 1 sign, 4 exponent (bias 7), 3 fraction bits; 0x7f is NaN."""
    out = np.zeros(256)
    for c in range(256):
        e, m = (c >> 3) & 15, c & 7
        v = (m / 8) * 2.0 ** -6 if e == 0 else (1 + m / 8) * 2.0 ** (e - 7)
        if e == 15 and m == 7:
            v = np.nan
        out[c] = -v if c & 128 else v
    return out


E4M3 = _decode_table()
_MAGNITUDES = E4M3[:127]            # 0 .. 448, ascending


def encode(x: np.ndarray) -> np.ndarray:
    """Nearest e4m3 code, ties to the even code, magnitudes above 448 to 448, NaN to NaN."""
    x = np.asarray(x, np.float64)
    size = np.minimum(np.abs(np.where(np.isnan(x), 0, x)), 448.0)
    up = np.clip(np.searchsorted(_MAGNITUDES, size), 1, 126)
    low, high = _MAGNITUDES[up - 1], _MAGNITUDES[up]
    mid = (low + high) / 2          # exact: neighbours differ in the last bit
    code = np.where((size > mid) | ((size == mid) & (up % 2 == 0)), up, up - 1)
    code = np.where(np.signbit(x), code | 128, code)
    return np.where(np.isnan(x), 127, code).astype(np.uint8)


def scale_exponent(a: float) -> int:
    """Least e with a <= 448 * 2^e, between -100 and 120."""
    e = -100
    while e < 120 and a > 448.0 * 2.0 ** e:
        e += 1
    return e


def _page(table, pages, b, j):
    if j >= table.shape[1]:
        return -1
    p = int(table[b, j])
    return p if 0 <= p < pages else -1


def append(cache, k, v, table, start, offsets):
    """In place.  k, v: float64 [tokens, H, D]."""
    data, scale, bounds = cache["data"], cache["scale"], cache["bounds"]
    pages, heads, _, T, _ = data.shape
    for b in range(len(start)):
        n = int(offsets[b + 1] - offsets[b])
        at = int(start[b])
        done = 0
        while done < n:
            j, slot = divmod(at + done, T)
            many = min(T - slot, n - done)
            page = _page(table, pages, b, j)
            if page >= 0:
                for h in range(heads):
                    for side, source in enumerate((k, v)):
                        x = source[offsets[b] + done:offsets[b] + done + many, h]
                        size = np.abs(x[np.isfinite(x)])
                        s = 2.0 ** scale_exponent(size.max() if size.size else 0.0)
                        if slot:
                            s = max(s, scale[page, h, side])
                        old = E4M3[data[page, h, side, :slot]] * (scale[page, h, side] / s)
                        data[page, h, side, :slot] = encode(old)
                        data[page, h, side, slot:slot + many] = encode(x / s)
                        data[page, h, side, slot + many:] = 0
                        scale[page, h, side] = s
                    key = np.nan_to_num(E4M3[data[page, h, 0, :slot + many]])
                    bounds[page, h, 0] = np.floor(key.min(0) / 4)
                    bounds[page, h, 1] = np.ceil(key.max(0) / 4)
            done += many


def attention(cache, q, table, lengths, softmax_scale, lists=None):
    """q: float64 [B, n, Hq, D]; lists: None or per (b, t, h) a sequence of
    block indices.  Returns out, lse, weights, and for error bounds: mass
    (softmax of |values|), reach (largest sum of |products| of a row, scaled),
    vmax (largest magnitude of a value that the row sees)."""
    data, scale = cache["data"], cache["scale"]
    pages, heads, _, T, D = data.shape
    B, n, Hq, _ = q.shape
    G, width = Hq // heads, table.shape[1]
    out, mass = np.zeros(q.shape), np.zeros(q.shape)
    lse = np.full(q.shape[:3], -np.inf)
    reach, vmax = np.zeros(q.shape[:3]), np.zeros(q.shape[:3])
    weights = np.zeros((B, heads, width))
    for b in range(B):
        length = min(max(int(lengths[b]), 0), width * T)
        have = -(-length // T)
        for t in range(n):
            last = length - n + t
            for h in range(heads):
                js = range(have) if lists is None else [j for j in lists[b][t][h] if 0 <= j < have]
                js = [j for j in js if _page(table, pages, b, j) >= 0 and j * T <= last]
                if not js:
                    continue
                page = [_page(table, pages, b, j) for j in js]
                see = (np.array(js)[:, None] * T + np.arange(T) <= last).ravel()
                block = np.repeat(js, T)[see]
                key = (E4M3[data[page, h, 0]] * scale[page, h, 0][:, None, None]).reshape(-1, D)[see]
                val = (E4M3[data[page, h, 1]] * scale[page, h, 1][:, None, None]).reshape(-1, D)[see]
                for r in range(h * G, (h + 1) * G):
                    s = key @ q[b, t, r] * softmax_scale
                    p = np.exp(s - s.max())
                    lse[b, t, r] = s.max() + np.log(p.sum())
                    p /= p.sum()
                    out[b, t, r] = p @ val
                    mass[b, t, r] = p @ np.abs(val)
                    reach[b, t, r] = (np.abs(key) @ np.abs(q[b, t, r])).max() * abs(softmax_scale)
                    vmax[b, t, r] = np.abs(val).max()
                    np.add.at(weights[b, h], block, p)
    return out, lse, weights, mass, reach, vmax


def select(cache, q, table, lengths, top, sink, recent):
    """Per (b, t, h) the ascending list of blocks, by exact arithmetic (Python
    ints; the product with the scale rounds to 32 bits as the definition says)."""
    bounds, scale = cache["bounds"].astype(np.int64), cache["scale"]
    pages, heads, _, D = bounds.shape
    T = cache["data"].shape[3]
    B, n, Hq, _ = q.shape
    G, width = Hq // heads, table.shape[1]
    lists = []
    for b in range(B):
        length = min(max(int(lengths[b]), 0), width * T)
        lists.append([])
        for t in range(n):
            have = max(0, (length - n + t) // T + 1)
            lists[-1].append([])
            for h in range(heads):
                x = q[b, t, h * G:(h + 1) * G]
                x = np.where(np.isfinite(x), x, 0)
                most = np.abs(x).max()
                e = max(int(np.frexp(most)[1]), -100) if most > 0 else 0
                qi = np.clip(np.rint(x * 2.0 ** (7 - e)), -127, 127).astype(np.int64)
                up, down = np.maximum(qi, 0).sum(0), np.minimum(qi, 0).sum(0)
                rank = []
                for j in range(have):
                    page = _page(table, pages, b, j)
                    if page < 0:
                        continue
                    whole = int(up @ bounds[page, h, 1] + down @ bounds[page, h, 0])
                    s = np.float32(np.float32(whole) * np.float32(scale[page, h, 0]))
                    always = j < sink or j + recent >= have
                    rank.append((0 if always else 1, 0.0 if always else -float(s), j))
                lists[-1][-1].append(sorted(j for _, _, j in sorted(rank)[:top]))
    return lists


def evict(score, weights, table, lengths, keep, block, sink, recent, decay):
    """Returns score, table, lengths, freed, freed counts."""
    B, width = table.shape
    out_s, out_t = np.zeros((B, width), np.int64), np.full((B, width), -1, np.int32)
    freed, counts = np.full((B, width), -1, np.int32), np.zeros(B, np.int32)
    out_l = np.zeros(B, np.int32)
    w = np.where(np.isnan(weights), 0, np.clip(np.asarray(weights, np.float64), 0, 2.0 ** 20))
    fixed = np.rint(w * 2.0 ** 30).astype(np.int64).sum(1)
    for b in range(B):
        length = min(max(int(lengths[b]), 0), width * block)
        have = -(-length // block)
        s = [int(score[b, j]) for j in range(have)]
        s = [x - (x >> decay) if decay else x for x in s]
        s = [x + int(fixed[b, j]) for j, x in enumerate(s)]
        leave = max(0, have - keep)
        may = range(sink, have - recent)
        gone = set(sorted(may, key=lambda j: (s[j], j))[:leave])
        stay = [j for j in range(have) if j not in gone]
        out_s[b, :len(stay)] = [s[j] for j in stay]
        out_t[b, :len(stay)] = table[b, stay]
        freed[b, :leave] = table[b, sorted(gone)]
        counts[b], out_l[b] = leave, length - leave * block
    return out_s, out_t, out_l, freed, counts
