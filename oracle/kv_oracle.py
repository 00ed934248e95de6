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


def rotate(x, positions, freq, axis, neighbours):
    """x: float32 [tokens, heads, D], positions: [axes, tokens].  Angles, sines and cosines in 64
    bits; sines, cosines, products and sums rounded to 32."""
    x = np.asarray(x, np.float32)
    out = x.copy()
    pairs = len(freq)
    for i in range(pairs):
        a = positions[min(int(axis[i]), len(positions) - 1)].astype(np.float64) * freq[i]
        c, s = (f(a).astype(np.float32)[:, None] for f in (np.cos, np.sin))
        m, n = (2 * i, 2 * i + 1) if neighbours else (i, i + pairs)
        out[:, :, m] = x[:, :, m] * c - x[:, :, n] * s
        out[:, :, n] = x[:, :, m] * s + x[:, :, n] * c
    return out


def _p40(p):
    """A probability in whole multiples of 2^-40, halves to even."""
    p = float(p)
    return 0 if p != p else round(min(max(p, 0.0), 1.0) * 2.0 ** 40)


def verify(target, draft, tokens, accept, sample, counts, lengths):
    """Python's whole numbers and fractions throughout.  Returns accepted, tokens, lengths."""
    from fractions import Fraction
    seqs, rows, vocab = target.shape
    n = rows - 1
    accepted, out, kept = [], np.full((seqs, rows), -1, np.int32), []
    for b in range(seqs):
        d = min(max(int(counts[b]), 0), n)
        a = 0
        while a < d:
            t = int(tokens[b, a])
            if not 0 <= t < vocab:
                break
            p, u = float(target[b, a, t]), float(accept[b, a])
            q = 1.0 if draft is None else float(draft[b, a, t])
            if all(np.isfinite([p, u, q])):
                good = Fraction(u) * Fraction(q) < Fraction(p)
            else:  # as 64-bit numbers compare: a NaN accepts nothing
                good = u * q < p
            if not good:
                break
            a += 1
        whole = [_p40(p) for p in target[b, a]]
        left = list(whole)
        if a < d:
            if draft is not None:
                left = [max(p - _p40(q), 0) for p, q in zip(whole, draft[b, a])]
            elif 0 <= int(tokens[b, a]) < vocab:
                left[int(tokens[b, a])] = 0
        if sum(left) == 0:
            left = whole
        out[b, :a] = tokens[b, :a]
        if sum(left):
            s = float(sample[b])
            u = 0 if s != s else min(max(int(min(max(s, -1.0), 2.0) * 2 ** 24), 0), 2 ** 24 - 1)
            border = u * sum(left) >> 24
            total = 0
            for i, w in enumerate(left):
                total += w
                if total > border:
                    out[b, a] = i
                    break
        accepted.append(a)
        kept.append(int(lengths[b]) - (d - a))
    return np.array(accepted, np.int32), out, np.array(kept, np.int32)


def resize(refs, table, lengths, want, block, freed=None, freed_counts=None):
    """One claim after the other.  Returns refs, table, limits, src, dst."""
    refs, table = refs.astype(np.int64).copy(), table.copy()
    pages, (seqs, width) = len(refs), table.shape
    real = lambda p: 0 <= p < pages  # noqa: E731
    held = [min(max(int(x), 0), width * block) for x in lengths]
    goal = [min(max(int(x), 0), width * block) for x in want]
    need = [-(-g // block) for g in goal]
    for b in range(seqs):
        for j in range(need[b], width):
            if real(table[b, j]):
                refs[table[b, j]] -= 1
            table[b, j] = -1
    if freed is not None:
        for row, count in zip(freed, freed_counts):
            for p in row[:max(0, int(count))]:
                if real(p):
                    refs[p] -= 1
    start = refs.copy()
    asked = [(b, j) for b in range(seqs) if goal[b] > held[b] for j in range(held[b] // block, need[b])]
    by_page = {}
    for b, j in asked:
        p = int(table[b, j])
        if real(p) and start[p] > 1:
            by_page.setdefault(p, []).append(b)
    free = [p for p in range(pages) if start[p] < 1]
    limits, src, dst = list(goal), np.full(seqs, -1, np.int32), np.full(seqs, -1, np.int32)
    claims = 0
    for b, j in asked:
        p = int(table[b, j])
        shared = real(p) and start[p] > 1
        if real(p) and not shared:
            continue
        if shared and len(by_page[p]) >= start[p] and max(by_page[p]) == b:
            served = claims <= len(free)
        else:
            served = claims < len(free)
            if served:
                new = free[claims]
                refs[new] = 1
                table[b, j] = new
                if shared:
                    refs[p] -= 1
                    if j == held[b] // block and held[b] % block:
                        src[b], dst[b] = p, new
            claims += 1
        if not served:
            limits[b] = min(limits[b], max(held[b], j * block))
    return refs.astype(np.int32), table, np.array(limits, np.int32), src, dst


def fork(refs, table, lengths, parents, block):
    """Returns refs, table, lengths."""
    refs = refs.astype(np.int64).copy()
    pages, (seqs, width) = len(refs), table.shape
    new = np.full((len(parents), width), -1, np.int32)
    kept = np.zeros(len(parents), np.int32)
    for r, s in enumerate(parents):
        if 0 <= s < seqs:
            kept[r] = min(max(int(lengths[s]), 0), width * block)
            many = -(-int(kept[r]) // block)
            new[r, :many] = table[s, :many]
    for t, by in ((new, 1), (table, -1)):
        for p in t.ravel():
            if 0 <= p < pages:
                refs[p] += by
    return refs.astype(np.int32), new, kept


def compact(refs, table):
    """Returns refs, table, src, dst, live, where."""
    pages = len(refs)
    used = [p for p in range(pages) if refs[p] > 0]
    n = len(used)
    holes = [p for p in range(n) if refs[p] <= 0]
    movers = [p for p in reversed(used) if p >= n]
    src, dst = (np.full(pages // 2, -1, np.int32) for _ in range(2))
    src[:len(movers)], dst[:len(holes)] = movers, holes
    where = np.full(pages, -1, np.int32)
    where[used] = used
    where[movers] = holes
    new_refs = np.zeros(pages, np.int32)
    for p in used:
        new_refs[where[p]] = refs[p]
    new_table = np.array([[where[p] if 0 <= p < pages else p for p in row] for row in table], np.int32)
    return new_refs, new_table.reshape(table.shape), src, dst, np.array([n], np.int32), where
