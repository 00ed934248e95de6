"""How the attention over the 8-bit paged cache is spread over a device
(hbfsim_b200/csrc/kv_plan.h), for devices of any number of SMs (a slice of a
GPU has fewer).  No GPU needed: the header is compiled for the host."""
import ctypes
import itertools
import shutil
import subprocess
from pathlib import Path

import pytest

CSRC = Path(__file__).resolve().parent.parent / "hbfsim_b200" / "csrc"
CALL = ["seqs", "tokens", "heads", "group", "dim", "block", "width", "top", "lists", "weights"]
PLAN = ["nt", "lists", "rows", "row_tiles", "units", "per_unit", "workers", "tiles", "whole", "warps",
        "team", "segments", "bytes", "each", "whole_tiles"]
SOURCE = """
#include "kv_plan.h"
extern "C" void plan(const unsigned* c, unsigned sms, unsigned long long* out)
{
    using namespace hbfb;
    const Plan p = plan_of(PlanCall{c[0], c[1], c[2], c[3], c[4], c[5], c[6], c[7], c[8] != 0, c[9] != 0}, sms);
    const unsigned long long x[] = {p.nt, p.lists, p.rows, p.row_tiles, p.units, p.per_unit, p.workers, p.tiles,
                                    p.whole, p.warps, p.team, p.segments, p.bytes,
                                    part_of(p.tiles, p.team, c[5] / 16), whole_tiles(p.nt, p.warps)};
    for (auto v : x) *out++ = v;
}
"""


@pytest.fixture(scope="module")
def plan(tmp_path_factory):
    compiler = shutil.which("g++") or pytest.skip("no host compiler")
    at = tmp_path_factory.mktemp("plan")
    (at / "plan.cpp").write_text(SOURCE)
    subprocess.run([compiler, "-std=c++17", "-O1", "-shared", "-fPIC", "-I", str(CSRC), "-o", str(at / "plan.so"),
                    str(at / "plan.cpp")], check=True)
    lib = ctypes.CDLL(str(at / "plan.so"))

    def call(sms, **sizes):
        given = (ctypes.c_uint * len(CALL))(*(int(sizes[k]) for k in CALL))
        out = (ctypes.c_ulonglong * len(PLAN))()
        lib.plan(given, ctypes.c_uint(sms), out)
        return dict(zip(PLAN, out))
    return call


def calls():
    for seqs, heads, group, tokens, dim, block in itertools.product(
            (1, 2, 7, 8, 16, 17, 32, 64, 65, 200), (1, 4, 8), (1, 8, 24), (1, 3, 16), (64, 256), (16, 64)):
        for tiles, lists, weights in itertools.product((0, 4, 32, 64, 68, 128, 132, 1024, 5000), (False, True),
                                                       (False, True)):
            blocks = -(-tiles * 16 // block)
            yield dict(seqs=seqs, heads=heads, group=group, tokens=tokens, dim=dim, block=block,
                       width=3 if lists else blocks, top=max(1, blocks) if lists else 0, lists=lists, weights=weights)


@pytest.mark.parametrize("sms", [1, 2, 7, 14, 16, 28, 32, 48, 63, 64, 74, 100, 132, 148, 160])
def test_forms_hold_on_any_device(plan, sms):
    for call in calls():
        p = plan(sms, **call)
        assert p["segments"] == call["seqs"] * p["lists"] * call["heads"] * p["row_tiles"]
        assert p["row_tiles"] * 8 * p["nt"] >= p["rows"] and p["workers"] >= 1
        assert p["team"] in (1, 2, 4, 8) and p["warps"] in (4, 8)
        if not p["whole"]:
            assert p["bytes"] > 0 or p["segments"] == 0
            continue
        assert p["bytes"] == 0
        # CTAs of 4 warps take a segment each: a team of them would index past the segments
        taken_by_one = p["team"] if p["warps"] > 4 else 1
        assert p["workers"] == p["segments"] * taken_by_one, call
        assert p["team"] == 1 or p["workers"] <= sms, "teams wait for one another's places"
        assert p["each"] * p["team"] >= p["tiles"] and p["each"] <= p["whole_tiles"], "room for the tiles' sums"
        assert not call["weights"] or p["lists"] * p["row_tiles"] == 1


def test_forms_of_a_whole_device(plan):
    """The forms that the comments' measurements were taken with, at 148 SMs."""
    shape = dict(tokens=1, heads=8, group=4, dim=128, block=16, top=0, lists=False, weights=True)
    for seqs, width, want in ((8, 38, (1, 8, 1)), (1, 128, (1, 8, 8)), (4, 256, (1, 8, 4)), (1, 1024, (1, 8, 8)),
                              (8, 128, (1, 8, 2)), (50, 38, (1, 4, 1)), (200, 128, (1, 4, 1)), (64, 2048, (0, 4, 1)),
                              (1, 16384, (0, 8, 8))):
        p = plan(148, seqs=seqs, width=width, **shape)
        assert (p["whole"], p["warps"], p["team"]) == want, (seqs, width)
