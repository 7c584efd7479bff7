"""How a call of paged attention is cut (plan_call in
undertow_amd/csrc/ut_paged_plan.h), on the CPU, for both cache
formats: what it launches covers the call, and it reserves no more than the
parts that can be made."""
import ctypes as C
import random
import subprocess
from pathlib import Path

import pytest

CSRC = Path(__file__).resolve().parents[1] / "undertow_amd" / "csrc"
CUS = 256

SRC = r"""
#include "ut_paged_plan.h"
extern "C" {
void costs(int bf16, ut::PlanCosts *c) { *c = bf16 ? ut::kCostsBf16 : ut::kCostsF16x2; }
void cut(const ut::PlanCosts *c, int cus, int units, int groups, int64_t each, int64_t listed, int lists,
         ut::PlanCall *out) {
    *out = ut::plan_call(*c, cus, units, groups, each, listed, lists);
}
int64_t ranges(int64_t W, int64_t most, float spread) { return ut::plan_ranges(W, (int32_t)most, spread); }
int64_t begin(int64_t W, int64_t N, int64_t r) { return ut::plan_begin(W, N, r); }
int64_t range_of(int64_t W, int64_t N, int64_t t) { return ut::plan_range_of(W, N, t); }
int64_t slot(int64_t r, int64_t begins) { return ut::plan_slot(r, begins != 0); }
}
"""


class Costs(C.Structure):
    _fields_ = [("waves", C.c_int32), ("lead", C.c_int32), ("ratio", C.c_int32), ("bytes_ratio", C.c_int32),
                ("join", C.c_float), ("brief", C.c_int32)]


class Call(C.Structure):
    _fields_ = [("whole", C.c_int32), ("most", C.c_int32), ("per", C.c_int32), ("chunks", C.c_int32),
                ("wide", C.c_int32), ("spread", C.c_float), ("slots", C.c_int64)]



@pytest.fixture(scope="module")
def cut(tmp_path_factory):
    d = tmp_path_factory.mktemp("cut")
    (d / "c.cpp").write_text(SRC)
    subprocess.run(["g++", "-std=c++17", "-O1", "-shared", "-fPIC", "-I", str(CSRC), "-o", str(d / "c.so"),
                    str(d / "c.cpp")], check=True)
    lib = C.CDLL(str(d / "c.so"))
    f, costs = lib.cut, {}
    f.restype, f.argtypes = None, [C.POINTER(Costs), C.c_int, C.c_int, C.c_int, C.c_int64, C.c_int64, C.c_int,
                                   C.POINTER(Call)]
    lib.costs.restype, lib.costs.argtypes = None, [C.c_int, C.POINTER(Costs)]
    for fmt in ("bf16", "f16x2"):
        costs[fmt] = Costs()
        lib.costs(fmt == "bf16", C.byref(costs[fmt]))

    def call(fmt, sequences, rows, heads, positions, lists=False):
        out, each = Call(), -(-positions // 32)
        f(costs[fmt], CUS, sequences, rows * -(-heads // 16), each, each, lists, out)
        return out
    call.costs = costs
    call.waves = {k: c.waves for k, c in costs.items()}
    for name in ("ranges", "begin", "range_of", "slot"):
        g = getattr(lib, name)
        g.restype, g.argtypes = C.c_int64, [C.c_int64, C.c_int64] + [C.c_int64] * (name in ("begin", "range_of"))
        setattr(call, name, g)
    lib.ranges.argtypes = [C.c_int64, C.c_int64, C.c_float]
    return call


@pytest.mark.parametrize("fmt", ["bf16", "f16x2"])
@pytest.mark.parametrize("seed", range(20))
def test_a_call_is_covered_and_reserves_what_its_parts_take(cut, fmt, seed):
    rng = random.Random(seed)
    log = lambda lo, hi: round(lo * (hi / lo) ** rng.random())
    for _ in range(200):
        B = log(1, 65535)
        M = log(1, max(1, 65535 // B))
        H = rng.choice([1, 16, 20, 64, 128, 160, 1000])
        p = cut(fmt, B, M, H, log(1, 2**31 - 1024))
        groups, waves = M * -(-H // 16), cut.waves[fmt]
        assert 1 <= p.per <= waves and p.per * p.chunks >= groups and p.per * (p.chunks - 1) < groups
        if p.whole:
            assert p.most == B and p.slots == 0
        elif p.most == 1:
            assert p.slots == 0
        else:  # ranges that run at once, two places each
            assert p.most * p.chunks <= CUS and p.slots == 2 * p.most * groups <= 2 * CUS * waves


@pytest.mark.parametrize("fmt", ["bf16", "f16x2"])
@pytest.mark.parametrize("B,M", [(1, 512), (1, 2048), (1, 8192), (1, 65535), (3, 777), (4, 256), (2, 20000)])
@pytest.mark.parametrize("positions", [100, 2000, 32768, 1 << 20])
def test_prompt_rows_leave_no_parts(cut, fmt, B, M, positions):
    p = cut(fmt, B, M, 128, max(M, positions))
    assert p.slots == 0 and (p.whole or p.most == 1)


def test_one_range_counts_its_rounds_over_the_cus(cut):
    """777 workgroups take four rounds over all sequences, 3 x 777 ten over one."""
    assert cut("bf16", 3, 777, 128, 1900).whole
    p = cut("bf16", 4, 256, 128, 4096)  # four rounds of one, or one of four: equal shares
    assert not p.whole and p.most == 1


@pytest.mark.parametrize("fmt,B,M,H,whole_at,cut_at", [
    ("bf16", 64, 1, 128, 600, 1024), ("bf16", 64, 4, 128, 1024, 4096), ("bf16", 256, 1, 128, 1024, 2048),
    ("bf16", 128, 2, 128, 1024, 4096), ("bf16", 32, 8, 128, 1024, 4096), ("bf16", 200, 1, 16, 300, 1000),
    ("bf16", 500, 1, 128, 500, 2000), ("f16x2", 128, 1, 128, 300, 600), ("f16x2", 64, 2, 128, 100, 600)])
def test_long_sequences_of_differing_lengths_are_cut(cut, fmt, B, M, H, whole_at, cut_at):
    """As measured on lengths spread evenly up to the table's width: whole
    sequences while they are short, ranges from there on at any length, also
    where the workgroups of whole sequences fill the device to the last CU."""
    assert cut(fmt, B, M, H, whole_at).whole and cut(fmt, B, M, H, whole_at // 4).whole
    for n in (cut_at, 2 * cut_at, 4 * cut_at, 32 * cut_at):
        assert not cut(fmt, B, M, H, n).whole, n


@pytest.mark.parametrize("fmt", ["bf16", "f16x2"])
def test_a_list_counts_in_full(cut, fmt):
    """Rows of a batch choose as many pages each: 256 lists of 16 pages of 64."""
    assert cut(fmt, 256, 1, 128, 1024, lists=True).whole


@pytest.mark.parametrize("fmt", ["bf16", "f16x2"])
@pytest.mark.parametrize("seed", range(30))
def test_every_tile_once_behind_the_empty_ones(cut, fmt, seed):
    """The row of tiles with empty ones before every unit but the first: each
    range finds the unit that it begins in, goes on from there and takes every
    tile once, and what joins a unit's parts finds each of them."""
    rng = random.Random(seed)
    lead = cut.costs[fmt].lead
    tiles = [rng.choice([0, 0, 1, 2, rng.randint(0, 40), rng.randint(0, 1000)]) for _ in range(rng.randint(1, 900))]
    total = [t + lead if t else 0 for t in tiles]  # a unit with its empty tiles
    if not any(tiles):
        return
    W = sum(total) - lead
    N = cut.ranges(W, rng.choice([2, 7, 64, 256]), rng.choice([0.5, 4.0, 64.0, 1e6]))
    first, at = [], 0  # first tile of each: `lead` tiles of the first one would stand before 0
    for t in total:
        first.append(at)
        at += t
    taken, parts = [[0] * t for t in tiles], {}
    for r in range(N):
        s, e = cut.begin(W, N, r), cut.begin(W, N, r + 1)
        assert s < e
        found = [u for u, t in enumerate(total) if first[u] <= s + lead < first[u] + t]
        assert len(found) == 1
        u, f, at = found[0], first[found[0]], s
        while True:  # the parts of a range, as the kernel walks them
            while at < e and u < len(tiles) and not tiles[u]:
                u += 1
            if at >= e or u == len(tiles):
                break
            b0, b1 = max(at - f, 0), min(e - f, tiles[u])
            if b0 >= b1:
                break
            for x in range(b0, b1):
                taken[u][x] += 1
            if (b0, b1) != (0, tiles[u]):
                assert parts.setdefault(cut.slot(r, s <= f), (u, r)) == (u, r)
            f += tiles[u] + lead
            at = f
            u += 1
    assert all(x == 1 for t in taken for x in t)
    assert all(0 <= k < 2 * N for k in parts)
    joined = []
    for u, t in enumerate(tiles):
        if t:
            r0, r1 = cut.range_of(W, N, first[u]), cut.range_of(W, N, first[u] + t - 1)
            if r1 > r0:
                joined += [(parts[cut.slot(r, r == r0)], (u, r)) for r in range(r0, r1 + 1)]
    assert all(a == b for a, b in joined) and len(joined) == len(parts)
