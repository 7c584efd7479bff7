"""How a batch over the paged cache is cut into ranges
(undertow_amd/csrc/ut_paged_plan.h), on the CPU: every tile is taken once,
parts of one sequence meet again, and no two parts share a place; and the
bounds of lengths and page ids."""
import ctypes as C
import random
import subprocess
from pathlib import Path

import pytest

CSRC = Path(__file__).resolve().parents[1] / "undertow_amd" / "csrc"

SRC = r"""
#include "ut_paged_plan.h"
extern "C" {
int64_t ranges(int64_t W, int64_t most, float spread) { return ut::plan_ranges(W, (int32_t)most, spread); }
int64_t begin(int64_t W, int64_t N, int64_t r) { return ut::plan_begin(W, N, r); }
int64_t range_of(int64_t W, int64_t N, int64_t t) { return ut::plan_range_of(W, N, t); }
int64_t slot(int64_t r, int64_t begins) { return ut::plan_slot(r, begins != 0); }
int len(int n, int64_t cap, int *bad) { bool b = false; int v = ut::plan_len(n, cap, b); *bad = b; return v; }
int page(int p, int n, int *bad) { bool b = false; int v = ut::plan_page(p, n, b); *bad = b; return v; }
}
"""


@pytest.fixture(scope="module")
def L(tmp_path_factory):
    d = tmp_path_factory.mktemp("plan")
    (d / "p.cpp").write_text(SRC)
    subprocess.run(["g++", "-std=c++17", "-O1", "-shared", "-fPIC", "-I", str(CSRC), "-o",
                    str(d / "p.so"), str(d / "p.cpp")], check=True)
    lib = C.CDLL(str(d / "p.so"))
    i = C.c_int64
    for f, n in (("ranges", 3), ("begin", 3), ("range_of", 3), ("slot", 2)):
        getattr(lib, f).restype, getattr(lib, f).argtypes = i, [i] * n
    lib.ranges.argtypes = [i, i, C.c_float]
    lib.len.argtypes = [C.c_int, i, C.POINTER(C.c_int)]
    lib.page.argtypes = [C.c_int, C.c_int, C.POINTER(C.c_int)]
    return lib


@pytest.mark.parametrize("seed", range(40))
def test_every_tile_once_and_parts_meet(L, seed):
    rng = random.Random(seed)
    tiles = [rng.choice([0, 1, 2, rng.randint(0, 40), rng.randint(0, 1000)]) for _ in range(rng.randint(1, 70))]
    W, most, spread = sum(tiles), rng.choice([1, 7, 64, 256, 512]), rng.choice([0.5, 4, 16, 64 * 16])
    N = L.ranges(W, most, spread)
    assert 1 <= N <= most and (N == 1 or N <= W)
    if W == 0:
        return
    assert N == min(most, W, max(1, int((W * spread) ** 0.5 + 0.5)))
    pre, at = [], 0
    for t in tiles:
        pre.append(at)
        at += t
    taken, parts = [0] * W, {}
    for r in range(N):
        s, e = L.begin(W, N, r), L.begin(W, N, r + 1)
        assert s < e  # no empty range
        for u, t in enumerate(tiles):
            a, b = max(s, pre[u]), min(e, pre[u] + t)
            if a >= b:
                continue
            for k in range(a, b):
                taken[k] += 1
                assert L.range_of(W, N, k) == r
            if b - a < t:
                parts.setdefault(L.slot(r, s <= pre[u]), []).append((u, r))
    assert taken == [1] * W
    assert all(len(v) == 1 for v in parts.values()) and all(0 <= k < 2 * N for k in parts)
    for u, t in enumerate(tiles):  # what joins the parts finds each of them
        if t:
            r0, r1 = L.range_of(W, N, pre[u]), L.range_of(W, N, pre[u] + t - 1)
            got = [parts[L.slot(r, r == r0)][0] for r in range(r0, r1 + 1)] if r1 > r0 else []
            assert got == [(u, r) for r in range(r0, r1 + 1)] * (r1 > r0)


def test_long_rows_stay_in_64_bits(L):
    W = 65535 * (1 << 26)  # the most sequences at the most tiles
    for N in (1, 255, 2048):
        assert L.begin(W, N, N) == W
        for r in (0, N // 2, N - 1):
            s, e = W * r // N, W * (r + 1) // N
            assert (L.begin(W, N, r), L.range_of(W, N, s), L.range_of(W, N, e - 1)) == (s, r, r)


@pytest.mark.parametrize("n,cap,want,bad", [(0, 64, 0, 0), (64, 64, 64, 0), (65, 64, 64, 1), (-1, 64, 0, 1),
                                            (2**31 - 1, 2**31 - 1, 2**31 - 1, 0), (-2**31, 128, 0, 1)])
def test_lengths_stay_within_the_table(L, n, cap, want, bad):
    b = C.c_int()
    assert (L.len(n, cap, C.byref(b)), b.value) == (want, bad)


@pytest.mark.parametrize("p,n,want,bad", [(0, 1, 0, 0), (6, 7, 6, 0), (7, 7, 0, 1), (-1, 7, 0, 1),
                                          (2**31 - 1, 7, 0, 1), (-2**31, 7, 0, 1)])
def test_pages_stay_within_the_pool(L, p, n, want, bad):
    b = C.c_int()
    assert (L.page(p, n, C.byref(b)), b.value) == (want, bad)
