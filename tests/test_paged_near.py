"""Which tiles of a sequence a windowed call takes and what its rows see in them
(undertow_amd/csrc/ut_paged_plan.h), on the CPU, against the definition; and how
calls over 8-bit pages are cut."""
import ctypes as C
import random
import subprocess
from pathlib import Path

import pytest

CSRC = Path(__file__).resolve().parents[1] / "undertow_amd" / "csrc"
TILE = 32

SRC = r"""
#include "ut_paged_plan.h"
extern "C" {
void near(int n, int M, int window, int sinks, int *out) {
    ut::NearCut c = ut::near_cut(n, M, window, sinks, 32);
    out[0] = c.start; out[1] = c.ts; out[2] = c.skip;
}
static ut::NearCut cut(const int *c) { return {c[0], c[1], c[2]}; }
int tile(const int *c, int x) { return ut::near_tile(cut(c), x, 32); }
int64_t most(int64_t M, int64_t window, int64_t sinks) { return ut::near_most(M, window, sinks, 32); }
int hidden(const int *c, int sinks, int v0, int count) { return ut::near_hidden(cut(c), sinks, v0, count); }
uint32_t seen(int v0, int n, int window, int sinks) { return ut::near_seen(v0, n, window, sinks); }
uint32_t some(const int *c, int v0, int n, int sinks) { return ut::near_some(cut(c), v0, n, sinks); }
uint32_t every(int v0, int n, int M, int window, int sinks) { return ut::near_every(v0, n, M, window, sinks); }
void plan(int cus, int units, int groups, int64_t each, int64_t listed, int lists, int64_t *out) {
    ut::PlanCall p = ut::plan_call(ut::kCostsI8, cus, units, groups, each, listed, lists);
    out[0] = p.whole; out[1] = p.most; out[2] = p.per; out[3] = p.chunks; out[4] = p.slots;
}
int waves(void) { return ut::kCostsI8.waves; }
int size(int call) { return call ? sizeof(ut::PlanCall) : sizeof(ut::PlanCosts); }
int places(int cus) { return cus * ut::kCostsI8.slots; }
}
"""


@pytest.fixture(scope="module")
def L(tmp_path_factory):
    d = tmp_path_factory.mktemp("near")
    (d / "n.cpp").write_text(SRC)
    subprocess.run(["g++", "-std=c++17", "-O1", "-fsanitize=undefined", "-fno-sanitize-recover", "-shared", "-fPIC", "-I", str(CSRC),
                    "-o", str(d / "n.so"), str(d / "n.cpp")], check=True)
    lib = C.CDLL(str(d / "n.so"))
    for f in ("seen", "some", "every"):
        getattr(lib, f).restype = C.c_uint32
    lib.most.restype, lib.most.argtypes = C.c_int64, [C.c_int64] * 3
    lib.plan.argtypes = [C.c_int] * 3 + [C.c_int64] * 2 + [C.c_int, C.POINTER(C.c_int64)]
    return lib


def sees(t, n, window, sinks):
    return 0 <= t < n and (t < sinks or t >= n - window)


def mask(v0, want):
    return sum(1 << i for i in range(TILE) if want(v0 + i))


@pytest.mark.parametrize("seed", range(60))
def test_tiles_hold_what_rows_see(L, seed):
    rng = random.Random(seed)
    for _ in range(12):
        n = rng.choice([0, 1, rng.randint(1, 70), rng.randint(1, 700)])
        M = rng.choice([1, 2, 3, rng.randint(1, 50), rng.randint(1, 200)])
        window = rng.choice([1, rng.randint(1, 40), rng.randint(1, 300), 1000])
        sinks = rng.choice([0, 1, 4, rng.randint(0, 70), rng.randint(0, 400), 5000])
        cut = (C.c_int * 3)()
        L.near(n, M, window, sinks, cut)
        start, ts, skip = cut
        ends = [n - M + 1 + j for j in range(M)]
        tiles = -(-n // TILE) - skip
        assert 0 <= tiles <= L.most(M, window, sinks) and skip >= 0 and 0 <= ts
        at = [L.tile(cut, x) for x in range(tiles)]
        assert at == sorted(set(at)) and all(v % TILE == 0 and v < n for v in at)
        held = {v + i for v in at for i in range(TILE)}
        some = {t for t in range(n) if any(sees(t, e, window, sinks) for e in ends)}
        assert some <= held
        for v0 in at:
            for e in rng.sample(ends, min(5, M)):
                assert L.seen(v0, e, window, sinks) == mask(v0, lambda t: sees(t, e, window, sinks))
            assert L.some(cut, v0, n, sinks) == mask(v0, lambda t: t in some)
            assert L.every(v0, n, M, window, sinks) == mask(v0, lambda t: all(sees(t, e, window, sinks) for e in ends))
            for g in range(0, TILE, 8):  # pages of such positions alone need no name
                if L.hidden(cut, sinks, v0 + g, 8):
                    assert not any(t in some for t in range(v0 + g, v0 + g + 8))


def test_the_widest_numbers(L):
    """Longest sequences, windows and counts of first positions: nothing passes
    32 bits (the library is built to end at an overflow)."""
    longest = 2**31 - 1024
    cut = (C.c_int * 3)()
    for n, M in ((longest, 1), (longest, 65535), (0, 65535), (5, 65535)):
        for window, sinks in ((1, 0), (longest, 0), (longest, longest), (1, longest), (4096, 64)):
            L.near(n, M, window, sinks, cut)
            tiles = -(-n // TILE) - cut[2]
            assert 0 <= tiles <= min(L.most(M, window, sinks), -(-n // TILE))
            for x in (0, tiles - 1, tiles + 7):
                v0 = L.tile(cut, max(x, 0))
                L.seen(v0, n, window, sinks), L.some(cut, v0, n, sinks), L.every(v0, n, M, window, sinks)


@pytest.mark.parametrize("seed", range(40))
def test_calls_over_8_bit_pages_are_cut(L, seed):
    """Every column group is taken, no more workgroups are asked for than have
    a place where there is something to join, and parts have theirs."""
    rng = random.Random(seed)
    for _ in range(20):
        cus = rng.choice([256, 256, 304, 8])
        units, groups = rng.choice([1, 2, 64, rng.randint(1, 700)]), rng.choice([1, 2, 4, 8, rng.randint(1, 4000)])
        each = rng.choice([1, 16, rng.randint(1, 2000)])
        out = (C.c_int64 * 5)()
        L.plan(cus, units, groups, each, min(each, rng.randint(1, 2000)), rng.random() < 0.5, out)
        whole, most, per, chunks, slots = out
        assert 1 <= per <= L.waves() and per * chunks >= groups and per * (chunks - 1) < groups
        if whole:
            assert most == units and slots == 0
        else:
            assert 1 <= most and (most == 1 or most * chunks <= L.places(cus))
            assert slots == (0 if most == 1 else 2 * most * groups)


def test_what_other_tests_hold_of_a_plan_has_its_size(L):
    import test_paged_cut as cut
    assert [L.size(0), L.size(1)] == [C.sizeof(cut.Costs), C.sizeof(cut.Call)]
