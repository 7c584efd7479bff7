// ut_paged_plan.h -- how a batch over the paged cache is cut into equal
// ranges of work, and the bounds of what its lengths and tables may say.
// Plain arithmetic for the kernels and for the host.  (Where every sequence is
// short, a workgroup takes one whole, and there are no ranges.)
//
// The sequences' tiles stand in one row, one sequence after another, W in
// all.  Range r of N takes the tiles [W r / N, W (r + 1) / N), so a ragged
// batch is cut as evenly as a square one, and a long sequence spreads over
// many ranges.  A sequence that begins inside a range costs that range its
// queries and its result: some empty tiles stand before each but the first
// for that.  A range meets at most one sequence whose first tile lies
// before it and one that goes on behind it; those two leave a partial result
// each (plan_slot), every other sequence in it is whole.
#pragma once

#include <cmath>
#include <cstdint>

#if defined(__HIPCC__)
#define UT_PLAN_FN __host__ __device__ inline
#else
#define UT_PLAN_FN inline
#endif

namespace ut {

// How many ranges.  A row of t tiles in x of them costs t / x tiles one after
// another, and its x parts are joined one after another: least at x = sqrt(t
// tile / join).  For `units` rows of W tiles together that is N = sqrt(W units
// tile / join) in all.  All parts share the memory they pass through: joined
// in `bytes` each at once, N = sqrt(W tile / bytes).  spread is the smaller of
// units tile / join and tile / bytes; `most` ranges at most, of one tile at least.
UT_PLAN_FN int32_t plan_ranges(int64_t W, int32_t most, float spread) {
    const float x = (float)W * spread, top = (float)most;
    int32_t n = most;
    if (x < top * top) {
#if defined(__HIP_DEVICE_COMPILE__)
        n = (int32_t)(__builtin_amdgcn_sqrtf(x) + 0.5f);  // the nearest or the next one: no matter
#else
        n = (int32_t)(sqrtf(x) + 0.5f);
#endif
        n = n < most ? n : most;
    }
    n = (int64_t)n < W ? n : (int32_t)W;
    return n < 1 ? 1 : n;
}
// (the longer ranges lie among the others: all in front, and so on the first
// XCDs, costs 64 long sequences 1 %)
UT_PLAN_FN int64_t plan_begin(int64_t W, int64_t N, int64_t r) { return W * r / N; }
// The range that holds tile t.
UT_PLAN_FN int64_t plan_range_of(int64_t W, int64_t N, int64_t t) { return ((t + 1) * N - 1) / W; }
// Where range r leaves its part of a sequence that begins in it, or of the one
// that began before it.
UT_PLAN_FN int64_t plan_slot(int64_t r, bool begins) { return 2 * r + (begins ? 1 : 0); }
// Positions of a sequence or a selection: tile and page counts may step past
// the end by some tiles and stay in 32 bits.
constexpr int64_t kMostPositions = INT32_MAX - 1023;
// A length cut to what the table can hold; a page id cut to the pool.
UT_PLAN_FN int32_t plan_len(int32_t n, int64_t cap, bool &bad) {
    if (n >= 0 && n <= cap) return n;
    bad = true;
    return n < 0 ? 0 : (int32_t)cap;
}
UT_PLAN_FN int32_t plan_page(int32_t p, int32_t n_pages, bool &bad) {
    if (p >= 0 && p < n_pages) return p;
    bad = true;
    return 0;
}

}  // namespace ut
