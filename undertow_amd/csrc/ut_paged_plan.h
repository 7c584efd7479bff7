// ut_paged_plan.h -- how a batch over the paged cache is cut into equal
// ranges of work, and the bounds of what its lengths and tables may say.
// Plain arithmetic for the kernels and for the host.  (Where every sequence is
// short by what the table holds, a workgroup takes one whole, and there are no
// ranges: plan_call.)
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

// Workgroups of the join that share a column group's dims.
constexpr int kPlanJoinSlices = 8;

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
// A call's cut, settled on the host by what the table holds at most.
struct PlanCosts {  // of a cache format
    int32_t waves;  // column groups of a workgroup at most
    // empty tiles that stand for the queries, first tiles and result of a
    // sequence that begins in a range
    int32_t lead;
    int32_t ratio;        // a tile's time to a part's in the join (plan_ranges)
    int32_t bytes_ratio;  // and to that of a column group's part's bytes, written and read
    float join;           // the join's launch, in tiles
    int32_t brief;        // a sequence of so few tiles does not pay for the cut (plan_call)
};
// lead: 64 sequences of up to 8192 positions take 135 us with 0, 132 with 2, 126
// with 4, 115 with 8, 117 with 16.  ratio: one row over 32768 positions 48 us
// with 2, 44 with 3, 42 with 4, 41 with 8, and 59 in as many ranges as CUs; 4
// rows over 500 positions 19.8, 20.8, 20.4, 24.3.  bytes_ratio (2 x 32 KB at a 5
// TB/s that all share): 5 x 4 rows over up to 2083 positions 39.3 us without,
// 36.4 with 150, 35.3 with 75; 49 rows of up to 24 20.3, 18.5, 24.7.
constexpr PlanCosts kCostsBf16 = {8, 8, 4, 150, 2.5f, 20};
// (a tile takes twice as long) lead: 11 x 3 rows 103 us with 0, 96.1 with 2, 96.4
// with 4, 99.7 with 8.  ratio: one row over 500 positions 22.0 us with 4, 19.5
// with 16; over 10000 43.2 in as many ranges as CUs, 40.0 with 16, 40.6 with 32.
// bytes_ratio: 63 x 4 rows of up to 25 positions 66.5 us without and with 280,
// 80.4 with 140.
constexpr PlanCosts kCostsF16x2 = {4, 4, 16, 280, 1.3f, 10};
struct PlanCall {
    int32_t whole;        // a range is a unit: no parts, no join
    int32_t most;         // ranges at most (whole: units)
    int32_t per, chunks;  // column groups of a workgroup, workgroups that share a range
    int32_t wide;         // the join takes 16 waves a workgroup
    float spread;         // plan_ranges'
    int64_t slots;        // places for parts: none for whole units, nor for one range
};
// Where n ranges (or whole units) leave CUs free, a call's heads are spread
// over them: a workgroup of few columns issues its queries, tiles' products and
// results sooner (one row over 509 positions 18.9 us with 8 column groups a
// workgroup, 15.8 with one; one row over 32 listed pages of 64 23.7 and 21.1).
inline void plan_heads(PlanCall &p, const PlanCosts &c, int32_t cus, int32_t groups, int32_t n) {
    const int32_t free = n < cus ? cus / n : 1;
    p.per = free < groups ? (groups + free - 1) / free : 1;
    p.per = p.per < c.waves ? p.per : c.waves;
    p.chunks = (groups + p.per - 1) / p.per;
    p.per = (groups + p.chunks - 1) / p.chunks;
}
// `units` units of `groups` column groups and of `each` tiles at most; of a list
// (`lists`) `listed` are to be expected, of a table half: a batch's lengths
// differ, and its longest sequence sets the table's width.
//
// Whole units, one or more after another on a CU, or equal ranges (the empty
// tiles do not count for the heads' spread) and their join, whichever takes
// fewer tiles' time: whole units that of the longest one, ranges that of the
// tiles there are.  Cut and whole, lengths spread evenly up to the longest: 64
// sequences of up to 1024 positions 45 and 48 us, of up to 8192 113 and 313; 256
// of up to 1024 105 and 85, of up to 4096 218 and 264; 64 x 4 of up to 1024 94 and
// 78, of up to 4096 189 and 245.  All of them that long: 256 of 2048 204 and 177,
// 64 x 4 of 4096 309 and 291; one of them, the others a sixteenth: 65 and 127, 75
// and 229; none of them, all a sixteenth of the table: 66 and 32, 55 and 38 (a
// table cut to the pages in use is cheaper).
// Up to `brief` tiles a sequence the ranges' tiles count in full: they save
// little where one is long, and cost more where all are.  64 of up to 600
// positions 40 and 34 us, all of them that long 47 and 36, one of them 32 and 34.
//
// Where a unit's column groups alone fill the CUs (prompt rows), there is one
// range: its workgroups each go through all units, in rounds over the CUs,
// leave no parts and need no join.  They have the same tiles each, where whole
// units of differing lengths leave CUs idle, so these have to be fewer by a
// tenth.  4 x 256 rows of 128 heads over up to 4096 positions (equal counts) take
// 1034 us whole and 741 as one range with lengths spread evenly, 1055 and 1048
// with equal ones; 3 x 777 over up to 1900 (whole 0.86 of the range) 1249 and 1368,
// 1341 and 1781; in f16 pairs (0.92) 5.35 ms and 4.63, 5.33 and 5.93.
inline PlanCall plan_call(const PlanCosts &c, int32_t cus, int32_t units, int32_t groups, int64_t each,
                          int64_t listed, bool lists) {
    PlanCall p{};
    const int64_t tiles = units * each, empty = (int64_t)(units - 1) * c.lead, W = tiles + empty;
    plan_heads(p, c, cus, groups, units);
    const int64_t turns = ((int64_t)units * p.chunks + cus - 1) / cus;
    const float whole = (float)(turns * (listed + c.lead) - c.lead);
    auto cut = [&](int32_t ratio) {
        p.spread = fminf((float)units * ratio, (float)c.bytes_ratio / (float)groups);
        plan_heads(p, c, cus, groups, plan_ranges(tiles, cus, p.spread));
        p.most = plan_ranges(W, p.chunks < cus ? cus / p.chunks : 1, p.spread);
    };
    cut(c.ratio);
    if (p.most == 1) {
        const int64_t rounds = ((int64_t)p.chunks + cus - 1) / cus;
        p.whole = units == 1 || whole < 0.9f * (float)(rounds * W);
    } else {
        const float there = lists || each <= c.brief ? (float)W : 0.5f * (float)tiles + (float)empty;
        p.whole = whole <= there / p.most + c.join + (float)p.most * groups / c.bytes_ratio;
    }
    if (p.whole) {
        plan_heads(p, c, cus, groups, units);
        p.most = units;
        return p;
    }
    if (p.most == 1) return p;
    // The join takes 16 waves a workgroup, and twice the ranges pay, where there
    // are few units of many parts: one row over 32768 positions 42.8 us with 4
    // waves, 39.5 with 16, 37.2 with the ranges (over 509, 8 parts, 15.5 and 15.9).
    p.wide = (int64_t)units * groups * kPlanJoinSlices <= cus && p.most > 16 * units;
    if (p.wide) cut(2 * c.ratio);
    p.slots = plan_slot(p.most, false) * groups;
    return p;
}
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
