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
struct PlanCostsMany : PlanCosts {
    int32_t slots;  // workgroups that run on a CU at a time
    int32_t few;    // lead where a workgroup has all of a unit's heads
};
inline int32_t plan_places(const PlanCosts &, int32_t cus) { return cus; }
inline int32_t plan_places(const PlanCostsMany &c, int32_t cus) { return cus * c.slots; }
inline int32_t plan_lead(const PlanCosts &c, int32_t) { return c.lead; }
// How many units' ranges pay with a wide join (plan_call).
inline int32_t plan_wide(const PlanCosts &, int32_t units, int32_t) { return 2 * units; }
inline int32_t plan_lead(const PlanCostsMany &c, int32_t groups) { return groups <= c.waves ? c.few : c.lead; }
inline int32_t plan_wide(const PlanCostsMany &c, int32_t units, int32_t groups) {
    return groups <= c.waves && units < 4 ? 8 : 2 * units;
}
// lead: 64 sequences of up to 8192 positions take 134 us with 0, 127 with 4, 117
// with 8, 118 with 16.  ratio: one row over 32768 positions 33.9 us with 2, 32.8
// with 4, 32.3 with 8; 4 rows over up to 500 14.7, 14.9, 15.4.  bytes_ratio (2 x
// 32 KB at a 5 TB/s that all share): 5 x 4 rows over up to 2083 positions 39.1 us
// without, 35.9 with 150, 32.8 with 75, which was the worst for short sequences
// (49 rows of up to 24) before these went whole.
constexpr PlanCosts kCostsBf16 = {8, 8, 4, 150, 2.5f, 20};
// (a tile takes twice as long) lead: 11 x 3 rows 104 to 111 us with 0, 96.2 with 2,
// 96.3 with 4, 99.4 with 8.  ratio: one row over 500 positions 18.6 us with 4, 15.8
// with 16 and 32; over 10000 40.1, 35.1 and 32.8.  bytes_ratio: 63 x 4 rows of up to
// 25 positions took 66.5 us without and with 280, 80.4 with 140, before these went
// whole (51.1).
constexpr PlanCosts kCostsF16x2 = {4, 4, 16, 280, 1.3f, 10};
// (two workgroups of four waves a CU; a part in f16 is half as many bytes)  ratio:
// one row over 32768 positions 42.3 us with 4, 36.7 with 8, 40.1 with 12, over 8192
// 26.1, 23.1 and 24.9.  bytes_ratio: 64 sequences of up to 600 44.4 us with 150, 37.5
// with 300, 35.4 with 600; 20 x 3 rows over up to 1500 50.5, 44.6 and 44.6; 12 of up
// to 3000 37.5, 35.0 and 32.8; 256 of up to 2048 133 with each.  lead: 256 of up to
// 1024 86.6 us with 4, 91.6 with 8, 93.6 with 14.  few: the same with 64 heads 60.5
// with 2, 56.9 with 4, 59.7 with 8, with 16 heads 37.3, 38.2 and 41.4.  (Heads are
// spread over the CUs, which then take two ranges each, and not over their places:
// one row over 32768 took 13 % more so.)
constexpr PlanCostsMany kCostsI8 = {{4, 8, 8, 300, 2.5f, 20}, 2, 4};
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
// results sooner (one row over 509 positions 18.4 us with 8 column groups a
// workgroup, 12.3 with one; one row over 32 listed pages of 64 23.1 and 16.0).
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
// sequences of up to 1024 positions 44 and 46 us, of up to 8192 117 and 347; 256
// of up to 1024 105 and 85, of up to 4096 220 and 257; 64 x 4 of up to 1024 94 and
// 76, of up to 4096 194 and 236.  All of them that long: 256 of 2048 204 and 177,
// 64 x 4 of 4096 309 and 291; one of them, the others a sixteenth: 65 and 127, 75
// and 229; none of them, all a sixteenth of the table: 66 and 32, 55 and 38 (a
// table cut to the pages in use is cheaper).
// Up to `brief` tiles a sequence the ranges' tiles count in full: they save
// little where one is long, and cost more where all are.  64 of up to 600
// positions 40 and 31 us, all of them that long 47 and 36, one of them 32 and 34.
//
// Where a unit's column groups alone fill the CUs (prompt rows), there is one
// range: its workgroups each go through all units, in rounds over the CUs,
// leave no parts and need no join.  Their tiles differ only by their rows' place
// in a unit, where whole units of differing lengths may leave CUs idle, so these
// have to be fewer by a tenth.  Of 128 heads, whole and as one range: 4 x 256 rows
// over up to 4096 positions 707 and 720 us, 3 x 777 over up to 1900 689 and 724 (in
// f16 pairs 2134 and 2243, in 8 bits 800 and 839), 5 x 300 over up to 300 176 and
// 201, 2 x 512 over up to 1024 211 and 207.
template <class Costs>
PlanCall plan_call(const Costs &c, int32_t cus, int32_t units, int32_t groups, int64_t each, int64_t listed,
                   bool lists) {
    PlanCall p{};
    const int32_t lead = plan_lead(c, groups);
    const int64_t tiles = units * each, empty = (int64_t)(units - 1) * lead, W = tiles + empty;
    plan_heads(p, c, cus, groups, units);
    const int32_t places = plan_places(c, cus);
    const int64_t turns = ((int64_t)units * p.chunks + places - 1) / places;
    const float whole = (float)(turns * (listed + lead) - lead);
    auto cut = [&](int32_t times) {
        p.spread = fminf((float)times * (float)c.ratio, (float)c.bytes_ratio / (float)groups);
        plan_heads(p, c, cus, groups, plan_ranges(tiles, places, p.spread));
        p.most = plan_ranges(W, p.chunks < places ? places / p.chunks : 1, p.spread);
    };
    cut(units);
    if (p.most == 1) {
        const int64_t rounds = ((int64_t)p.chunks + places - 1) / places;
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
    // are few units of many parts: one row over 32768 positions 38.4 us with 4
    // waves, 33.9 with 16, 32.8 with the ranges (over 509, 8 parts, they gain nothing).
    // A few units of 8-bit pages whose heads a workgroup has all take few places, so
    // that they get eight units' in all: 64 heads over 32768 positions 32.4 us with
    // twice, 32.6 with four times, 30.2 with eight times the ranges, 16 heads 28.2,
    // 26.3 and 24.1, two rows of 16 heads over up to 4096 17.2, 17.2 and 15.4, four
    // 17.6, 19.2 and 17.7; 128 heads over 32768 36.7, 38.4 and 37.6.
    p.wide = (int64_t)units * groups * kPlanJoinSlices <= cus && p.most > 16 * units;
    if (p.wide) cut(plan_wide(c, units, groups));
    p.slots = plan_slot(p.most, false) * groups;
    return p;
}
// Rows with a window: of the positions before its end a row sees the last
// `window` and the first `sinks`.  A sequence's rows end at n - M + 1 .. n.  Its
// tiles are the first `ts`, which hold the first positions, and those from the one
// on where the first row's window begins; `skip` tiles between them are left out.
struct NearCut {
    int32_t start;  // the first row's window
    int32_t ts, skip;
};
UT_PLAN_FN NearCut near_cut(int32_t n, int32_t M, int32_t window, int32_t sinks, int32_t tile) {
    const int32_t end = n - M + 1, start = end > window ? end - window : 0, from = start / tile;
    const int32_t s = sinks < n ? sinks : n, ts = (int32_t)(((int64_t)s + tile - 1) / tile);
    return {start, ts < from ? ts : from, ts < from ? from - ts : 0};
}
// The first position of tile x.
UT_PLAN_FN int32_t near_tile(const NearCut &c, int32_t x, int32_t tile) { return (x >= c.ts ? x + c.skip : x) * tile; }
// Tiles of a sequence at most.  (The windows may begin and end inside a tile, and
// so may the first positions.)
UT_PLAN_FN int64_t near_most(int64_t M, int64_t window, int64_t sinks, int64_t tile) {
    return (window + M - 1 + tile - 1) / tile + 1 + (sinks + tile - 1) / tile;
}
// No row sees any of the `count` positions from v0 on.
UT_PLAN_FN bool near_hidden(const NearCut &c, int32_t sinks, int32_t v0, int32_t count) {
    return v0 >= sinks && v0 + count <= c.start;
}
// The visible positions of the 32 from v0 on: for a row that ends at n, for some
// row of a sequence (windows follow on one another: together they are one run), and
// for every row.
UT_PLAN_FN uint32_t low_bits(int32_t c) { return c >= 32 ? ~0u : c <= 0 ? 0u : (1u << c) - 1u; }
UT_PLAN_FN uint32_t near_seen(int32_t v0, int32_t n, int32_t window, int32_t sinks) {
    const int32_t from = n > window ? n - window - v0 : 0;
    return low_bits(n - v0) & (~low_bits(from) | low_bits(sinks - v0));
}
UT_PLAN_FN uint32_t near_some(const NearCut &c, int32_t v0, int32_t n, int32_t sinks) {
    return low_bits(n - v0) & (~low_bits(c.start - v0) | low_bits(sinks - v0));
}
UT_PLAN_FN uint32_t near_every(int32_t v0, int32_t n, int32_t M, int32_t window, int32_t sinks) {
    return near_seen(v0, n, window, sinks) & low_bits(n - M + 1 - v0);
}
// Positions of a sequence or a selection: tile and page counts may step past
// the end by some tiles and stay in 32 bits.
constexpr int64_t kMostPositions = INT32_MAX - 1023;
// Workgroups along a grid's first axis, where pages set them: 2^22, and of larger
// ones as many as have fewer than 2^32 threads, the most that a launch takes.
constexpr int64_t most_groups(int64_t threads) {
    const int64_t n = ((int64_t(1) << 32) - 1) / threads;
    return n < (1 << 22) ? n : 1 << 22;
}
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
