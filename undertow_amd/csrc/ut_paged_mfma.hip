// ut_paged_mfma.hip -- attention over the paged latent cache on the matrix
// cores, for latent 512 + rope 64 and pages of 8 positions and more.
//
// For a row's heads q_h and the positions t it sees, one pass over the cache:
//   s_ht = scale (q_h . [latent_t | krot_t]),
//   out_h = sum_t e^(s_ht - m_h) latent_t / sum_t e^(s_ht - m_h),
// with m_h the largest score so far, or one not far below it.
//
// Each position is 1152 bytes (f16x2: 2304) and costs 128 heads 2 * 128 *
// (576 + 512) operations: at 5.1 TB/s and 1.2 PFLOP/s (a large copy's and a
// large matrix product's rates) 0.23 ns against 0.23 ns, so memory and matrix
// cores have to be busy all the time, and together.  Hence:
// - 16 columns (heads of one row) a wave with the whole latent width in
//   registers (128 of context, 72 of queries), so that scores, weights and
//   contexts never leave the wave.  32 columns spill; two waves to a column
//   group, each with half of the tiles, took 145 us instead of 130 (64
//   sequences of up to 8192 positions).
// - eight such waves over one tile of 32 positions in LDS: K is read from it
//   as it lies, V transposed by the LDS reads, and three further tiles are on
//   their way, straight to LDS.
// - equal ranges of the whole batch's tiles, one workgroup a CU
//   (ut_paged_plan.h), and a join of what the ranges leave (k_paged_join); whole
//   sequences, or one range, where there is nothing to join.
//
// A tile of 128 heads takes 1.95 us: 1.17 PFLOP/s and, with one row a sequence,
// 4.8 TB/s over 256 CUs; the LDS reads alone would take 1.1 us of it (K 288 KB
// at 558 B/ns, V 256 KB at 431, as measured by themselves).  64 ragged
// sequences of up to 8192 positions (329 MB): 115 us, of which products and
// copies 70, the start 9 (lengths 1.4, queries issued 4.6, first tiles 8.7 us
// from the start), partial results written 5 to 10, their join 16 (82 MB each
// way).
#include <type_traits>

#include "ut_paged.h"

namespace ut {

typedef __bf16 pbf16x8 __attribute__((ext_vector_type(8)));
typedef __bf16 pbf16x4 __attribute__((ext_vector_type(4)));
typedef __bf16 pbf16x2 __attribute__((ext_vector_type(2)));
typedef _Float16 pf16x8 __attribute__((ext_vector_type(8)));
typedef float pf32x4 __attribute__((ext_vector_type(4)));
typedef uint32_t pu32x4 __attribute__((ext_vector_type(4)));
typedef __attribute__((address_space(3))) uint8_t lds_u8;

constexpr int kPT = 32;             // positions per tile
constexpr int kPL = 512, kPD = 576;
constexpr int kCols = 16;           // heads per column group (a wave's)
static_assert(kPlanJoinSlices * 64 == kPL, "a workgroup of the join takes 64 dims");
constexpr float kLog2e = 1.44269504088896341f;
constexpr float kLow = -3.402823466e38f;  // the offset before any score

struct PagedMfmaArgs {
    PagedArgs a;
    int32_t units;    // sequences, or rows where each has pages of its own
    int32_t groups;   // column groups (16 heads of one row) of a unit
    int32_t chunks;   // workgroups that share a unit's positions
    int32_t per;      // column groups of a workgroup
    int32_t most;     // ranges at most
    float spread;     // plan_ranges'
    int32_t whole;    // a range is a unit (most: units), and there is no join
    float *part_o;    // [slot][group][128 quads][16 columns][4]
    float *part_ml;   // [slot][group][16 columns][2]
    int64_t *plan;    // [units] first tile of each, then W (where there is more than one range)
    int32_t lead;     // empty tiles before every unit with tiles but the first
};

// What a call's rows see: all positions up to their own, the listed pages, or
// the first ones and a window.
enum { kAll, kListed, kNear };

// With a window a sequence's tiles are its first `ts`, which hold the first
// positions, and those from the one on where the first row's window begins;
// `skip` tiles between them are left out.
struct NearCut {
    int32_t start;  // the first row's window
    int32_t ts, skip;
};
__device__ __forceinline__ NearCut near_cut(const PagedArgs &a, int32_t n) {
    const int32_t end = n - a.M + 1, start = end > a.window ? end - a.window : 0, from = start / kPT;
    const int32_t s = a.sinks < n ? a.sinks : n, ts = (int32_t)(((int64_t)s + kPT - 1) / kPT);
    return {start, ts < from ? ts : from, ts < from ? from - ts : 0};
}

// Tiles of a unit.
template <int KIND> __device__ __forceinline__ int32_t unit_tiles(const PagedArgs &a, int u) {
    if (KIND != kListed) {
        const int32_t n = paged_len(a, u), tiles = (int32_t)(((int64_t)n + kPT - 1) / kPT);
        return KIND == kNear ? tiles - near_cut(a, n).skip : tiles;
    }
    const int b = u / a.M, n = paged_len(a, b) - a.M + (u - b * a.M) + 1;
    return n > 0 ? (int32_t)((((int64_t)a.top_k << a.shift) + kPT - 1) / kPT) : 0;
}

// The sum of v over the workgroup's threads before this one, and in all.
template <int NW> __device__ __forceinline__ int64_t block_scan(int64_t v, int64_t *s, int64_t &all) {
    const int lane = threadIdx.x & 63, w = threadIdx.x >> 6;
    int64_t x = v;
    for (int off = 1; off < 64; off <<= 1) {
        const int64_t y = __shfl_up(x, off, 64);
        if (lane >= off) x += y;
    }
    __syncthreads();
    if (lane == 63) s[w] = x;
    __syncthreads();
    int64_t before = x - v;
    all = 0;
    for (int i = 0; i < NW; i++) {
        if (i < w) before += s[i];
        all += s[i];
    }
    return before;
}

// A value that every lane has, in scalar registers.
__device__ __forceinline__ int64_t uniform(int64_t v) {
    const uint32_t lo = __builtin_amdgcn_readfirstlane((uint32_t)v);
    return (int64_t)((uint64_t)__builtin_amdgcn_readfirstlane((uint32_t)((uint64_t)v >> 32)) << 32 | lo);
}

struct Range {
    int64_t W, s, e;  // the range takes tiles [s, e) of W
    int u;               // the unit that holds tile s, and its first tile (behind its empty ones)
    int64_t first;
};

// Every workgroup works its range out from the lengths.  `leave`: the units'
// first tiles are written down for the join.
template <int KIND, int NW>
__device__ bool find_range(const PagedMfmaArgs &p, int64_t r, bool leave, Range &g) {
    __shared__ int64_t s[NW];
    __shared__ int64_t found[2];
    const int tid = threadIdx.x;
    if (p.whole) {
        const PagedArgs &a = p.a;
        const int u = (int)r;
        g = {0, 0, __builtin_amdgcn_readfirstlane(unit_tiles<KIND>(a, u)), u, 0};
        if (KIND == kListed && g.e > 0) {
            // a list's tiles up to its last page that the row sees (one at least)
            const int b = u / a.M, n = paged_len(a, b) - a.M + (u - b * a.M) + 1;
            int64_t end = 0;
            for (int32_t i = 0; i < a.top_k; i += 64) {
                const int32_t at = i + (tid & 63), page = at < a.top_k ? a.sel[(int64_t)u * a.top_k + at] : -1;
                const uint64_t seen = __ballot(page >= 0 && ((int64_t)page << a.shift) < n);
                if (seen) end = i + 64 - __builtin_clzll(seen);
            }
            const int64_t tiles = ((end << a.shift) + kPT - 1) / kPT;
            g.e = uniform(tiles > 0 ? tiles : 1);
        }
        return g.e > 0;
    }
    if (p.units <= 64) {
        // every wave by itself
        const int lane = tid & 63;
        int32_t t = lane < p.units ? unit_tiles<KIND>(p.a, lane) : 0;
        t += t > 0 ? p.lead : 0;
        int64_t x = t;
        for (int off = 1; off < 64; off <<= 1) {
            const int64_t y = __shfl_up(x, off, 64);
            if (lane >= off) x += y;
        }
        const int64_t all = uniform(__shfl(x, 63, 64)), pre = x - t;
        g.W = all > 0 ? all - p.lead : 0;
        if (leave && tid < p.units) p.plan[tid] = pre;
        if (leave && tid == 0) p.plan[p.units] = g.W;
        if (g.W == 0) return false;
        const int64_t N = plan_ranges(g.W, p.most, p.spread);
        if (r >= N) return false;
        g.s = plan_begin(g.W, N, r);
        g.e = plan_begin(g.W, N, r + 1);
        const int64_t at = g.s + p.lead;
        const int lead = __builtin_ctzll(__ballot(pre <= at && at < pre + t));
        g.u = __builtin_amdgcn_readfirstlane(lead);
        g.first = uniform(__shfl(pre, lead, 64));
        return true;
    }
    int64_t W = 0;
    int64_t t, pre;  // the last turn's
    for (int c = 0; c < p.units; c += NW * 64) {
        const int u = c + tid;
        int64_t all;
        t = u < p.units ? unit_tiles<KIND>(p.a, u) : 0;
        // lead tiles before each unit that has tiles, but for the row's first
        t += t > 0 ? p.lead : 0;
        pre = W + block_scan<NW>(t, s, all);
        if (leave && u < p.units) p.plan[u] = pre;
        W += all;
    }
    W -= W > 0 ? p.lead : 0;
    if (leave && tid == 0) p.plan[p.units] = W;
    g.W = W = uniform(W);
    if (W == 0) return false;
    const int64_t N = plan_ranges(W, p.most, p.spread);
    if (r >= N) return false;
    g.s = plan_begin(W, N, r);
    g.e = plan_begin(W, N, r + 1);
    // unit u: [pre - lead, pre - lead + t), the first unit's lead before 0
    const int64_t at = g.s + p.lead;
    if (p.units <= NW * 64) {
        if (pre <= at && at < pre + t) {
            found[0] = tid;
            found[1] = pre;
        }
    } else {
        int64_t sum = 0;
        for (int c = 0; c < p.units && sum <= at; c += NW * 64) {
            const int u = c + tid;
            int64_t all;
            t = u < p.units ? unit_tiles<KIND>(p.a, u) : 0;
            t += t > 0 ? p.lead : 0;
            pre = sum + block_scan<NW>(t, s, all);
            if (pre <= at && at < pre + t) {
                found[0] = u;
                found[1] = pre;
            }
            sum += all;
        }
    }
    __syncthreads();
    g.u = __builtin_amdgcn_readfirstlane((int)found[0]);
    g.first = uniform(found[1]);
    return true;
}

// ------------------------------------------------------------- the tile ---
// A tile holds 32 positions in LDS as blocks of 1 KiB: block (rg, cg) has rows
// 8 rg .. 8 rg + 7 and 128 bytes (64 values) of each, the bytes that one load
// instruction of a wave brings, straight to LDS: nine column blocks a plane.
// In a row's 128 bytes the eight 16-byte chunks are XORed with tile_swz(row),
// so that the score reads (16 rows, one chunk) and the transposing reads (8
// rows, two chunks) both meet each of the LDS's 16 slots of 16 bytes once.
__device__ __forceinline__ int tile_swz(int row) { return row & 7; }

// A column's lanes l, l ^ 16, l ^ 32, l ^ 48 combined.
__device__ __forceinline__ float col_max(float v) {
    auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    v = fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1]));
    r = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    return fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1]));
}
__device__ __forceinline__ float col_sum(float v) {
    auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    v = __fadd_rn(__uint_as_float(r[0]), __uint_as_float(r[1]));
    r = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    return __fadd_rn(__uint_as_float(r[0]), __uint_as_float(r[1]));
}
// LDS by its 32-bit address.
template <class V> __device__ __forceinline__ V lds_read(uint32_t at) {
    return *(const __attribute__((address_space(3))) V *)at;
}
__device__ __forceinline__ pu32x4 tr_read(uint32_t x, uint32_t y) {
    typedef __attribute__((address_space(3))) pbf16x4 lds4;
    const pbf16x4 a = __builtin_amdgcn_ds_read_tr16_b64_v4bf16((lds4 *)x);
    const pbf16x4 b = __builtin_amdgcn_ds_read_tr16_b64_v4bf16((lds4 *)y);
    return __builtin_bit_cast(pu32x4, __builtin_shufflevector(a, b, 0, 1, 2, 3, 4, 5, 6, 7));
}

// A lane's first score read and first transposing read in a tile.  The others
// lie 1 KiB steps away, with chunk bits flipped: chunk 4 (ks & 1) + g in the
// score reads (^ 64 bytes), 2 (mt & 3) + .. in the transposing ones (^ 32, ^ 64).
struct LaneAddr {
    uint32_t k, v;
    uint32_t r, s;  // 8-bit pages: rotary keys and scales
};
template <int PLANES> __device__ __forceinline__ LaneAddr lane_addr(int l) {
    const int row = l & 15, g = l >> 4, j = l & 15, r = 4 * g + (j >> 2);
    return {(uint32_t)((row >> 3) * 9 * PLANES * 1024 + (row & 7) * 128 + ((g ^ tile_swz(row)) << 4)),
            (uint32_t)((r >> 3) * 9 * PLANES * 1024 + (r & 7) * 128 + ((((j & 3) >> 1) ^ tile_swz(r)) << 4) +
                       8 * (j & 1)), 0, 0};
}

// bf16 pages: queries and weights in bf16.
struct MfmaBf16 {
    static constexpr bool kCodes = false;
    static constexpr int kStages = 4, kRow = kPD * 2 * 1, kBlocks = 9 * 1, kTile = 4 * kBlocks * 1024, kValues = 0;
    __device__ __forceinline__ static LaneAddr addr(int l) { return lane_addr<1>(l); }
    template <class W> __device__ __forceinline__ static float unit(const W &) { return 1.0f; }
    static constexpr PlanCosts kCosts = kCostsBf16;
    static constexpr int kPlanes = 1, kWaves = kCosts.waves;
    static constexpr bool kBetween = false;  // copies between the products (the branches cost registers)
    static constexpr int kDepth = 4;
    static constexpr float kRise = 11.5f;  // log2 units a score may exceed the offset (8 nats)
    typedef __bf16 out_t;
    struct Query {
        pbf16x8 q[18];
    };
    // column l & 15, dims 32 ks + 8 (l >> 4) + [0, 8); the scale that the scores then need
    __device__ __forceinline__ static float load(Query &x, const void *qabs, const void *qrope, int64_t row, int g) {
        const __bf16 *qa = (const __bf16 *)qabs + row * kPL, *qr = (const __bf16 *)qrope + row * (kPD - kPL);
#pragma unroll
        for (int ks = 0; ks < 18; ks++) x.q[ks] = *(const pbf16x8 *)(ks < 16 ? qa + 32 * ks + 8 * g : qr + 32 * (ks - 16) + 8 * g);
        return 1.0f;
    }
    // waits for the loads here: left to their first use, the wait would stand
    // in the loop and hold up the copies too
    __device__ __forceinline__ static void arrive(Query &x, float) {
#pragma unroll
        for (int ks = 0; ks < 18; ks++) asm volatile("" : "+v"(x.q[ks]));
    }
    // both halves of the tile in turn, kDepth reads ahead of the products;
    // between(i) behind product i
    template <class B> __device__ __forceinline__ static void scores(const Query &x, uint32_t T, pf32x4 (&s)[2], B &&between) {
        s[0] = s[1] = pf32x4{0.0f, 0.0f, 0.0f, 0.0f};
        pbf16x8 k[36];
        auto read = [&](int i) {
            k[i] = lds_read<pbf16x8>((T ^ (((i >> 1) & 1) << 6)) + (i >> 2) * 1024 + (i & 1) * 18 * 1024);
        };
#pragma unroll
        for (int i = 0; i < kDepth; i++) read(i);
        __builtin_amdgcn_sched_barrier(0);
#pragma unroll
        for (int i = 0; i < 36; i++) {
            s[i & 1] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(k[i], x.q[i >> 1], s[i & 1], 0, 0, 0);
            if (i + kDepth < 36) read(i + kDepth);
            between(i);
            __builtin_amdgcn_sched_barrier(0);
        }
    }
    struct Weights {
        pbf16x8 p;
    };
    // Weights in bf16, as V is: the matrix cores take both operands in one type,
    // and two products a weight (its high and low part) would be half as many
    // again.  Each is off by 2^-8 at most; the sum is of the rounded ones that V
    // meets, so that what all values share is unchanged.  Contexts lie 1.8e-3 to
    // 2.0e-3 from 64 bits; their own rounding to bf16 alone makes 1.7e-3.
    __device__ __forceinline__ static float weigh(Weights &x, const float (&e)[8]) {
        float sum = 0.0f;
        const pbf16x2 one = {(__bf16)1.0f, (__bf16)1.0f};
#pragma unroll
        for (int i = 0; i < 8; i += 2) {
            const pbf16x2 v = {(__bf16)e[i], (__bf16)e[i + 1]};
            sum = __builtin_amdgcn_fdot2_f32_bf16(v, one, sum, false);
            x.p[i] = v[0];
            x.p[i + 1] = v[1];
        }
        return sum;
    }
    __device__ __forceinline__ static void context(const Weights &x, uint32_t T, pf32x4 (&o)[32]) {
        pu32x4 v[32];
        auto read = [&](int i) {
            const uint32_t b = (T ^ ((i & 3) << 5)) + (i >> 2) * 1024;
            v[i] = tr_read(b, b + 18 * 1024);
        };
#pragma unroll
        for (int i = 0; i < kDepth; i++) read(i);
        __builtin_amdgcn_sched_barrier(0);
#pragma unroll
        for (int i = 0; i < 32; i++) {
            o[i] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(pbf16x8, v[i]), x.p, o[i], 0, 0, 0);
            if (i + kDepth < 32) read(i + kDepth);
            __builtin_amdgcn_sched_barrier(0);
        }
    }
};

// f16x2 pages.  Every operand is a pair of f16, and a product is taken as
// hi*hi + lo*hi + hi*lo (lo*lo lies 2^-22 below).  Stored low parts are
// scaled by 2^11: the scores' sum with them is scaled back at its end, and in
// the context such a part meets the weight's high part times 2^-11, so that
// all three products add up in one accumulator.  Queries are scaled by a power
// of two to a maximum in [2^14, 2^15) and weights by 2^14 (at most 2^15), so
// that neither their low parts nor the scaled high parts fall out of f16's
// range where they matter.  Three products a score bound it: 33 rows of 128
// heads over up to 4099 positions (61 GFLOP in f16) take 96 us, floor 52.
struct MfmaF16x2 {
    static constexpr bool kCodes = false;
    static constexpr int kStages = 2, kRow = kPD * 2 * 2, kBlocks = 9 * 2, kTile = 4 * kBlocks * 1024, kValues = 0;
    __device__ __forceinline__ static LaneAddr addr(int l) { return lane_addr<2>(l); }
    template <class W> __device__ __forceinline__ static float unit(const W &) { return 1.0f; }
    static constexpr PlanCosts kCosts = kCostsF16x2;
    static constexpr int kPlanes = 2, kWaves = kCosts.waves;
    static constexpr bool kBetween = true;
    static constexpr int kDepth = 4;
    static constexpr float kRise = 1.0f;
    typedef float out_t;
    struct Query {
        pf16x8 h[18], l[18];
    };
    __device__ __forceinline__ static float load(Query &x, const void *qabs, const void *qrope, int64_t row, int g) {
        const float *qa = (const float *)qabs + row * kPL, *qr = (const float *)qrope + row * (kPD - kPL);
        float top = 0.0f;
#pragma unroll
        for (int ks = 0; ks < 18; ks++)
#pragma unroll
            for (int i = 0; i < 8; i++) top = fmaxf(top, fabsf((ks < 16 ? qa + 32 * ks : qr + 32 * (ks - 16))[8 * g + i]));
        top = col_max(top);
        // 2^e <= top < 2^(e + 1)
        const int e = (int)(__float_as_uint(top) >> 23) - 127;
        const int up = top > 0.0f && top < INFINITY ? (14 - e < 120 ? 14 - e : 120) : 0;
#pragma unroll
        for (int ks = 0; ks < 18; ks++)
#pragma unroll
            for (int i = 0; i < 8; i++) {
                const float v = ldexpf((ks < 16 ? qa + 32 * ks : qr + 32 * (ks - 16))[8 * g + i], up);
                const _Float16 h = (_Float16)v;
                x.h[ks][i] = h;
                x.l[ks][i] = (_Float16)__fsub_rn(v, (float)h);
            }
        return ldexpf(1.0f, -up);
    }
    __device__ __forceinline__ static void arrive(Query &, float) {}  // converted: they are there
    // three sums a half tile, so that no product waits for the one before it
    template <class B> __device__ __forceinline__ static void scores(const Query &x, uint32_t T, pf32x4 (&s)[2], B &&between) {
        s[0] = s[1] = pf32x4{0.0f, 0.0f, 0.0f, 0.0f};
        pf32x4 t[2] = {s[0], s[0]}, v[2] = {s[0], s[0]};
        pf16x8 k[36], d[36];  // high and low parts
        auto read = [&](int i) {
            const uint32_t b = (T ^ (((i >> 1) & 1) << 6)) + (i >> 2) * 1024 + (i & 1) * 36 * 1024;
            k[i] = lds_read<pf16x8>(b);
            d[i] = lds_read<pf16x8>(b + 9 * 1024);
        };
#pragma unroll
        for (int i = 0; i < kDepth; i++) read(i);
        __builtin_amdgcn_sched_barrier(0);
#pragma unroll
        for (int i = 0; i < 36; i += 2) {
#pragma unroll
            for (int e = 0; e < 2; e++) s[e] = __builtin_amdgcn_mfma_f32_16x16x32_f16(k[i + e], x.h[i >> 1], s[e], 0, 0, 0);
#pragma unroll
            for (int e = 0; e < 2; e++) t[e] = __builtin_amdgcn_mfma_f32_16x16x32_f16(k[i + e], x.l[i >> 1], t[e], 0, 0, 0);
#pragma unroll
            for (int e = 0; e < 2; e++) v[e] = __builtin_amdgcn_mfma_f32_16x16x32_f16(d[i + e], x.h[i >> 1], v[e], 0, 0, 0);
#pragma unroll
            for (int e = 0; e < 2; e++)
                if (i + e + kDepth < 36) read(i + e + kDepth);
            between(i);
            between(i + 1);
            __builtin_amdgcn_sched_barrier(0);
        }
#pragma unroll
        for (int e = 0; e < 2; e++)
#pragma unroll
            for (int i = 0; i < 4; i++)
                s[e][i] = __fadd_rn(s[e][i], __builtin_fmaf(v[e][i], 1.0f / kF16x2Step, t[e][i]));
    }
    struct Weights {
        pf16x8 h, l, d;
    };
    __device__ __forceinline__ static float weigh(Weights &x, const float (&e)[8]) {
        float sum = 0.0f;
#pragma unroll
        for (int i = 0; i < 8; i++) {
            const float v = __fmul_rn(e[i], 16384.0f);
            sum = __fadd_rn(sum, v);
            x.h[i] = (_Float16)v;
            x.l[i] = (_Float16)__fsub_rn(v, (float)x.h[i]);
        }
        x.d = x.h * (_Float16)(1.0f / kF16x2Step);
        return sum;
    }
    __device__ __forceinline__ static void context(const Weights &x, uint32_t T, pf32x4 (&o)[32]) {
        pu32x4 h[32], d[32];
        auto read = [&](int i) {
            const uint32_t b = (T ^ ((i & 3) << 5)) + (i >> 2) * 1024;
            h[i] = tr_read(b, b + 36 * 1024);
            d[i] = tr_read(b + 9 * 1024, b + 45 * 1024);
        };
#pragma unroll
        for (int i = 0; i < kDepth; i++) read(i);
        __builtin_amdgcn_sched_barrier(0);
#pragma unroll
        for (int i = 0; i < 32; i += 2) {
#pragma unroll
            for (int e = 0; e < 2; e++) o[i + e] = __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(pf16x8, h[i + e]), x.l, o[i + e], 0, 0, 0);
#pragma unroll
            for (int e = 0; e < 2; e++) o[i + e] = __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(pf16x8, d[i + e]), x.d, o[i + e], 0, 0, 0);
#pragma unroll
            for (int e = 0; e < 2; e++) o[i + e] = __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(pf16x8, h[i + e]), x.h, o[i + e], 0, 0, 0);
#pragma unroll
            for (int e = 0; e < 2; e++)
                if (i + e + kDepth < 32) read(i + e + kDepth);
            __builtin_amdgcn_sched_barrier(0);
        }
    }
};

// 8-bit pages.  Scores are products of integers: a query's parts, each scaled to
// 32512 at its largest, are split in two digits of 8 bits, x = 256 hi + lo, and
// meet the codes as they lie in LDS on the int8 matrix cores, two products of
// twice the bf16 rate for one; the sums are exact in 32 bits, and a query is off
// by 2^-16 of its part's largest at most.
//   s = (q_lat . c_lat) step_lat scale_t,lat + (q_rope . c_rope) step_rope scale_t,rope
// Values: codes as f16, which holds them exactly, converted once for all waves
// a tile ahead of their use; a weight meets its position's scale before it is
// rounded to f16, w = e^(s - m) scale_t,lat.  Scales may be of any size, so a
// column's weights are taken times a power of two g that puts the largest so far
// at 2^10 to 2^15: one loses bits from 2^-24 of the largest down.  g moves, as the
// offset m does, only where a weight would pass 2^15.
typedef int pi32x4 __attribute__((ext_vector_type(4)));
typedef _Float16 pf16x2 __attribute__((ext_vector_type(2)));
struct MfmaI8 {
    static constexpr bool kCodes = true;
    // a tile: 32 x 512 latent codes in 16 blocks as above, 32 x 64 rotary ones, 32 pairs of scales
    static constexpr int kStages = 5, kRow = kPD, kBlocks = 4, kRope = 16 * 1024, kScales = 18 * 1024;
    static constexpr int kTile = kScales + 256, kValues = 2 * 32 * 1024;  // two tiles' values
    static constexpr PlanCosts kCosts = kCostsI8;
    static constexpr int kPlanes = 1, kWaves = kCosts.waves;
    static constexpr bool kBetween = false;
    static constexpr int kDepth = 4, kAhead = 2;
    static constexpr float kRise = 11.5f;
    typedef __bf16 out_t;
    // The rotary codes of row r, 64 bytes: chunks of 16 XORed with (r >> 2) & 3, so
    // that 16 rows' chunks meet the LDS's 16 slots once.
    __device__ __forceinline__ static uint32_t rope_off(int t, int rb) {
        const int row = (t >> 2) & 7;
        return row * kPD + (((t & 3) ^ (((8 * rb + row) >> 2) & 3)) << 4);
    }
    __device__ __forceinline__ static LaneAddr addr(int l) {
        const int row = l & 15, g = l >> 4, j = l & 15, r = 4 * g + (j >> 2);
        return {(uint32_t)((row >> 3) * kBlocks * 1024 + (row & 7) * 128 + ((g ^ tile_swz(row)) << 4)),
                (uint32_t)((r >> 3) * 8 * 1024 + (r & 7) * 128 + ((((j & 3) >> 1) ^ tile_swz(r)) << 4) + 8 * (j & 1)),
                (uint32_t)(kRope + row * 64 + ((g ^ (row >> 2)) << 4)), (uint32_t)(kScales + 32 * g)};
    }
    // Of a power of two.
    __device__ __forceinline__ static float inverse(float g) { return __uint_as_float((254u << 23) - __float_as_uint(g)); }
    // 16 dims of a step of 64 in two register quads: bf16, then high and low digits
    struct Query {
        pu32x4 w[18];
        float lat, rope;  // a digit's worth in each part, times the scores' scale
    };
    __device__ __forceinline__ static float load(Query &x, const void *qabs, const void *qrope, int64_t row, int g) {
        const __bf16 *qa = (const __bf16 *)qabs + row * kPL, *qr = (const __bf16 *)qrope + row * (kPD - kPL);
#pragma unroll
        for (int i = 0; i < 18; i++) x.w[i] = *(const pu32x4 *)((i < 16 ? qa + 32 * (i & ~1) : qr) + 16 * g + 8 * (i & 1));
        return 1.0f;
    }
    // Part [I0, I1) of the words to digits.
    template <int I0, int I1> __device__ __forceinline__ static float digits(Query &x) {
        typedef uint16_t u16x2 __attribute__((ext_vector_type(2)));
        u16x2 most = {0, 0};
#pragma unroll
        for (int i = I0; i < I1; i++)
#pragma unroll
            for (int k = 0; k < 4; k++)
                most = __builtin_elementwise_max(most, __builtin_bit_cast(u16x2, x.w[i][k] & 0x7fff7fffu));
        // bits of |q|: NaN lies above infinity
        uint32_t top = (uint32_t)(most[0] > most[1] ? most[0] : most[1]) << 16;
        auto r = __builtin_amdgcn_permlane32_swap(top, top, false, false);
        top = r[0] > r[1] ? r[0] : r[1];
        r = __builtin_amdgcn_permlane16_swap(top, top, false, false);
        top = r[0] > r[1] ? r[0] : r[1];
        const bool finite = top < 0x7f800000u;
        float m = __uint_as_float(top), down = 1.0f;
        // (the quotient stays in range: tiny queries are taken times 2^64, which changes no bit of them)
        const bool tiny = top > 0 && top < 0x10000000u;
        if (__any(tiny)) {
            const float up = tiny ? 0x1p64f : 1.0f;
            m *= up;
            down = tiny ? 0x1p-64f : 1.0f;
#pragma unroll
            for (int i = I0; i < I1; i++)
#pragma unroll
                for (int k = 0; k < 4; k++) {
                    const uint32_t v = x.w[i][k];
                    const uint32_t lo = __float_as_uint(__fmul_rn(__uint_as_float(v << 16), up));
                    const uint32_t hi = __float_as_uint(__fmul_rn(__uint_as_float(v & 0xffff0000u), up));
                    x.w[i][k] = (lo >> 16) | (hi & 0xffff0000u);
                }
        }
        const float f = finite && top > 0 ? 32512.0f / m : 0.0f;
        // 1.5 * 2^23 + 128 in front: the sum's low 16 bits are x + 128 to the nearest x
        constexpr float kFront = 12582912.0f + 128.0f;
#pragma unroll
        for (int i = I0; i < I1; i += 2) {
            uint32_t d[2][4];
#pragma unroll
            for (int h = 0; h < 2; h++)
#pragma unroll
                for (int k = 0; k < 4; k += 2) {
                    uint32_t two[2];
#pragma unroll
                    for (int e = 0; e < 2; e++) {
                        const uint32_t v = x.w[i + h][k + e];
                        const uint32_t a = __float_as_uint(__builtin_fmaf(__uint_as_float(v << 16), f, kFront));
                        const uint32_t b = __float_as_uint(__builtin_fmaf(__uint_as_float(v & 0xffff0000u), f, kFront));
                        two[e] = __builtin_amdgcn_perm(b, a, 0x05040100u);
                    }
                    d[0][2 * h + k / 2] = __builtin_amdgcn_perm(two[1], two[0], 0x07050301u);
                    d[1][2 * h + k / 2] = __builtin_amdgcn_perm(two[1], two[0], 0x06040200u) ^ 0x80808080u;
                }
#pragma unroll
            for (int h = 0; h < 2; h++) x.w[i + h] = pu32x4{d[h][0], d[h][1], d[h][2], d[h][3]};
        }
        return finite ? __fmul_rn(__fmul_rn(m, 1.0f / 32512.0f), down) : __uint_as_float(0x7fc00000u);
    }
    __device__ __forceinline__ static void arrive(Query &x, float c) {
        x.lat = __fmul_rn(digits<0, 16>(x), c);
        x.rope = __fmul_rn(digits<16, 18>(x), c);
#pragma unroll
        for (int i = 0; i < 18; i++) asm volatile("" : "+v"(x.w[i]));
    }
    template <class W> __device__ __forceinline__ static float unit(const W &w) { return inverse(w.g); }
    // The tile's halves one after the other (their sums together would not fit
    // the registers, and a reload would wait for the copies), the rotary part first.
    __device__ __forceinline__ static void scores(const Query &x, uint32_t T, const LaneAddr &ad, float (&t)[8]) {
        const pi32x4 zero = {0, 0, 0, 0};
#pragma unroll
        for (int half = 0; half < 2; half++) {
            pi32x4 h = zero, d = zero, rh, rd, k[9];
            auto read = [&](int i) {
                if (i == 0) k[i] = lds_read<pi32x4>(T + ad.r + half * 1024);
                else k[i] = lds_read<pi32x4>(((T + ad.k) ^ (((i - 1) & 1) << 6)) + ((i - 1) >> 1) * 1024 + half * 2 * kBlocks * 1024);
            };
#pragma unroll
            for (int i = 0; i < kAhead; i++) read(i);
            __builtin_amdgcn_sched_barrier(0);
#pragma unroll
            for (int i = 0; i < 9; i++) {
                const int q = i == 0 ? 16 : 2 * (i - 1);
                const pi32x4 qh = __builtin_bit_cast(pi32x4, x.w[q]), qd = __builtin_bit_cast(pi32x4, x.w[q + 1]);
                if (i == 0) {
                    rh = __builtin_amdgcn_mfma_i32_16x16x64_i8(k[i], qh, zero, 0, 0, 0);
                    rd = __builtin_amdgcn_mfma_i32_16x16x64_i8(k[i], qd, zero, 0, 0, 0);
                } else {
                    h = __builtin_amdgcn_mfma_i32_16x16x64_i8(k[i], qh, h, 0, 0, 0);
                    d = __builtin_amdgcn_mfma_i32_16x16x64_i8(k[i], qd, d, 0, 0, 0);
                }
                if (i + kAhead < 9) read(i + kAhead);
                if (i == 2)
#pragma unroll
                    for (int e = 0; e < 4; e++) t[4 * half + e] = __fmul_rn((float)((rh[e] << 8) + rd[e]), x.rope);
                __builtin_amdgcn_sched_barrier(0);
            }
            // (a tile's scales: latent and rotary by turns)
            pf32x4 s[2];
#pragma unroll
            for (int i = 0; i < 2; i++) s[i] = lds_read<pf32x4>(T + ad.s + half * 128 + i * 16);
#pragma unroll
            for (int e = 0; e < 4; e++) {
                const float lat = __fmul_rn((float)((h[e] << 8) + d[e]), x.lat);
                t[4 * half + e] = __builtin_fmaf(lat, s[e >> 1][2 * (e & 1)], __fmul_rn(t[4 * half + e], s[e >> 1][2 * (e & 1) + 1]));
            }
            __builtin_amdgcn_sched_barrier(0);
        }
    }
    // The latent scales of a lane's positions.
    __device__ __forceinline__ static void scales(uint32_t T, const LaneAddr &ad, float (&s)[8]) {
#pragma unroll
        for (int i = 0; i < 4; i++) {
            const pf32x4 v = lds_read<pf32x4>(T + ad.s + (i >> 1) * 128 + (i & 1) * 16);
            s[2 * i] = v[0];
            s[2 * i + 1] = v[2];
        }
    }
    __device__ __forceinline__ static void context(const pf16x8 &p, uint32_t T, pf32x4 (&o)[32]) {
        pu32x4 v[32];
        auto read = [&](int i) {
            const uint32_t b = (T ^ ((i & 3) << 5)) + (i >> 2) * 1024;
            v[i] = tr_read(b, b + 16 * 1024);
        };
#pragma unroll
        for (int i = 0; i < kDepth; i++) read(i);
        __builtin_amdgcn_sched_barrier(0);
#pragma unroll
        for (int i = 0; i < 32; i++) {
            o[i] = __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(pf16x8, v[i]), p, o[i], 0, 0, 0);
            if (i + kDepth < 32) read(i + kDepth);
            __builtin_amdgcn_sched_barrier(0);
        }
    }
};

// A tile's latent codes to f16 values, in the blocks of 8 rows and 64 values
// that the transposing reads take: eight waves, two of the 16 blocks of codes
// each.  A lane's 16 codes become two chunks; lanes of a row's two halves write
// theirs in opposite order, so that no two meet in a slot.
//   f16(code) = (1024 + (code + 128)) - 1152, each step exact.
template <int PART> __device__ __forceinline__ void convert_block(const pu32x4 &c, uint32_t to, int block, int l) {
    const int row = l >> 3, in = (l & 7) ^ tile_swz(row), e = PART ^ (in >> 2);
    const pf16x2 off = {(_Float16)-1152.0f, (_Float16)-1152.0f};
    pu32x4 v;
#pragma unroll
    for (int k = 0; k < 2; k++) {
        const uint32_t u = (e ? c[2 + k] : c[k]) ^ 0x80808080u;
        v[2 * k] = __builtin_bit_cast(uint32_t, __builtin_bit_cast(pf16x2, __builtin_amdgcn_perm(0x64646464u, u, 0x04010400u)) + off);
        v[2 * k + 1] = __builtin_bit_cast(uint32_t, __builtin_bit_cast(pf16x2, __builtin_amdgcn_perm(0x64646464u, u, 0x04030402u)) + off);
    }
    const uint32_t at = to + ((block >> 2) * 8 + 2 * (block & 3) + (in >> 2)) * 1024 + row * 128 + (((2 * (in & 3) + e) ^ tile_swz(row)) << 4);
    *(__attribute__((address_space(3))) pu32x4 *)at = v;
}
// The lane, as if not known yet: what is worked out of it is worked out anew for
// each tile, since the products need the registers that it would be kept in.
__device__ __forceinline__ int lane_anew() {
    int l = threadIdx.x & 63;
    asm volatile("" : "+v"(l));
    return l;
}
__device__ __forceinline__ pu32x4 codes_of(uint32_t from, int block, int l) { return lds_read<pu32x4>(from + block * 1024 + l * 16); }
__device__ __forceinline__ void convert_tile(uint32_t from, uint32_t to, int w) {
    const int l = lane_anew();
    const pu32x4 a = codes_of(from, w, l), b = codes_of(from, w + 8, l);
    convert_block<0>(a, to, w, l);
    convert_block<1>(a, to, w, l);
    convert_block<0>(b, to, w + 8, l);
    convert_block<1>(b, to, w + 8, l);
}

// One wave's columns: 16 heads of one query row, the whole latent width.
template <class F> struct Wave {
    typename F::Query q;
    pf32x4 o[32];  // context^T: dim 16 mt + 4 (l >> 4) + i, column l & 15
    float m, l;    // softmax offset (log2 units) and sum
    float top, g;  // 8-bit pages: the largest weight times its position's scale (of this lane's), and a power
                   // of two, the same for a column, that such products are in the context's sum by
};

// One tile: S^T = K Q^T (positions x columns), the online softmax per column,
// O^T += V^T P.  A lane of S holds positions 4 g + i and 16 + 4 g + i of one
// column (g = lane >> 4); the second product takes its positions in that very
// order (V's rows are read to match), so P goes from one product into the
// other without leaving the lane.  The offset m moves only where a score
// exceeds it by more than kRise.
// seen: the tile's visible positions.  A hidden position's score is replaced,
// whatever it is; what V holds there must be finite (tile_clear).
template <class F, class B>
__device__ __forceinline__ void tile_step(Wave<F> &w, const LaneAddr &ad, uint32_t T, uint32_t seen, float c, int g, B &&between) {
    pf32x4 s[2];
    F::scores(w.q, T + ad.k, s, between);
    const uint32_t mine = seen >> (4 * g);
    float t[8];
#pragma unroll
    for (int i = 0; i < 8; i++) t[i] = __fmul_rn(s[i >> 2][i & 3], c);
    if (seen != ~0u)
#pragma unroll
        for (int i = 0; i < 8; i++)
            if (!((mine >> ((i >> 2) * 16 + (i & 3))) & 1)) t[i] = -INFINITY;
    float top = fmaxf(fmaxf(fmaxf(t[0], t[1]), fmaxf(t[2], t[3])), fmaxf(fmaxf(t[4], t[5]), fmaxf(t[6], t[7])));
    top = col_max(top);
    const bool jump = top > __fadd_rn(w.m, F::kRise);
    if (__any(jump)) {
        const float mn = jump ? top : w.m, f = __builtin_amdgcn_exp2f(w.m - mn);
        // (a column's first scores meet zeros)
        if (__any(jump && w.m > kLow))
#pragma unroll
            for (int mt = 0; mt < 32; mt++) w.o[mt] *= f;
        w.m = mn;
        w.l *= f;
    }
#pragma unroll
    for (int i = 0; i < 8; i++) t[i] = __builtin_amdgcn_exp2f(t[i] - w.m);
    typename F::Weights p;
    w.l = __fadd_rn(w.l, F::weigh(p, t));
    F::context(p, T + ad.v, w.o);
}

// The same with 8-bit pages: T's codes and scales, V's values.
__device__ __forceinline__ void tile_codes(Wave<MfmaI8> &w, uint32_t T, uint32_t V, uint32_t seen) {
    typedef MfmaI8 F;
    const int l = lane_anew(), g = l >> 4;
    const LaneAddr ad = F::addr(l);
    float t[8];
    F::scores(w.q, T, ad, t);
    const uint32_t mine = seen >> (4 * g);
    if (seen != ~0u)
#pragma unroll
        for (int i = 0; i < 8; i++)
            if (!((mine >> ((i >> 2) * 16 + (i & 3))) & 1)) t[i] = -INFINITY;
    auto most = [](const float (&v)[8]) {
        return fmaxf(fmaxf(fmaxf(v[0], v[1]), fmaxf(v[2], v[3])), fmaxf(fmaxf(v[4], v[5]), fmaxf(v[6], v[7])));
    };
    float f = 1.0f;
    float top = most(t);
    if (__any(top > __fadd_rn(w.m, F::kRise))) {
        top = col_max(top);
        const float mn = top > __fadd_rn(w.m, F::kRise) ? top : w.m;
        f = __builtin_amdgcn_exp2f(w.m - mn);
        w.m = mn;
        w.l *= f;
        w.top *= f;
    }
    float e[8];
#pragma unroll
    for (int i = 0; i < 8; i++) e[i] = __builtin_amdgcn_exp2f(t[i] - w.m);
    __builtin_amdgcn_sched_barrier(0);
    float s[8];
    F::scales(T, ad, s);
    // (a hidden position's scale is any)
    if (seen != ~0u)
#pragma unroll
        for (int i = 0; i < 8; i++)
            if (!((mine >> ((i >> 2) * 16 + (i & 3))) & 1)) s[i] = 0.0f;
    w.l = __fadd_rn(w.l, __fadd_rn(__fadd_rn(__fadd_rn(e[0], e[1]), __fadd_rn(e[2], e[3])), __fadd_rn(__fadd_rn(e[4], e[5]), __fadd_rn(e[6], e[7]))));
#pragma unroll
    for (int i = 0; i < 8; i++) e[i] = __fmul_rn(e[i], s[i]);
    w.top = fmaxf(w.top, most(e));
    const bool moved = __any(f != 1.0f);
    if (moved || __any(__fmul_rn(w.top, w.g) > 32768.0f)) {
        // g for the column's largest, which its lanes share from here on
        w.top = col_max(w.top);
        const int up = (int)(__float_as_uint(w.top) >> 23) - 127;
        const float gn = w.top > 0.0f ? __uint_as_float((uint32_t)(127 + (10 - up < 120 ? 10 - up : 120)) << 23) : w.g;
        const float by = __fmul_rn(__fmul_rn(f, gn), F::inverse(w.g));
        w.g = gn;
#pragma unroll
        for (int mt = 0; mt < 32; mt++) w.o[mt] *= by;
    }
    pf16x8 p;
#pragma unroll
    for (int i = 0; i < 8; i++) p[i] = (_Float16)__fmul_rn(e[i], w.g);
    F::context(p, V + ad.v, w.o);
}

// The latent values of a tile's rows: hidden rows are cleared before V meets
// them (0 * NaN is NaN), 64 chunks of 16 bytes a plane.
template <class F> __device__ __forceinline__ uint8_t *tile_chunk(uint8_t *T, int row, int c) {
    return T + ((row >> 3) * 9 * F::kPlanes + (c >> 6) * 9 + ((c & 63) >> 3)) * 1024 + (row & 7) * 128 +
           (((c & 7) ^ tile_swz(row)) << 4);
}
template <class F> __device__ __forceinline__ void tile_clear(uint8_t *T, uint32_t rows) {
#pragma unroll 1
    for (int i = threadIdx.x; i < 32 * 64 * F::kPlanes; i += F::kWaves * 64)
        if ((rows >> (i & 31)) & 1) *(pu32x4 *)tile_chunk<F>(T, i & 31, i >> 5) = pu32x4{0, 0, 0, 0};
}
// Whether one of the rows holds a value that is not finite (this thread's share).
template <class F> __device__ __forceinline__ bool tile_odd(uint8_t *T, uint32_t rows) {
    const uint32_t ones = F::kPlanes == 1 ? 0x7f80u : 0x7c00u;  // the exponent's bits
    bool odd = false;
#pragma unroll 1
    for (int i = threadIdx.x; i < 32 * 64 * F::kPlanes; i += F::kWaves * 64)
        if ((rows >> (i & 31)) & 1) {
            const pu32x4 v = *(const pu32x4 *)tile_chunk<F>(T, i & 31, i >> 5);
#pragma unroll
            for (int k = 0; k < 4; k++)
                odd |= (v[k] & ones) == ones || ((v[k] >> 16) & ones) == ones;
        }
    return odd;
}

// What a wave needs to look positions up: unit u's sequence and row.
struct Lookup {
    const_i32 *table, *sel;  // the sequence's row of the table, the row's pages
    int32_t n, top_k, shift;
    int32_t window, sinks;  // with a window
    NearCut cut;
};
// The first position of the unit's tile x.
template <int KIND> __device__ __forceinline__ int32_t tile_at(const Lookup &k, int32_t x) {
    return (KIND == kNear && x >= k.cut.ts ? x + k.cut.skip : x) * kPT;
}
// The page of the sequence that holds the unit's position v0; one that it
// does have, where there is none or it lies behind the end.
template <int KIND> __device__ __forceinline__ int32_t page_of(const Lookup &k, int32_t v0) {
    if (KIND == kListed) {
        const int32_t i = v0 >> k.shift;
        return i < k.top_k ? k.sel[i] : 0;
    }
    // (eight positions that no row sees: their page need not be named)
    if (KIND == kNear && v0 >= k.sinks && v0 + 8 <= k.cut.start) return -1;
    return (v0 < k.n ? v0 : k.n - 1) >> k.shift;
}
template <int KIND> __device__ __forceinline__ int32_t page_entry(const Lookup &k, int32_t page) {
    // the pool's first page stands in for one that is not listed or not seen: the
    // table need not name any but the listed ones
    const bool none = KIND == kNear ? page < 0 : KIND == kListed && (page < 0 || ((int64_t)page << k.shift) >= k.n);
    const int32_t entry = k.table[none ? 0 : page];
    return none ? 0 : entry;
}
__device__ __forceinline__ uint32_t low_bits(int32_t c) { return c >= 32 ? ~0u : c <= 0 ? 0u : (1u << c) - 1u; }
// The visible positions of the tile at v0 for a row that sees n.
template <int KIND>
__device__ __forceinline__ uint32_t visible(const Lookup &k, int32_t v0, int32_t n) {
    if (KIND == kAll) return low_bits(n - v0);
    if (KIND == kNear) {
        // the window's positions from `lo` on
        const int32_t lo = n > k.window ? n - k.window - v0 : 0;
        const uint32_t near = lo <= 0 ? ~0u : lo >= 32 ? 0u : ~0u << lo;
        return low_bits(n - v0) & (near | low_bits(k.sinks - v0));
    }
    const int per = k.shift >= 5 ? 32 : 1 << k.shift;
    uint32_t m = 0;
    for (int i = 0; i < 32; i += per) {
        const int32_t v = v0 + i, at = v >> k.shift;
        const int32_t page = at < k.top_k ? k.sel[at] : -1;
        const int64_t c = page < 0 ? 0 : n - (((int64_t)page << k.shift) + (v & ((1 << k.shift) - 1)));
        const uint32_t ones = c >= per ? (per == 32 ? ~0u : (1u << per) - 1u) : c <= 0 ? 0u : (1u << c) - 1u;
        m |= ones << i;
    }
    return m;
}

// What some row of a unit sees of tile x, and what each of the M rows does.
// (Windows follow on one another: what some row sees is one run, too.)
template <int KIND> __device__ __forceinline__ uint32_t some_see(const Lookup &k, int32_t x, int32_t len) {
    const int32_t v0 = tile_at<KIND>(k, x), lo = KIND == kNear ? k.cut.start - v0 : 0;
    return low_bits(len - v0) & (lo <= 0 ? ~0u : (lo >= 32 ? 0u : ~0u << lo) | low_bits(k.sinks - v0));
}
template <int KIND> __device__ __forceinline__ uint32_t all_see(const Lookup &k, int32_t x, int32_t len, int32_t M) {
    const int32_t v0 = tile_at<KIND>(k, x);
    const uint32_t last = KIND == kNear ? visible<KIND>(k, v0, len) : ~0u;
    return last & low_bits(len - M + 1 - v0);
}

// Column block I of a lane's row, 128 bytes apart there and 1 KiB apart in
// LDS, straight to LDS.  An instruction's offset counts on both sides, so lds
// steps by the rest.  Written out, since the compiler would have every later
// LDS read wait for every copy under way: the kernel waits itself.  Nothing
// is loaded into a register, and the address is read when the instruction
// issues.  (m0 is reserved: the compiler takes no clobber of it and sets it anew
// where it needs it, which it does nowhere in these kernels.)
template <int I> __device__ __forceinline__ void copy_block(uint32_t off, const uint8_t *src, uint32_t lds) {
    asm volatile("s_mov_b32 m0, %2\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %0, %1 offset:%3"
                 :
                 : "v"(off), "s"(src), "s"(lds + I * (1024 - 128)), "n"(I * 128)
                 : "memory");
}
template <int I, int N> __device__ __forceinline__ void copy_blocks(uint32_t off, const uint8_t *src, uint32_t lds) {
    if constexpr (I < N) {
        copy_block<I>(off, src, lds);
        copy_blocks<I + 1, N>(off, src, lds);
    }
}
// Block i of N, i known where this is expanded.
template <int I, int N> __device__ __forceinline__ void copy_nth(int i, uint32_t off, const uint8_t *src, uint32_t lds) {
    if constexpr (I < N) {
        if (i == I) copy_block<I>(off, src, lds);
        else copy_nth<I + 1, N>(i, off, src, lds);
    }
}

// s_waitcnt of at most n vector memory operations under way (a tile's copies
// are 5 of one half of the waves and 4 of the other; waiting for the fewer
// suits both)
constexpr int kWaitVm0 = 0x0f70, kWaitVm4 = 0x0f74, kWaitVm8 = 0x0f78;
// The same for tiles of codes, three copies each, with all LDS operations done
// (the values that this wave has converted).
constexpr int kWaitAll0 = 0x0070, kWaitAll3 = 0x0073, kWaitAll6 = 0x0076, kWaitAll9 = 0x0079;
// All but the copies of the last `ahead` tiles have landed, for every wave.
template <class F> __device__ __forceinline__ void wait_tiles(int32_t ahead, int32_t most) {
    __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
    ahead = ahead < most ? ahead : most;
    if constexpr (F::kCodes) {
        if (ahead >= 3) __builtin_amdgcn_s_waitcnt(kWaitAll9);
        else if (ahead == 2) __builtin_amdgcn_s_waitcnt(kWaitAll6);
        else if (ahead == 1) __builtin_amdgcn_s_waitcnt(kWaitAll3);
        else __builtin_amdgcn_s_waitcnt(kWaitAll0);
    } else {
        if (ahead >= 2) __builtin_amdgcn_s_waitcnt(kWaitVm8);
        else if (ahead == 1) __builtin_amdgcn_s_waitcnt(kWaitVm4);
        else __builtin_amdgcn_s_waitcnt(kWaitVm0);
    }
    __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
    __builtin_amdgcn_s_barrier();
    __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
}

// The part of a range that lies in one unit.
struct Seg {
    int32_t u, j, h0, b0, b1, tiles, len, n;
    int64_t first, row;
    Lookup lk;
};
// Goes over a range's parts.
template <int KIND> struct Walk {
    int32_t u;
    int64_t first, at;
    __device__ __forceinline__ bool next(const PagedMfmaArgs &p, const Range &rg, int gr, Seg &q) {
        const PagedArgs &a = p.a;
        int32_t tiles = 0;
        while (at < rg.e && !(tiles = __builtin_amdgcn_readfirstlane(unit_tiles<KIND>(a, u)))) u++;
        q.b0 = at > first ? (int32_t)(at - first) : 0;
        q.b1 = rg.e - first < tiles ? (int32_t)(rg.e - first) : tiles;
        if (q.b0 >= q.b1) return false;
        constexpr bool SPARSE = KIND == kListed;
        const int per_row = (a.H + kCols - 1) / kCols, b = SPARSE ? u / a.M : u;
        q.u = u;
        q.j = SPARSE ? u - b * a.M : gr / per_row;
        q.h0 = (SPARSE ? gr : gr % per_row) * kCols;
        q.tiles = tiles;
        q.len = __builtin_amdgcn_readfirstlane(paged_len(a, b));
        q.n = q.len - a.M + q.j + 1;
        q.first = first;
        q.row = ((int64_t)b * a.M + q.j) * a.H;
        q.lk.table = (const_i32 *)(a.table + (int64_t)b * a.stride);
        q.lk.sel = SPARSE ? (const_i32 *)(a.sel + (int64_t)u * a.top_k) : nullptr;
        q.lk.n = SPARSE ? q.n : q.len;
        q.lk.top_k = a.top_k;
        q.lk.shift = a.shift;
        if (KIND == kNear) {
            q.lk.window = a.window;
            q.lk.sinks = a.sinks;
            q.lk.cut = near_cut(a, q.len);
        }
        first += tiles + p.lead;
        at = first;
        u++;
        return true;
    }
};

// A workgroup is F::kWaves waves, each with a column group of its own, over
// the same tiles.  Four (f16x2: two) tiles fit the LDS: the products of one
// run while the next three (one) are on their way.  A table entry is read a
// tile before its copy, and the copies issue between the products.
template <class F, int KIND>
__global__ __launch_bounds__(F::kWaves * 64, F::kWaves / 4) void k_paged_mfma(PagedMfmaArgs p) {
    constexpr bool SPARSE = KIND == kListed, CODES = F::kCodes;
    constexpr int NW = F::kWaves, PL = F::kPlanes, STAGES = F::kStages, ROW = F::kRow, TILE = F::kTile;
    __shared__ __attribute__((aligned(1024))) uint8_t stage[STAGES * TILE + F::kValues];
    __shared__ int s_odd;
    const PagedArgs &a = p.a;
    const int tid = threadIdx.x, w = __builtin_amdgcn_readfirstlane(tid >> 6), l = tid & 63, g = l >> 4, col = l & 15;
    const int share = gridDim.x >> 3;
    const int id = (blockIdx.x & 7) * share + (blockIdx.x >> 3);  // neighbours on one XCD
    const int r = id / p.chunks, chunk = id - r * p.chunks;
    // units without positions: zeros
    const int64_t vec = (int64_t)(SPARSE ? 1 : a.M) * a.H * kPL * (int)sizeof(typename F::out_t) / 16;
    for (int u = id; u < p.units; u += gridDim.x)
        if (unit_tiles<KIND>(a, u) == 0)
            for (int64_t i = tid; i < vec; i += NW * 64) ((pu32x4 *)a.out)[u * vec + i] = pu32x4{0, 0, 0, 0};
    Range rg;
    if (r >= p.most || !find_range<KIND, NW>(p, r, p.most > 1 && r == 0 && chunk == 0, rg)) return;
    const int grp = chunk * p.per + w;
    const bool active = w < p.per && grp < p.groups;
    const int gr = active ? grp : 0;
    const LaneAddr ad = F::addr(l);
    const uint32_t stage0 = (uint32_t)(uintptr_t)(lds_u8 *)stage;
    // copies: wave w brings row block w & 3 and, where two waves share it, half of its column blocks
    // (of codes: two latent blocks each, then the first four the rotary keys, the others the scales)
    const int rb = w & 3, c0 = NW == 8 && w >= 4 ? (CODES ? 2 : 5) : 0;
    constexpr int COPIES = CODES ? 2 : NW == 4 ? 9 * PL : 4;  // and a fifth (of codes: third) of waves 0 to 3
    Wave<F> wv;
    bool bad = false;
    // the next copy: its table entry, and where it goes
    int32_t entry = 0;
    uint32_t off, dst, off3, dst3;
    const uint8_t *src, *src3;
    auto aim = [&](const Seg &q, int32_t x) {
        // the lane's place in a block, worked out anew: it would be kept in
        // registers that the products need
        int t = threadIdx.x;
        asm volatile("" : "+v"(t));
        off = ((t >> 3) & 7) * ROW + (((t & 7) ^ tile_swz(8 * rb + ((t >> 3) & 7))) << 4);
        const int32_t phys = plan_page(entry, a.n_pages, bad);
        const int32_t at = (phys << a.shift) + ((tile_at<KIND>(q.lk, x) + 8 * rb) & ((1 << a.shift) - 1));
        src = (const uint8_t *)uniform((int64_t)a.pages + (int64_t)at * ROW + c0 * 128);
        const uint32_t slot = stage0 + (x - q.b0) % STAGES * TILE;
        dst = __builtin_amdgcn_readfirstlane(slot + (rb * F::kBlocks + c0) * 1024);
        if constexpr (CODES) {
            off3 = w < 4 ? F::rope_off(t, rb) : (t & 63) * 16;
            src3 = (const uint8_t *)uniform(w < 4 ? (int64_t)a.pages + (int64_t)at * ROW + kPL : (int64_t)(a.scales + at));
            dst3 = __builtin_amdgcn_readfirstlane(slot + (w < 4 ? F::kRope + rb * 512 : F::kScales + rb * 64));
        }
    };
    auto fifth = [&]() {
        if (!CODES && NW == 8 && w < 4) copy_block<4>(off, src, dst);
        if (CODES && l < (w < 4 ? 32 : 4)) copy_block<0>(off3, src3, dst3);
    };
    auto entry_of = [&](const Seg &q, int32_t x) { return page_entry<KIND>(q.lk, page_of<KIND>(q.lk, tile_at<KIND>(q.lk, x) + 8 * rb)); };
    // the row of a wave's column group (kNear: a unit is a sequence)
    auto row_of = [&](int wave) {
        const int grp = chunk * p.per + wave, last = p.groups - 1;
        return (grp < last ? grp : last) / ((a.H + kCols - 1) / kCols);
    };
    auto start = [&](const Seg &q) {
        for (int32_t x = q.b0; x < q.b1 && x < q.b0 + STAGES - 1; x++) {
            entry = entry_of(q, x);
            aim(q, x);
            copy_blocks<0, COPIES>(off, src, dst);
            fifth();
        }
        entry = entry_of(q, q.b0 + STAGES - 1);
    };
    Walk<KIND> walk = {rg.u, rg.first, rg.s};
    Seg q;
    if (!walk.next(p, rg, gr, q)) return;
    bool begun = false;
    while (true) {
        const int64_t row = q.row + (q.h0 + col < a.H ? q.h0 + col : a.H - 1);
        const float c = a.scale * kLog2e * F::load(wv.q, a.qabs, a.qrope, row, g);
        if (!begun) start(q);
        begun = true;
        F::arrive(wv.q, c);
        wv.m = kLow;
        wv.l = 0.0f;
        if constexpr (CODES) {
            wv.top = 0.0f;
            wv.g = 0x1p120f;
            // the first tile's values
            wait_tiles<F>(q.b1 - 1 - q.b0, STAGES - 2);
            convert_tile(stage0, stage0 + STAGES * TILE, w);
        }
#pragma unroll
        for (int mt = 0; mt < 32; mt++) wv.o[mt] = pf32x4{0.0f, 0.0f, 0.0f, 0.0f};
        uint32_t seen = visible<KIND>(q.lk, tile_at<KIND>(q.lk, q.b0), q.n);
        for (int32_t x = q.b0; x < q.b1; x++) {
            const uint32_t ps = (uint32_t)(x - q.b0) % STAGES * TILE;
            uint8_t *T = stage + ps;
            // tile x's copies have landed (of codes: tile x + 1's, and x's values
            // stand): those of the tiles behind it may be on their way
            wait_tiles<F>(q.b1 - 1 - x - (CODES ? 1 : 0), STAGES - 2 - (CODES ? 1 : 0));
            bool due = x + STAGES - 1 < q.b1;
            if (due) {
                aim(q, x + STAGES - 1);
                if (!F::kBetween) {
                    copy_blocks<0, COPIES>(off, src, dst);
                    fifth();
                }
            }
            if constexpr (CODES) {
                // (codes are finite, so that what a row does not see of them needs no care)
                constexpr uint32_t HALF = F::kValues / 2;
                const int32_t page = page_of<KIND>(q.lk, tile_at<KIND>(q.lk, x + STAGES) + 8 * rb);
                const uint32_t V = stage0 + STAGES * TILE, par = (uint32_t)(x - q.b0) & 1;
                const bool more = x + 1 < q.b1;
                const uint32_t from = stage0 + (uint32_t)(x + 1 - q.b0) % STAGES * TILE, to = V + (par ^ 1) * HALF;
                if (more) convert_tile(from, to, w);
                if (active && seen) tile_codes(wv, stage0 + ps, V + par * HALF, seen);
                entry = page_entry<KIND>(q.lk, page);
                seen = visible<KIND>(q.lk, tile_at<KIND>(q.lk, x + 1), q.n);
            } else {
            // what some row of the unit sees, and what every one does
            const uint32_t most = SPARSE ? seen : some_see<KIND>(q.lk, x, q.len);
            const uint32_t least = SPARSE ? seen : all_see<KIND>(q.lk, x, q.len, a.M);
            bool odd = false;
            if (least != ~0u) {
                // a value that is not finite where only later rows look: those
                // rows first, then it is cleared for the rows before (with a
                // window: each wave's row by itself)
                if (most != ~0u) tile_clear<F>(T, ~most);
                if (least != most) {
                    if (tid == 0) s_odd = 0;
                    __syncthreads();
                    if (tile_odd<F>(T, most & ~least)) s_odd = 1;
                }
                __syncthreads();
                odd = least != most && __builtin_amdgcn_readfirstlane(s_odd);
            }
            const int32_t page = page_of<KIND>(q.lk, tile_at<KIND>(q.lk, x + STAGES) + 8 * rb);
            uint32_t now = most;
            int turn = 0;  // a wave
            if (KIND == kNear && odd) {
                tile_clear<F>(T, ~visible<KIND>(q.lk, tile_at<KIND>(q.lk, x), q.len - a.M + row_of(0) + 1));
                __syncthreads();
            }
            do {
                if (active && seen && (!odd || (KIND == kNear ? q.j == row_of(turn) : seen == now)))
                    tile_step<F>(wv, ad, stage0 + ps, seen, c, g, [&](int i) {
                        // a copy every few products
                        constexpr int EVERY = 36 / COPIES;
                        if (F::kBetween && i % EVERY == 0 && due) copy_nth<0, COPIES>(i / EVERY, off, src, dst);
                    });
                else if (F::kBetween && due)
                    copy_blocks<0, COPIES>(off, src, dst);
                due = false;
                if (!odd) break;
                if constexpr (KIND == kNear) {
                    // the tile anew, for the next row that a wave has
                    while (++turn < p.per && row_of(turn) == row_of(turn - 1)) {}
                    if (turn >= p.per) break;
                    __syncthreads();
                    entry = entry_of(q, x);
                    aim(q, x);
                    copy_blocks<0, COPIES>(off, src, dst);
                    fifth();
                    __builtin_amdgcn_s_waitcnt(kWaitVm0);
                    __syncthreads();
                    tile_clear<F>(T, ~visible<KIND>(q.lk, tile_at<KIND>(q.lk, x), q.len - a.M + row_of(turn) + 1));
                    __syncthreads();
                    continue;
                }
                if (now == least) break;
                __syncthreads();
                tile_clear<F>(T, now & ~(now >> 1));
                __syncthreads();
                now >>= 1;
            } while (true);
            entry = page_entry<KIND>(q.lk, page);
            seen = visible<KIND>(q.lk, tile_at<KIND>(q.lk, x + 1), q.n);
            }
        }
        __syncthreads();  // the stages may be filled again: with the next part's first tiles
        Seg nx;
        const bool more = walk.next(p, rg, gr, nx);
        if (more) start(nx);
        // ---- the unit's context, or this range's part of it
        const float sum = col_sum(wv.l);
        if (active && ((SPARSE && p.whole) || (q.b0 == 0 && q.b1 == q.tiles))) {
            const float inv = (sum == 0.0f ? 0.0f : 1.0f / sum) * F::unit(wv);
            const int lo = CODES ? lane_anew() : l, ho = q.h0 + (lo & 15);
            typename F::out_t *out = (typename F::out_t *)a.out + (CODES ? q.row + (ho < a.H ? ho : a.H - 1) : row) * kPL + 4 * (lo >> 4);
            if (ho < a.H)
#pragma unroll
                for (int mt = 0; mt < 32; mt++) {
                    typedef typename F::out_t o4 __attribute__((ext_vector_type(4)));
                    o4 v;
#pragma unroll
                    for (int i = 0; i < 4; i++) v[i] = (typename F::out_t)__fmul_rn(wv.o[mt][i], inv);
                    *(o4 *)(out + 16 * mt) = v;
                }
        } else if (active) {
            const int64_t slot = plan_slot(r, rg.s <= q.first) * p.groups + grp;
            pf32x4 *po = (pf32x4 *)p.part_o + slot * 128 * kCols + g * kCols + col;
#pragma unroll
            for (int mt = 0; mt < 32; mt++) po[mt * 4 * kCols] = CODES ? wv.o[mt] * F::unit(wv) : wv.o[mt];
            if (g == 0) *(float2 *)(p.part_ml + (slot * kCols + col) * 2) = make_float2(wv.m, sum);
        }
        if (!more) break;
        q = nx;
    }
    if (bad && l == 0) *a.err = 1;
}

// Joins the parts of a unit that lies in more than one range:
// out = sum_r o_r 2^(m_r - M) / sum_r l_r 2^(m_r - M).  A workgroup takes one
// column group and 64 dims, each of its NW waves every NW-th part, as many at a
// time as there are, with all their loads under way; the waves' results meet
// in LDS.  Bound by the parts' bytes: 82 MB in 16.9 us (4.9 TB/s); 8 parts of
// one row take 4.2.
template <class F, int KIND, int NW> __global__ __launch_bounds__(NW * 64) void k_paged_join(PagedMfmaArgs p) {
    typedef typename F::out_t o4 __attribute__((ext_vector_type(4)));
    __shared__ __attribute__((aligned(16))) pf32x4 so[NW][16][kCols + 1];  // one more: other banks
    __shared__ float2 sml[NW][kCols];
    const PagedArgs &a = p.a;
    const int u = blockIdx.x / p.groups, grp = blockIdx.x - u * p.groups, tid = threadIdx.x;
    const int w = tid >> 6, col = tid & 15, qd = (tid >> 4) & 3;
    const int64_t W = p.plan[p.units], first = p.plan[u];
    const int64_t tiles = unit_tiles<KIND>(a, u);
    if (tiles == 0) return;
    const int64_t N = plan_ranges(W, p.most, p.spread);
    const int r0 = (int)plan_range_of(W, N, first), r1 = (int)plan_range_of(W, N, first + tiles - 1);
    if (r0 == r1) return;
    float m = kLow, L = 0.0f;
    pf32x4 t[4] = {};
    // some parts: r and every NW-th behind it
    auto add = [&](int r, auto many) {
        constexpr int COUNT = decltype(many)::value;
        float2 ml[COUNT];
        pf32x4 v[COUNT][4];
#pragma unroll
        for (int i = 0; i < COUNT; i++) {
            const int x = r + NW * i;
            const int64_t slot = plan_slot(x, x == r0) * p.groups + grp;
            ml[i] = *(const float2 *)(p.part_ml + (slot * kCols + col) * 2);
#pragma unroll
            for (int k = 0; k < 4; k++)
                v[i][k] = ((const pf32x4 *)p.part_o)[(slot * 128 + blockIdx.y * 16 + qd + 4 * k) * kCols + col];
        }
        float mn = m;
#pragma unroll
        for (int i = 0; i < COUNT; i++) mn = fmaxf(mn, ml[i].x);
        const float f0 = __builtin_amdgcn_exp2f(m - mn);
        L *= f0;
#pragma unroll
        for (int k = 0; k < 4; k++) t[k] *= f0;
#pragma unroll
        for (int i = 0; i < COUNT; i++) {
            const float f = __builtin_amdgcn_exp2f(ml[i].x - mn);
            L = __builtin_fmaf(ml[i].y, f, L);
#pragma unroll
            for (int k = 0; k < 4; k++)
#pragma unroll
                for (int e = 0; e < 4; e++) t[k][e] = __builtin_fmaf(v[i][k][e], f, t[k][e]);
        }
        m = mn;
    };
    int r = r0 + w;
    for (; r + 7 * NW <= r1; r += 8 * NW) add(r, std::integral_constant<int, 8>());
    if (r + 3 * NW <= r1) {
        add(r, std::integral_constant<int, 4>());
        r += 4 * NW;
    }
    if (r + NW <= r1) {
        add(r, std::integral_constant<int, 2>());
        r += 2 * NW;
    }
    if (r <= r1) add(r, std::integral_constant<int, 1>());
    if (qd == 0) sml[w][col] = make_float2(m, L);
#pragma unroll
    for (int k = 0; k < 4; k++) so[w][qd + 4 * k][col] = t[k];
    __syncthreads();
    // thread: four dims (tid & 15) of column tid >> 4
    if (tid >= 256) return;
    const int c = tid >> 4, d = tid & 15;
    float M = kLow, sum = 0.0f;
#pragma unroll
    for (int i = 0; i < NW; i++) M = fmaxf(M, sml[i][c].x);
    pf32x4 o = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
    for (int i = 0; i < NW; i++) {
        const float f = __builtin_amdgcn_exp2f(sml[i][c].x - M);
        const pf32x4 v = so[i][d][c];
        sum = __builtin_fmaf(sml[i][c].y, f, sum);
#pragma unroll
        for (int e = 0; e < 4; e++) o[e] = __builtin_fmaf(v[e], f, o[e]);
    }
    const float inv = sum == 0.0f ? 0.0f : 1.0f / sum;
    o4 v;
#pragma unroll
    for (int e = 0; e < 4; e++) v[e] = (typename F::out_t)__fmul_rn(o[e], inv);
    constexpr bool SPARSE = KIND == kListed;
    const int per_row = (a.H + kCols - 1) / kCols;
    const int64_t row = SPARSE ? u : (int64_t)u * a.M + grp / per_row;
    const int h = (SPARSE ? grp : grp % per_row) * kCols + c;
    if (h < a.H) *(o4 *)((typename F::out_t *)a.out + (row * a.H + h) * kPL + blockIdx.y * 64 + 4 * d) = v;
}

bool paged_mfma_ok(const PagedArgs &a) { return a.L == kPL && a.P == kPD - kPL && a.shift >= 3; }

template <class F, int KIND> static int32_t launch_fmt(ut_ctx *ctx, const PagedArgs &a) {
    constexpr bool SPARSE = KIND == kListed;
    PagedMfmaArgs p{};
    p.a = a;
    p.units = SPARSE ? a.B * a.M : a.B;
    p.groups = (SPARSE ? 1 : a.M) * ((a.H + kCols - 1) / kCols);
    const int64_t cap = (int64_t)(SPARSE ? a.top_k : a.max_pages) << a.shift;
    p.lead = F::kCosts.lead;
    // (a window's rows see the window and up to M - 1 positions more, which may
    // begin and end inside a tile, and so may the first positions)
    const int64_t near = ((int64_t)a.window + a.M - 1 + kPT - 1) / kPT + 1 + ((int64_t)a.sinks + kPT - 1) / kPT;
    const int64_t held = (cap + kPT - 1) / kPT, each = KIND == kNear && near < held ? near : held;
    // (no more pages are to be expected of a list than the table holds: 20 rows of
    // one page and 12 places in f16 pairs 33.0 us cut, 18.6 whole)
    const int64_t listed = (((int64_t)(a.top_k < a.max_pages ? a.top_k : a.max_pages) << a.shift) + kPT - 1) / kPT;
    const PlanCall plan =
        plan_call(F::kCosts, ctx->multiprocessors, p.units, p.groups, each, SPARSE ? listed : each, SPARSE || each < held);
    p.whole = plan.whole;
    p.most = plan.most;
    p.per = plan.per;
    p.chunks = plan.chunks;
    p.spread = plan.spread;
    auto launch = [&]() -> int32_t {
        const int64_t wgs = ((int64_t)p.most * p.chunks + 7) / 8 * 8;
        int tok = timing_begin(ctx, "paged_mfma");
        hipLaunchKernelGGL((k_paged_mfma<F, KIND>), dim3((unsigned)wgs), dim3(F::kWaves * 64), 0, ctx->stream, p);
        timing_end(ctx, tok);
        return launch_check(ctx, "k_paged_mfma");
    };
    if (plan.slots == 0) return launch();  // nothing is left to join
    ScratchPlan scratch;
    scratch.add((size_t)plan.slots * kPL * kCols * 4);
    scratch.add((size_t)plan.slots * kCols * 8);
    scratch.add((size_t)(p.units + 1) * 8);
    std::vector<void *> ptrs;
    UT_TRY(scratch_acquire(ctx, scratch, ptrs));
    p.part_o = (float *)ptrs[0];
    p.part_ml = (float *)ptrs[1];
    p.plan = (int64_t *)ptrs[2];
    UT_TRY(launch());
    const dim3 grid((unsigned)((int64_t)p.units * p.groups), kPlanJoinSlices);
    int tok = timing_begin(ctx, "paged_join");
    if (plan.wide)
        hipLaunchKernelGGL((k_paged_join<F, KIND, 16>), grid, dim3(1024), 0, ctx->stream, p);
    else
        hipLaunchKernelGGL((k_paged_join<F, KIND, 4>), grid, dim3(256), 0, ctx->stream, p);
    timing_end(ctx, tok);
    return launch_check(ctx, "k_paged_join");
}

int32_t launch_paged_mfma(ut_ctx *ctx, const PagedArgs &a, int32_t fmt) {
    auto launch = [&](auto f) {
        typedef decltype(f) F;
        return a.sel ? launch_fmt<F, kListed>(ctx, a) : a.window ? launch_fmt<F, kNear>(ctx, a) : launch_fmt<F, kAll>(ctx, a);
    };
    return fmt == UT_KV_BF16 ? launch(MfmaBf16()) : fmt == UT_KV_I8 ? launch(MfmaI8()) : launch(MfmaF16x2());
}

}  // namespace ut
