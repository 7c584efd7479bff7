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

// Tiles of a unit.
template <bool SPARSE> __device__ __forceinline__ int32_t unit_tiles(const PagedArgs &a, int u) {
    if (!SPARSE) return (int32_t)(((int64_t)paged_len(a, u) + kPT - 1) / kPT);
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
template <bool SPARSE, int NW>
__device__ bool find_range(const PagedMfmaArgs &p, int64_t r, bool leave, Range &g) {
    __shared__ int64_t s[NW];
    __shared__ int64_t found[2];
    const int tid = threadIdx.x;
    if (p.whole) {
        const PagedArgs &a = p.a;
        const int u = (int)r;
        g = {0, 0, __builtin_amdgcn_readfirstlane(unit_tiles<SPARSE>(a, u)), u, 0};
        if (SPARSE && g.e > 0) {
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
        int32_t t = lane < p.units ? unit_tiles<SPARSE>(p.a, lane) : 0;
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
        t = u < p.units ? unit_tiles<SPARSE>(p.a, u) : 0;
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
            t = u < p.units ? unit_tiles<SPARSE>(p.a, u) : 0;
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
};
template <int PLANES> __device__ __forceinline__ LaneAddr lane_addr(int l) {
    const int row = l & 15, g = l >> 4, j = l & 15, r = 4 * g + (j >> 2);
    return {(uint32_t)((row >> 3) * 9 * PLANES * 1024 + (row & 7) * 128 + ((g ^ tile_swz(row)) << 4)),
            (uint32_t)((r >> 3) * 9 * PLANES * 1024 + (r & 7) * 128 + ((((j & 3) >> 1) ^ tile_swz(r)) << 4) +
                       8 * (j & 1))};
}

// bf16 pages: queries and weights in bf16.
struct MfmaBf16 {
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
    __device__ __forceinline__ static void arrive(Query &x) {
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
    __device__ __forceinline__ static void arrive(Query &) {}  // converted: they are there
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

// One wave's columns: 16 heads of one query row, the whole latent width.
template <class F> struct Wave {
    typename F::Query q;
    pf32x4 o[32];  // context^T: dim 16 mt + 4 (l >> 4) + i, column l & 15
    float m, l;    // softmax offset (log2 units) and sum
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
};
// The page of the sequence that holds the unit's position v0; one that it
// does have, where there is none or it lies behind the end.
template <bool SPARSE> __device__ __forceinline__ int32_t page_of(const Lookup &k, int32_t v0) {
    if (SPARSE) {
        const int32_t i = v0 >> k.shift;
        return i < k.top_k ? k.sel[i] : 0;
    }
    return (v0 < k.n ? v0 : k.n - 1) >> k.shift;
}
template <bool SPARSE> __device__ __forceinline__ int32_t page_entry(const Lookup &k, int32_t page) {
    // the pool's first page stands in for one that is not listed or not seen: the
    // table need not name any but the listed ones
    const bool none = SPARSE && (page < 0 || ((int64_t)page << k.shift) >= k.n);
    const int32_t entry = k.table[none ? 0 : page];
    return none ? 0 : entry;
}
// The visible positions of the tile at v0 for a row that sees n.
template <bool SPARSE>
__device__ __forceinline__ uint32_t visible(const Lookup &k, int32_t v0, int32_t n) {
    if (!SPARSE) {
        const int32_t c = n - v0;
        return c >= 32 ? ~0u : c <= 0 ? 0u : (1u << c) - 1u;
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

// The part of a range that lies in one unit.
struct Seg {
    int32_t u, j, h0, b0, b1, tiles, len, n;
    int64_t first, row;
    Lookup lk;
};
// Goes over a range's parts.
template <bool SPARSE> struct Walk {
    int32_t u;
    int64_t first, at;
    __device__ __forceinline__ bool next(const PagedMfmaArgs &p, const Range &rg, int gr, Seg &q) {
        const PagedArgs &a = p.a;
        int32_t tiles = 0;
        while (at < rg.e && !(tiles = __builtin_amdgcn_readfirstlane(unit_tiles<SPARSE>(a, u)))) u++;
        q.b0 = at > first ? (int32_t)(at - first) : 0;
        q.b1 = rg.e - first < tiles ? (int32_t)(rg.e - first) : tiles;
        if (q.b0 >= q.b1) return false;
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
template <class F, bool SPARSE>
__global__ __launch_bounds__(F::kWaves * 64, F::kWaves / 4) void k_paged_mfma(PagedMfmaArgs p) {
    constexpr int NW = F::kWaves, PL = F::kPlanes, STAGES = 4 / PL, ROW = kPD * 2 * PL, TILE = 36 * PL * 1024;
    __shared__ __attribute__((aligned(1024))) uint8_t stage[STAGES * TILE];
    __shared__ int s_odd;
    const PagedArgs &a = p.a;
    const int tid = threadIdx.x, w = __builtin_amdgcn_readfirstlane(tid >> 6), l = tid & 63, g = l >> 4, col = l & 15;
    const int share = gridDim.x >> 3;
    const int id = (blockIdx.x & 7) * share + (blockIdx.x >> 3);  // neighbours on one XCD
    const int r = id / p.chunks, chunk = id - r * p.chunks;
    // units without positions: zeros
    const int64_t vec = (int64_t)(SPARSE ? 1 : a.M) * a.H * kPL * (int)sizeof(typename F::out_t) / 16;
    for (int u = id; u < p.units; u += gridDim.x)
        if (unit_tiles<SPARSE>(a, u) == 0)
            for (int64_t i = tid; i < vec; i += NW * 64) ((pu32x4 *)a.out)[u * vec + i] = pu32x4{0, 0, 0, 0};
    Range rg;
    if (r >= p.most || !find_range<SPARSE, NW>(p, r, p.most > 1 && r == 0 && chunk == 0, rg)) return;
    const int grp = chunk * p.per + w;
    const bool active = w < p.per && grp < p.groups;
    const int gr = active ? grp : 0;
    const LaneAddr ad = lane_addr<PL>(l);
    const uint32_t stage0 = (uint32_t)(uintptr_t)(lds_u8 *)stage;
    // copies: wave w brings row block w & 3 and, where two waves share it, half of its column blocks
    const int rb = w & 3, c0 = NW == 8 && w >= 4 ? 5 : 0;
    constexpr int COPIES = NW == 4 ? 9 * PL : 4;  // and a fifth of waves 0 to 3
    Wave<F> wv;
    bool bad = false;
    // the next copy: its table entry, and where it goes
    int32_t entry = 0;
    uint32_t off, dst;
    const uint8_t *src;
    auto aim = [&](const Seg &q, int32_t x) {
        // the lane's place in a block, worked out anew: it would be kept in
        // registers that the products need
        int t = threadIdx.x;
        asm volatile("" : "+v"(t));
        off = ((t >> 3) & 7) * ROW + (((t & 7) ^ tile_swz(8 * rb + ((t >> 3) & 7))) << 4);
        const int32_t phys = plan_page(entry, a.n_pages, bad);
        const int32_t at = (phys << a.shift) + ((x * kPT + 8 * rb) & ((1 << a.shift) - 1));
        src = (const uint8_t *)uniform((int64_t)a.pages + (int64_t)at * ROW + c0 * 128);
        dst = __builtin_amdgcn_readfirstlane(stage0 + (x - q.b0) % STAGES * TILE + (rb * 9 * PL + c0) * 1024);
    };
    auto fifth = [&]() {
        if (NW == 8 && w < 4) copy_block<4>(off, src, dst);
    };
    auto entry_of = [&](const Seg &q, int32_t x) { return page_entry<SPARSE>(q.lk, page_of<SPARSE>(q.lk, x * kPT + 8 * rb)); };
    auto start = [&](const Seg &q) {
        for (int32_t x = q.b0; x < q.b1 && x < q.b0 + STAGES - 1; x++) {
            entry = entry_of(q, x);
            aim(q, x);
            copy_blocks<0, COPIES>(off, src, dst);
            fifth();
        }
        entry = entry_of(q, q.b0 + STAGES - 1);
    };
    Walk<SPARSE> walk = {rg.u, rg.first, rg.s};
    Seg q;
    if (!walk.next(p, rg, gr, q)) return;
    bool begun = false;
    while (true) {
        const int64_t row = q.row + (q.h0 + col < a.H ? q.h0 + col : a.H - 1);
        const float c = a.scale * kLog2e * F::load(wv.q, a.qabs, a.qrope, row, g);
        if (!begun) start(q);
        begun = true;
        F::arrive(wv.q);
        wv.m = kLow;
        wv.l = 0.0f;
#pragma unroll
        for (int mt = 0; mt < 32; mt++) wv.o[mt] = pf32x4{0.0f, 0.0f, 0.0f, 0.0f};
        uint32_t seen = visible<SPARSE>(q.lk, q.b0 * kPT, q.n);
        for (int32_t x = q.b0; x < q.b1; x++) {
            const uint32_t ps = (uint32_t)(x - q.b0) % STAGES * TILE;
            uint8_t *T = stage + ps;
            // tile x's copies have landed: those of the tiles behind it may be on their way
            const int32_t ahead = q.b1 - 1 - x < STAGES - 2 ? q.b1 - 1 - x : STAGES - 2;
            if (ahead >= 2) __builtin_amdgcn_s_waitcnt(kWaitVm8);
            else if (ahead == 1) __builtin_amdgcn_s_waitcnt(kWaitVm4);
            else __builtin_amdgcn_s_waitcnt(kWaitVm0);
            __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
            __builtin_amdgcn_s_barrier();
            __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
            bool due = x + STAGES - 1 < q.b1;
            if (due) {
                aim(q, x + STAGES - 1);
                if (!F::kBetween) {
                    copy_blocks<0, COPIES>(off, src, dst);
                    fifth();
                }
            }
            // what the unit's last row sees, and its first one
            const uint32_t most = SPARSE ? seen : visible<false>(q.lk, x * kPT, q.len);
            const uint32_t least = SPARSE ? seen : visible<false>(q.lk, x * kPT, q.len - a.M + 1);
            bool odd = false;
            if (least != ~0u) {
                // a value that is not finite where only later rows look: those
                // rows first, then it is cleared for the rows before
                if (most != ~0u) tile_clear<F>(T, ~most);
                if (least != most) {
                    if (tid == 0) s_odd = 0;
                    __syncthreads();
                    if (tile_odd<F>(T, most & ~least)) s_odd = 1;
                }
                __syncthreads();
                odd = least != most && __builtin_amdgcn_readfirstlane(s_odd);
            }
            const int32_t page = page_of<SPARSE>(q.lk, (x + STAGES) * kPT + 8 * rb);
            uint32_t now = most;
            do {
                if (active && seen && (!odd || seen == now))
                    tile_step<F>(wv, ad, stage0 + ps, seen, c, g, [&](int i) {
                        // a copy every few products
                        constexpr int EVERY = 36 / COPIES;
                        if (F::kBetween && i % EVERY == 0 && due) copy_nth<0, COPIES>(i / EVERY, off, src, dst);
                    });
                else if (F::kBetween && due)
                    copy_blocks<0, COPIES>(off, src, dst);
                due = false;
                if (!odd || now == least) break;
                __syncthreads();
                tile_clear<F>(T, now & ~(now >> 1));
                __syncthreads();
                now >>= 1;
            } while (true);
            entry = page_entry<SPARSE>(q.lk, page);
            seen = visible<SPARSE>(q.lk, (x + 1) * kPT, q.n);
        }
        __syncthreads();  // the stages may be filled again: with the next part's first tiles
        Seg nx;
        const bool more = walk.next(p, rg, gr, nx);
        if (more) start(nx);
        // ---- the unit's context, or this range's part of it
        const float sum = col_sum(wv.l);
        if (active && ((SPARSE && p.whole) || (q.b0 == 0 && q.b1 == q.tiles))) {
            const float inv = sum == 0.0f ? 0.0f : 1.0f / sum;
            typename F::out_t *out = (typename F::out_t *)a.out + row * kPL + 4 * g;
            if (q.h0 + col < a.H)
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
            for (int mt = 0; mt < 32; mt++) po[mt * 4 * kCols] = wv.o[mt];
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
template <class F, bool SPARSE, int NW> __global__ __launch_bounds__(NW * 64) void k_paged_join(PagedMfmaArgs p) {
    typedef typename F::out_t o4 __attribute__((ext_vector_type(4)));
    __shared__ __attribute__((aligned(16))) pf32x4 so[NW][16][kCols + 1];  // one more: other banks
    __shared__ float2 sml[NW][kCols];
    const PagedArgs &a = p.a;
    const int u = blockIdx.x / p.groups, grp = blockIdx.x - u * p.groups, tid = threadIdx.x;
    const int w = tid >> 6, col = tid & 15, qd = (tid >> 4) & 3;
    const int64_t W = p.plan[p.units], first = p.plan[u];
    const int64_t tiles = unit_tiles<SPARSE>(a, u);
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
    const int per_row = (a.H + kCols - 1) / kCols;
    const int64_t row = SPARSE ? u : (int64_t)u * a.M + grp / per_row;
    const int h = (SPARSE ? grp : grp % per_row) * kCols + c;
    if (h < a.H) *(o4 *)((typename F::out_t *)a.out + (row * a.H + h) * kPL + blockIdx.y * 64 + 4 * d) = v;
}

bool paged_mfma_ok(const PagedArgs &a) { return a.L == kPL && a.P == kPD - kPL && a.shift >= 3; }

template <class F, bool SPARSE> static int32_t launch_fmt(ut_ctx *ctx, const PagedArgs &a) {
    PagedMfmaArgs p{};
    p.a = a;
    p.units = SPARSE ? a.B * a.M : a.B;
    p.groups = (SPARSE ? 1 : a.M) * ((a.H + kCols - 1) / kCols);
    const int64_t cap = (int64_t)(SPARSE ? a.top_k : a.max_pages) << a.shift;
    p.lead = F::kCosts.lead;
    const int64_t each = (cap + kPT - 1) / kPT;
    // (no more pages are to be expected of a list than the table holds: 20 rows of
    // one page and 12 places in f16 pairs 33.0 us cut, 18.6 whole)
    const int64_t listed = (((int64_t)(a.top_k < a.max_pages ? a.top_k : a.max_pages) << a.shift) + kPT - 1) / kPT;
    const PlanCall plan =
        plan_call(F::kCosts, ctx->multiprocessors, p.units, p.groups, each, SPARSE ? listed : each, SPARSE);
    p.whole = plan.whole;
    p.most = plan.most;
    p.per = plan.per;
    p.chunks = plan.chunks;
    p.spread = plan.spread;
    auto launch = [&]() -> int32_t {
        const int64_t wgs = ((int64_t)p.most * p.chunks + 7) / 8 * 8;
        int tok = timing_begin(ctx, "paged_mfma");
        hipLaunchKernelGGL((k_paged_mfma<F, SPARSE>), dim3((unsigned)wgs), dim3(F::kWaves * 64), 0, ctx->stream, p);
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
        hipLaunchKernelGGL((k_paged_join<F, SPARSE, 16>), grid, dim3(1024), 0, ctx->stream, p);
    else
        hipLaunchKernelGGL((k_paged_join<F, SPARSE, 4>), grid, dim3(256), 0, ctx->stream, p);
    timing_end(ctx, tok);
    return launch_check(ctx, "k_paged_join");
}

int32_t launch_paged_mfma(ut_ctx *ctx, const PagedArgs &a, int32_t fmt) {
    if (fmt == UT_KV_BF16) return a.sel ? launch_fmt<MfmaBf16, true>(ctx, a) : launch_fmt<MfmaBf16, false>(ctx, a);
    return a.sel ? launch_fmt<MfmaF16x2, true>(ctx, a) : launch_fmt<MfmaF16x2, false>(ctx, a);
}

}  // namespace ut
