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
//
// With a window a unit is a sequence's tiles that some row sees, first ones and
// window, numbered without those between: one row over 1024 of 16384 positions
// 15.3 us in all, 13 x 3 rows of 64 heads over 777 of up to 5003 in f16x2 45.8.
#include <type_traits>

#include "ut_paged_attend.h"

namespace ut {

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
    static constexpr bool kCodes = false;
    static constexpr PlanCosts kCosts = kCostsBf16;
    static constexpr int kPlanes = 1, kWaves = kCosts.waves;
    static constexpr bool kBetween = false;  // copies between the products (the branches cost registers)
    static constexpr int kDepth = 4;
    static constexpr float kRise = 11.5f;  // log2 units a score may exceed the offset (8 nats)
    typedef __bf16 out_t;
    typedef float part_t;
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
    static constexpr bool kCodes = false;
    static constexpr PlanCosts kCosts = kCostsF16x2;
    static constexpr int kPlanes = 2, kWaves = kCosts.waves;
    static constexpr bool kBetween = true;
    static constexpr int kDepth = 4;
    static constexpr float kRise = 1.0f;
    typedef float out_t;
    typedef float part_t;
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

// A workgroup is F::kWaves waves, each with a column group of its own, over
// the same tiles.  Four (f16x2: two) tiles fit the LDS: the products of one
// run while the next three (one) are on their way.  A table entry is read a
// tile before its copy, and the copies issue between the products.
// FEW: some waves have no heads, and load no queries (one row over 509 positions
// 15.5 us where all load some, 12.3 so; with the branch where all have heads, 64
// sequences of up to 8192 positions 121 us instead of 117).
template <class F, int KIND, bool OWN, bool FEW>
__global__ __launch_bounds__(F::kWaves * 64, F::kWaves / 4) void k_paged_mfma(PagedMfmaArgs p) {
    constexpr bool SPARSE = KIND == kListed;
    constexpr int NW = F::kWaves, PL = F::kPlanes, STAGES = 4 / PL, ROW = kPD * 2 * PL, TILE = 36 * PL * 1024;
    __shared__ __attribute__((aligned(1024))) uint8_t stage[STAGES * TILE];
    __shared__ int s_odd;
    const PagedArgs &a = p.a;
    const int tid = threadIdx.x, w = __builtin_amdgcn_readfirstlane(tid >> 6), l = tid & 63, g = l >> 4, col = l & 15;
    int r, chunk;
    const int id = place<OWN>(p.chunks, r, chunk);
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
        const int32_t at = (phys << a.shift) + ((tile_at<KIND>(q.lk, x) + 8 * rb) & ((1 << a.shift) - 1));
        src = (const uint8_t *)uniform((int64_t)a.pages + (int64_t)at * ROW + c0 * 128);
        dst = __builtin_amdgcn_readfirstlane(stage0 + (x - q.b0) % STAGES * TILE + (rb * 9 * PL + c0) * 1024);
    };
    auto fifth = [&]() {
        if (NW == 8 && w < 4) copy_block<4>(off, src, dst);
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
    Walk<KIND, OWN> walk = walk_of<KIND, OWN>(p, rg, chunk);
    Seg q;
    if (!walk.next(p, rg, gr, q)) return;
    bool begun = false;
    while (true) {
        const int64_t row = q.row + (q.h0 + col < a.H ? q.h0 + col : a.H - 1);
        float c = 0.0f;
        if (!FEW || active) c = a.scale * kLog2e * F::load(wv.q, a.qabs, a.qrope, row, g);
        if (!begun) start(q);
        begun = true;
        if (!FEW || active) {
            F::arrive(wv.q);
            wv.m = kLow;
            wv.l = 0.0f;
#pragma unroll
            for (int mt = 0; mt < 32; mt++) wv.o[mt] = pf32x4{0.0f, 0.0f, 0.0f, 0.0f};
        }
        uint32_t seen = visible<KIND>(q.lk, tile_at<KIND>(q.lk, q.b0), q.n);
        for (int32_t x = q.b0; x < q.b1; x++) {
            const uint32_t ps = (uint32_t)(x - q.b0) % STAGES * TILE;
            uint8_t *T = stage + ps;
            // tile x's copies have landed: those of the tiles behind it may be on
            // their way (a tile's copies are 5 of one half of the waves and 4 of the
            // other; waiting for the fewer suits both)
            const int32_t ahead = q.b1 - 1 - x < STAGES - 2 ? q.b1 - 1 - x : STAGES - 2;
            if (ahead >= 2) __builtin_amdgcn_s_waitcnt(wait_vm(8));
            else if (ahead == 1) __builtin_amdgcn_s_waitcnt(wait_vm(4));
            else __builtin_amdgcn_s_waitcnt(wait_vm(0));
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
            // what some row of the unit sees, and what every one does
            const uint32_t most = SPARSE ? seen : some_see<KIND>(q.lk, x, q.len);
            const uint32_t least = SPARSE ? seen : all_see<KIND>(q.lk, x, q.len, OWN ? q.rows : a.M);
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
                tile_clear<F>(T, ~visible<KIND>(q.lk, tile_at<KIND>(q.lk, x), (OWN ? q.base : q.len - a.M + 1) + row_of(0)));
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
                    __builtin_amdgcn_s_waitcnt(wait_vm(0));
                    __syncthreads();
                    tile_clear<F>(T, ~visible<KIND>(q.lk, tile_at<KIND>(q.lk, x), (OWN ? q.base : q.len - a.M + 1) + row_of(turn)));
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
// out = sum_r o_r 2^(m_r - M) / sum_r l_r 2^(m_r - M); of 8-bit pages the contexts
// have offsets of their own, k_r and K.  A workgroup takes one column group and 16
// NQ dims, each of its NW waves every NW-th part, as many at a time as there are,
// with all their loads under way; the waves' results meet in LDS.  Bound by the
// parts' bytes: 82 MB in 16.9 us (4.9 TB/s); 8 parts of one row take 4.2.  NQ = 1
// where that gives no more workgroups than CUs: one row over 32768 positions in 8
// bits 39.1 us with 4, 36.8 with 1 (bf16 34.0 and 32.8, f16x2 54.2 and 52.2); two
// such rows, on 512 workgroups, 44.8 and 46.0 (bf16 45.7 and 44.9).
template <class F, int KIND, int NW, int NQ> __global__ __launch_bounds__(NW * 64) void k_paged_join(PagedMfmaArgs p) {
    typedef typename F::out_t o4 __attribute__((ext_vector_type(4)));
    typedef typename F::part_t p4 __attribute__((ext_vector_type(4)));
    __shared__ __attribute__((aligned(16))) pf32x4 so[NW][4 * NQ][kCols + 1];  // one more: other banks
    __shared__ float2 sml[NW][kCols];
    __shared__ float sk[NW][kCols];  // 8-bit pages
    const PagedArgs &a = p.a;
    const int u = blockIdx.x / p.groups, grp = blockIdx.x - u * p.groups, tid = threadIdx.x;
    const int w = tid >> 6, col = tid & 15, qd = (tid >> 4) & 3;
    const int64_t W = p.plan[p.units], first = p.plan[u];
    const int64_t tiles = unit_tiles<KIND>(a, u);
    if (tiles == 0) return;
    const int64_t N = plan_ranges(W, p.most, p.spread);
    const int r0 = (int)plan_range_of(W, N, first), r1 = (int)plan_range_of(W, N, first + tiles - 1);
    if (r0 == r1) return;
    float m = kLow, L = 0.0f, at = kLow;
    pf32x4 t[NQ] = {};
    // some parts: r and every NW-th behind it
    auto add = [&](int r, auto many) {
        constexpr int COUNT = decltype(many)::value;
        float2 ml[COUNT];
        float k[COUNT];  // the contexts' offsets
        p4 v[COUNT][NQ];
#pragma unroll
        for (int i = 0; i < COUNT; i++) {
            const int x = r + NW * i;
            const int64_t slot = plan_slot(x, x == r0) * p.groups + grp;
            if constexpr (F::kCodes) {
                const float4 x = *(const float4 *)(p.part_ml + (slot * kCols + col) * 4);
                ml[i] = make_float2(x.x, x.y);
                k[i] = x.z;
            } else {
                ml[i] = *(const float2 *)(p.part_ml + (slot * kCols + col) * 2);
                k[i] = kLow;  // (none: as the sum's)
            }
#pragma unroll
            for (int j = 0; j < NQ; j++)
                v[i][j] = ((const p4 *)p.part_o)[(slot * 128 + blockIdx.y * 4 * NQ + qd + 4 * j) * kCols + col];
        }
        float mn = m, kn = at;
#pragma unroll
        for (int i = 0; i < COUNT; i++) {
            mn = fmaxf(mn, ml[i].x);
            if constexpr (F::kCodes) kn = fmaxf(kn, k[i]);
        }
        const float f0 = __builtin_amdgcn_exp2f(m - mn), g0 = F::kCodes ? __builtin_amdgcn_exp2f(at - kn) : f0;
        L *= f0;
#pragma unroll
        for (int j = 0; j < NQ; j++) t[j] *= g0;
#pragma unroll
        for (int i = 0; i < COUNT; i++) {
            const float f = __builtin_amdgcn_exp2f(ml[i].x - mn), g = F::kCodes ? __builtin_amdgcn_exp2f(k[i] - kn) : f;
            L = __builtin_fmaf(ml[i].y, f, L);
#pragma unroll
            for (int j = 0; j < NQ; j++)
#pragma unroll
                for (int e = 0; e < 4; e++) t[j][e] = __builtin_fmaf((float)v[i][j][e], g, t[j][e]);
        }
        at = kn;
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
    if (F::kCodes && qd == 0) sk[w][col] = at;
#pragma unroll
    for (int k = 0; k < NQ; k++) so[w][qd + 4 * k][col] = t[k];
    __syncthreads();
    // thread: four dims of a column (and of those behind it that have no thread)
    constexpr bool SPARSE = KIND == kListed;
    const int per_row = (a.H + kCols - 1) / kCols, d = tid % (4 * NQ);
    const int64_t row = SPARSE ? u : (int64_t)u * a.M + grp / per_row;
#pragma unroll
    for (int c = tid / (4 * NQ); c < kCols; c += 16 * NW / NQ) {
        float M = kLow, K = kLow, sum = 0.0f;
#pragma unroll
        for (int i = 0; i < NW; i++) {
            M = fmaxf(M, sml[i][c].x);
            if (F::kCodes) K = fmaxf(K, sk[i][c]);
        }
        pf32x4 o = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
        for (int i = 0; i < NW; i++) {
            const float f = __builtin_amdgcn_exp2f(sml[i][c].x - M), g = F::kCodes ? __builtin_amdgcn_exp2f(sk[i][c] - K) : f;
            const pf32x4 v = so[i][d][c];
            sum = __builtin_fmaf(sml[i][c].y, f, sum);
#pragma unroll
            for (int e = 0; e < 4; e++) o[e] = __builtin_fmaf(v[e], g, o[e]);
        }
        const float inv = sum == 0.0f ? 0.0f : 1.0f / sum;
        o4 v;
#pragma unroll
        for (int e = 0; e < 4; e++) {
            const float x = __fmul_rn(o[e], inv);
            v[e] = (typename F::out_t)(F::kCodes ? ldexpf(x, (int)(K - M)) : x);
        }
        const int h = (SPARSE ? grp : grp % per_row) * kCols + c;
        if (h < a.H) *(o4 *)((typename F::out_t *)a.out + (row * a.H + h) * kPL + blockIdx.y * 16 * NQ + 4 * d) = v;
    }
}

bool paged_mfma_ok(const PagedArgs &a) { return a.L == kPL && a.P == kPD - kPL && a.shift >= 3; }

template <class F, int KIND> static int32_t launch_fmt(ut_ctx *ctx, const PagedArgs &a) {
    constexpr bool SPARSE = KIND == kListed;
    PagedMfmaArgs p{};
    p.a = a;
    p.units = SPARSE ? a.B * a.M : a.B;
    p.groups = (SPARSE ? 1 : a.M) * ((a.H + kCols - 1) / kCols);
    const int64_t cap = (int64_t)(SPARSE ? a.top_k : a.max_pages) << a.shift;
    p.lead = plan_lead(F::kCosts, p.groups);
    const int64_t near = near_most(a.M, a.window, a.sinks, kPT);
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
    // prompts: no parts, and rows whose ends lie more than a tile apart
    const bool own = plan.slots == 0 && a.M > kPT;
    auto launch = [&]() -> int32_t {
        const unsigned wgs = (unsigned)(((int64_t)p.most * p.chunks + 7) / 8 * 8);
        int tok = timing_begin(ctx, F::kCodes ? "paged_codes" : "paged_mfma");
        if constexpr (F::kCodes) launch_codes(ctx, p, KIND, own, wgs);
        else if (KIND != kListed && own)
            hipLaunchKernelGGL((k_paged_mfma<F, KIND, KIND != kListed, false>), dim3(wgs), dim3(F::kWaves * 64), 0, ctx->stream, p);
        else if (p.per < F::kCosts.waves)
            hipLaunchKernelGGL((k_paged_mfma<F, KIND, false, true>), dim3(wgs), dim3(F::kWaves * 64), 0, ctx->stream, p);
        else
            hipLaunchKernelGGL((k_paged_mfma<F, KIND, false, false>), dim3(wgs), dim3(F::kWaves * 64), 0, ctx->stream, p);
        timing_end(ctx, tok);
        return launch_check(ctx, F::kCodes ? "k_paged_codes" : "k_paged_mfma");
    };
    if (plan.slots == 0) return launch();  // nothing is left to join
    ScratchPlan scratch;
    scratch.add((size_t)plan.slots * kPL * kCols * sizeof(typename F::part_t));
    scratch.add((size_t)plan.slots * kCols * (F::kCodes ? 16 : 8));
    scratch.add((size_t)(p.units + 1) * 8);
    std::vector<void *> ptrs;
    UT_TRY(scratch_acquire(ctx, scratch, ptrs));
    p.part_o = ptrs[0];
    p.part_ml = (float *)ptrs[1];
    p.plan = (int64_t *)ptrs[2];
    UT_TRY(launch());
    const dim3 grid((unsigned)((int64_t)p.units * p.groups), kPlanJoinSlices);
    int tok = timing_begin(ctx, "paged_join");
    // (8-bit pages: one wave where a unit has few parts, so that more workgroups run at a time: 256
    // sequences of up to 2048 positions 148 us with four, 137 with two, 133 with one)
    if (F::kCodes && p.most <= 8 * p.units)
        hipLaunchKernelGGL((k_paged_join<F, KIND, 1, 4>), grid, dim3(64), 0, ctx->stream, p);
    else if (plan.wide && (int64_t)grid.x * 4 * kPlanJoinSlices <= ctx->multiprocessors)
        hipLaunchKernelGGL((k_paged_join<F, KIND, 16, 1>), dim3(grid.x, 4 * kPlanJoinSlices), dim3(1024), 0, ctx->stream, p);
    else if (plan.wide)
        hipLaunchKernelGGL((k_paged_join<F, KIND, 16, 4>), grid, dim3(1024), 0, ctx->stream, p);
    else
        hipLaunchKernelGGL((k_paged_join<F, KIND, 4, 4>), grid, dim3(256), 0, ctx->stream, p);
    timing_end(ctx, tok);
    return launch_check(ctx, "k_paged_join");
}

int32_t launch_paged_mfma(ut_ctx *ctx, const PagedArgs &a, int32_t fmt) {
    auto launch = [&](auto f) {
        typedef decltype(f) F;
        return a.sel ? launch_fmt<F, kListed>(ctx, a) : a.window ? launch_fmt<F, kNear>(ctx, a) : launch_fmt<F, kAll>(ctx, a);
    };
    return fmt == UT_KV_BF16 ? launch(MfmaBf16()) : fmt == UT_KV_I8 ? launch(CodesI8()) : launch(MfmaF16x2());
}

}  // namespace ut
