// ut_paged_codes.hip -- attention over 8-bit pages on the matrix cores, for
// latent 512 + rope 64 and pages of 8 positions and more.
//
// With codes c and scales a, of a position's latent and of its rotary key:
//   s_ht = scale (a_t q_h^lat . c_t^lat + a'_t q_h^rope . c_t^rope),
//   out_h = sum_t e^(s_ht - m_h) a_t c_t^lat / sum_t e^(s_ht - m_h).
//
// Scores are products of integers: each part of a query, scaled to 32512 at its
// largest, is split in two digits of 8 bits, x = 256 hi + lo, that meet the codes
// as they lie in LDS on the int8 matrix cores: two products of twice the bf16
// rate for one of it, sums exact in 32 bits, a query off by 2^-16 of its part's
// largest at most.  Values: codes as f16, which holds them exactly, converted once
// for a workgroup's waves; a weight meets its position's scale before it is
// rounded to f16, w = 2^up e^(s - m) a, the largest so far at 2^10 to 2^16, so that
// one loses bits from 2^-24 of the largest down.  Scales may be of any size, and
// the sum of the weights themselves, in f32, must not depend on that: a column has
// an offset m for its scores and a power of two, up, for its products.  m does
// what it can of both: up is 0 as long as m, so chosen, puts the largest weight, or
// the sum where that is larger, at 2^-10 to 2^60 when it moves (2^90 before it has
// to move; the sum of 2^31 of those stays in f32).  So weights below 2^-116 of the
// sum may be lost, and nothing above them.  All are powers of two, so that a move
// changes no bit.  (What a query's digit is worth is an f32 number, and its product
// with the codes' sum another: scores of parts whose largest value lies below 2^-100
// lose bits, above 2^100 they may overflow.)
//
// A position is 584 bytes, half a bf16 one, for the same products at the same
// rate, so that memory bounds up to some 64 heads and the matrix cores 128.  A
// wave has its columns' whole context and queries in registers (two waves a SIMD),
// and what it does between products (conversion, scales, softmax, look-ups) takes
// as long as they do: the two waves of a SIMD must not do that at the same time.
// Hence two workgroups a CU, four waves each, that know nothing of one another, and
// a higher priority for the one that is past its scores.  What bounds it now, with
// tiles of 32 positions:
// - 128 heads: instructions.  A tile takes 2.4 us a CU where its data come from L2
//   (512 prompt rows over 8192 positions 1220 us, 0.91 PFLOP/s; without the priority
//   6 % more; bf16 pages, which need no conversion, 1020), 2.6 to 2.8 with the traffic
//   of decoding: 64 sequences of up to 8192 118 us, as bf16.
// - 16 heads: memory, 1.03 us a tile and CU (4.7 TB/s), once it runs: 37 sequences
//   of up to 12001 46 us in all (132 MB), of which its start, the ranges' ends and
//   the join take 18.
// - few rows: latency.  Of a call over one tile, 9.7 us, the lengths and the range
//   take 0.8, the walk's values 0.5, the queries' issue 0.8 and their digits 1.1,
//   the tile 1.9, the end 1.5.
#include "ut_paged_attend.h"

namespace ut {

typedef int pi32x4 __attribute__((ext_vector_type(4)));
typedef _Float16 pf16x2 __attribute__((ext_vector_type(2)));
typedef uint32_t pu32x2 __attribute__((ext_vector_type(2)));

constexpr int kCW = kCostsI8.waves, kCodesPerCu = kCostsI8.slots;
// LDS: two tiles of codes (32 x 512 latent ones in 16 blocks of 8 rows and 128
// bytes, 32 x 64 rotary ones), the scales of four tiles, one tile's values, the columns' up.
constexpr int kCBlocks = 4, kCRope = 16 * 1024, kCTile = 18 * 1024, kCStages = 2;
constexpr int kCScales = kCStages * kCTile, kCValues = kCScales + 4 * 256, kCUps = kCValues + 32 * 1024, kCLds = kCUps + kCW * 64;
static_assert(kCodesPerCu * (kCLds + 1024) <= 160 * 1024, "the workgroups of a CU share its LDS");
constexpr int kCCopies = 6;  // of a wave and tile: four latent blocks, rotary codes, scales
// log2 of the largest weight, or of the sum where that is larger: 60 at most and -10 at
// least after m moves, and by how much a weight may rise above that before it has to
constexpr float kCMost = 60.0f, kCLeast = 10.0f, kCRise = 30.0f;
// the largest product that f16 is to hold, and a little less than its log2
constexpr float kCTop = 61440.0f, kCTopLog = 15.9f;

// The lane, as if not known yet: what is worked out of it is worked out anew for
// each tile, since the products need the registers that it would be kept in.
__device__ __forceinline__ int lane_anew() {
    int l = threadIdx.x & 63;
    asm volatile("" : "+v"(l));
    return l;
}
// A column's 16 heads: queries as digits, 16 dims of a step of 64 in w[2 ks]
// (high) and w[2 ks + 1] (low).
struct CodesWave {
    pu32x4 w[18];
    float lat, rope;  // what a digit is worth in each part, times the scores' scale
    pf32x4 o[32];     // context^T: dim 16 mt + 4 (l >> 4) + i, column l & 15
    float m, l;       // offset (a whole number of log2 units) and sum
    bool ups;         // some column's up is not 0: all are in LDS, where they take no registers from the products
};
// The power of two that a column's products of weights and scales are taken times,
// of a wave's at U.
__device__ __forceinline__ __attribute__((address_space(3))) int *column_up(uint32_t U) {
    return (__attribute__((address_space(3))) int *)(U + (lane_anew() & 15) * 4);
}

// The rotary codes of row r, 64 bytes: chunks of 16 XORed with 0, 2, 3 and 1 for the
// rows 0 to 3, .. 12 to 15, so that the 16 lanes that a read takes at a time (0 to 3
// with 12 to 15 and 20 to 27, the others likewise) meet the LDS's 16 slots once.
__device__ __forceinline__ int rope_swz(int row) { return (0x78 >> ((row >> 1) & 6)) & 3; }

// Part [I0, I1) of the words, bf16, to digits; what a digit is worth.
template <int I0, int I1> __device__ __forceinline__ float query_digits(pu32x4 (&w)[18]) {
    typedef uint16_t u16x2 __attribute__((ext_vector_type(2)));
    u16x2 most = {0, 0};
#pragma unroll
    for (int i = I0; i < I1; i++)
#pragma unroll
        for (int k = 0; k < 4; k++) most = __builtin_elementwise_max(most, __builtin_bit_cast(u16x2, w[i][k] & 0x7fff7fffu));
    // bits of |q|: NaN lies above infinity
    uint32_t top = (uint32_t)(most[0] > most[1] ? most[0] : most[1]) << 16;
    auto r = __builtin_amdgcn_permlane32_swap(top, top, false, false);
    top = r[0] > r[1] ? r[0] : r[1];
    r = __builtin_amdgcn_permlane16_swap(top, top, false, false);
    top = r[0] > r[1] ? r[0] : r[1];
    const bool finite = top < 0x7f800000u, tiny = top > 0 && top < 0x10000000u;
    float m = __uint_as_float(top), down = 1.0f;
    // (the quotient stays in range: tiny queries are taken times 2^64, which changes no bit of them)
    if (__any(tiny)) {
        const float up = tiny ? 0x1p64f : 1.0f;
        m *= up;
        down = tiny ? 0x1p-64f : 1.0f;
#pragma unroll
        for (int i = I0; i < I1; i++)
#pragma unroll
            for (int k = 0; k < 4; k++) {
                const uint32_t v = w[i][k];
                const uint32_t lo = __float_as_uint(__fmul_rn(__uint_as_float(v << 16), up));
                const uint32_t hi = __float_as_uint(__fmul_rn(__uint_as_float(v & 0xffff0000u), up));
                w[i][k] = (lo >> 16) | (hi & 0xffff0000u);
            }
    }
    const float f = finite && top > 0 ? 32512.0f / m : 0.0f;
    // 1.5 * 2^23 + 128 in front: the sum's low 16 bits are x + 128, x the nearest
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
                    const uint32_t v = w[i + h][k + e];
                    const uint32_t a = __float_as_uint(__builtin_fmaf(__uint_as_float(v << 16), f, kFront));
                    const uint32_t b = __float_as_uint(__builtin_fmaf(__uint_as_float(v & 0xffff0000u), f, kFront));
                    two[e] = __builtin_amdgcn_perm(b, a, 0x05040100u);
                }
                d[0][2 * h + k / 2] = __builtin_amdgcn_perm(two[1], two[0], 0x07050301u);
                d[1][2 * h + k / 2] = __builtin_amdgcn_perm(two[1], two[0], 0x06040200u) ^ 0x80808080u;
            }
#pragma unroll
        for (int h = 0; h < 2; h++) w[i + h] = pu32x4{d[h][0], d[h][1], d[h][2], d[h][3]};
    }
    return finite ? __fmul_rn(__fmul_rn(m, 1.0f / 32512.0f), down) : __uint_as_float(0x7fc00000u);
}

// A tile's latent codes (LDS address T) to f16 values (V), in blocks of 8 rows
// and 64 values that the transposing reads take; wave w: row block w.  A lane
// takes 16 codes of a row, which become two of a block's eight chunks of a row:
// those of odd blocks are XORed with one more, so that the eight lanes of a row
// write to different slots (with reads of 8 codes, in halves by turns, that met in
// slots, 512 prompt rows over 8192 positions take 3 % more).
//   f16(code) = (1024 + (code + 128)) - 1152, each step exact.
__device__ __forceinline__ void convert_tile(uint32_t T, uint32_t V, int w) {
    const pf16x2 off = {(_Float16)-1152.0f, (_Float16)-1152.0f};
    const int l = lane_anew(), row = l >> 3, in = (l & 7) ^ row;
    const uint32_t src = T + w * kCBlocks * 1024 + l * 16;
    const uint32_t dst = V + (w * 8 + (in >> 2)) * 1024 + row * 128 + (((2 * (in & 3)) ^ (in >> 2) ^ row) << 4);
    pu32x4 c[4];
#pragma unroll
    for (int i = 0; i < 4; i++) c[i] = lds_read<pu32x4>(src + i * 1024);
#pragma unroll
    for (int i = 0; i < 8; i++) {
        pu32x4 v;
#pragma unroll
        for (int k = 0; k < 4; k++)
            v[k] = __builtin_bit_cast(uint32_t, __builtin_bit_cast(pf16x2, __builtin_amdgcn_perm(0x64646464u, c[i >> 1][2 * (i & 1) + (k >> 1)] ^ 0x80808080u,
                                                                                                k & 1 ? 0x04030402u : 0x04010400u)) + off);
        *(__attribute__((address_space(3))) pu32x4 *)((dst ^ (i & 1 ? 16 : 0)) + (i >> 1) * 2 * 1024) = v;
    }
}

// A lane's scores t, less the offset m, of positions 4 g + i and 16 + 4 g + i of
// its column, and their latent scales s.  T: the codes, S: the scales.  The rotary
// parts of both halves of the tile, then the latent ones of one half after the
// other (all sums together would not fit the registers, and a reload would wait
// for the copies under way).
__device__ __forceinline__ void tile_scores(const CodesWave &x, uint32_t T, uint32_t S, float m, float (&t)[8], float (&s)[8]) {
    constexpr int kAhead = 2;
    const int l = lane_anew(), row = l & 15, g = l >> 4;
    const uint32_t ak = T + (row >> 3) * kCBlocks * 1024 + (row & 7) * 128 + ((g ^ tile_swz(row)) << 4);
    const uint32_t ar = T + kCRope + row * 64 + ((g ^ rope_swz(row)) << 4), as = S + 32 * g;
    const pi32x4 zero = {0, 0, 0, 0};
    pi32x4 k[18], h[2], d[2];
    pf32x4 v[2];  // a half's scales, latent and rotary by turns
    auto read = [&](int i) {
        if (i < 2) k[i] = lds_read<pi32x4>(ar + i * 1024);
        else k[i] = lds_read<pi32x4>((ak ^ ((i & 1) << 6)) + (((i - 2) & 7) >> 1) * 1024 + ((i - 2) >> 3) * 2 * kCBlocks * 1024);
    };
#pragma unroll
    for (int i = 0; i < kAhead; i++) read(i);
    __builtin_amdgcn_sched_barrier(0);
#pragma unroll
    for (int i = 0; i < 18; i++) {
        const int half = (i - 2) >> 3, q = i < 2 ? 16 : 2 * ((i - 2) & 7), to = i == 1;
        const pi32x4 qh = __builtin_bit_cast(pi32x4, x.w[q]), qd = __builtin_bit_cast(pi32x4, x.w[q + 1]);
        const bool first = i < 2 || i == 2 || i == 10;
        h[to] = __builtin_amdgcn_mfma_i32_16x16x64_i8(k[i], qh, first ? zero : h[to], 0, 0, 0);
        d[to] = __builtin_amdgcn_mfma_i32_16x16x64_i8(k[i], qd, first ? zero : d[to], 0, 0, 0);
        if (i + kAhead < 18) read(i + kAhead);
        if (i == 1)
#pragma unroll
            for (int e = 0; e < 8; e++) t[e] = __fmul_rn((float)((h[e >> 2][e & 3] << 8) + d[e >> 2][e & 3]), x.rope);
        if (i == 8 || i == 16)
#pragma unroll
            for (int e = 0; e < 2; e++) v[e] = lds_read<pf32x4>(as + half * 128 + e * 16);
        __builtin_amdgcn_sched_barrier(0);
        if (i == 9 || i == 17) {
#pragma unroll
            for (int e = 0; e < 4; e++) {
                const float lat = __fmul_rn((float)((h[0][e] << 8) + d[0][e]), x.lat);
                s[4 * half + e] = v[e >> 1][2 * (e & 1)];
                t[4 * half + e] = __builtin_fmaf(lat, s[4 * half + e], __builtin_fmaf(t[4 * half + e], v[e >> 1][2 * (e & 1) + 1], -m));
            }
            __builtin_amdgcn_sched_barrier(0);
        }
    }
}

// The weights of a tile's scores, each times its position's scale.  seen: the
// tile's visible positions; fresh: some column has met no score but -inf yet.  Codes
// are finite, so that what a row does not see of them needs no care.
__device__ __forceinline__ pf16x8 tile_weights(CodesWave &w, uint32_t U, uint32_t S, uint32_t seen, bool &fresh, float (&t)[8], float (&s)[8]) {
    const int g = lane_anew() >> 4;
    const uint32_t mine = seen >> (4 * g);
    auto hidden = [&](int i) { return !((mine >> ((i >> 2) * 16 + (i & 3))) & 1); };
    if (seen != ~0u)
#pragma unroll
        for (int i = 0; i < 8; i++)
            if (hidden(i)) {  // a hidden position's scale is any
                t[i] = -INFINITY;
                s[i] = 0.0f;
            }
    // (one that is out of range so has a weight below 2^-116 of the sum, or a product below 2^-24)
    auto times_up = [&]() {
        if (w.ups) {
            const int up = *column_up(U);
#pragma unroll
            for (int i = 0; i < 8; i++) s[i] = fminf(fmaxf(ldexpf(s[i], up), kLow), -kLow);
        }
    };
    times_up();
    float e[8];
#pragma unroll
    for (int i = 0; i < 8; i++) e[i] = __builtin_amdgcn_exp2f(t[i]);
    auto most = [](const float (&v)[8]) {
        return fmaxf(fmaxf(fmaxf(v[0], v[1]), fmaxf(v[2], v[3])), fmaxf(fmaxf(v[4], v[5]), fmaxf(v[6], v[7])));
    };
    float size = 0.0f;
#pragma unroll
    for (int i = 0; i < 8; i++) size = fmaxf(size, fabsf(__fmul_rn(e[i], s[i])));
    if (fresh || __any(size > kCTop || most(t) > kCMost + kCRise)) {
        int up0 = 0;
        if (w.ups) {  // the scales anew
            up0 = *column_up(U);
#pragma unroll
            for (int i = 0; i < 8; i += 2) {
                const pf32x4 v = lds_read<pf32x4>(S + 32 * g + (i >> 2) * 128 + (i & 2) * 8);
                s[i] = hidden(i) ? 0.0f : v[0];
                s[i + 1] = hidden(i + 1) ? 0.0f : v[2];
            }
        }
        // the largest product and weight, and the sum, less m; scales below f32's normal
        // numbers, and 0, count as the least of those: what is so put too low has 13 bits to spare
        float u = -INFINITY;
#pragma unroll
        for (int i = 0; i < 8; i++) u = fmaxf(u, t[i] + fmaxf(__builtin_amdgcn_logf(fabsf(s[i])), -126.0f));
        u = col_max(u);
        const float sum = col_sum(w.l), top = fmaxf(col_max(most(t)), __builtin_amdgcn_logf(sum));
        const bool none = sum == 0.0f, rise = none || u + (float)up0 > kCTopLog;
        const bool move = (rise || top > kCMost + kCRise) && fabsf(top) < INFINITY;
        // where products of size 1 are to lie, less m; the weights of size 1 beside them if that may be
        const float to = rise ? floorf(u - 10.0f) : -(float)up0;
        const float by = move ? fminf(fmaxf(to, floorf(top - kCMost)), floorf(top + kCLeast)) : 0.0f;
        const int up = move ? (int)(by - to) : up0;
        const float f = none ? 0.0f : __builtin_amdgcn_exp2f((float)(up - up0) - by);
#pragma unroll
        for (int mt = 0; mt < 32; mt++) w.o[mt] *= f;
        w.l = ldexpf(w.l, (int)-by);
        w.m += by;
        w.ups = __any(up != 0);
        if (w.ups) *column_up(U) = up;
        times_up();
#pragma unroll
        for (int i = 0; i < 8; i++) e[i] = __builtin_amdgcn_exp2f(t[i] - by);
        fresh = __any(top == -INFINITY);
    }
    w.l = __fadd_rn(w.l, __fadd_rn(__fadd_rn(__fadd_rn(e[0], e[1]), __fadd_rn(e[2], e[3])), __fadd_rn(__fadd_rn(e[4], e[5]), __fadd_rn(e[6], e[7]))));
    pf16x8 p;
#pragma unroll
    for (int i = 0; i < 8; i++) p[i] = (_Float16)__fmul_rn(e[i], s[i]);
    return p;
}

// The context's products with a tile's values at V.
__device__ __forceinline__ void tile_context(CodesWave &w, const pf16x8 &p, uint32_t V) {
    constexpr int kAhead = 4;
    const int l = lane_anew(), g = l >> 4, j = l & 15, r = 4 * g + (j >> 2);
    const uint32_t at = V + (r >> 3) * 8 * 1024 + (r & 7) * 128 + ((((j & 3) >> 1) ^ tile_swz(r)) << 4) + 8 * (j & 1);
    pu32x4 v[32];
    auto read = [&](int i) {
        const uint32_t b = (at ^ ((i & 3) << 5) ^ ((i & 4) << 2)) + (i >> 2) * 1024;
        v[i] = tr_read(b, b + 16 * 1024);
    };
#pragma unroll
    for (int i = 0; i < kAhead; i++) read(i);
    __builtin_amdgcn_sched_barrier(0);
#pragma unroll
    for (int i = 0; i < 32; i++) {
        w.o[i] = __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(pf16x8, v[i]), p, w.o[i], 0, 0, 0);
        if (i + kAhead < 32) read(i + kAhead);
        __builtin_amdgcn_sched_barrier(0);
    }
}

// Waits for this wave's LDS operations and all but its last `copies` copies, then
// for the workgroup's other waves.
template <int COPIES> __device__ __forceinline__ void meet() {
    __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
    // (lgkmcnt 0; vmcnt 63 where the copies do not matter)
    __builtin_amdgcn_s_waitcnt(COPIES < 0 ? 0xc07f : 0x0070 | COPIES);
    __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
    __builtin_amdgcn_s_barrier();
    __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
}

// A column group's queries (under(): what is to start behind their loads), and
// nothing summed up yet; only under() for a wave without one.
template <class B> __device__ __forceinline__ void load_queries(const PagedArgs &a, const Seg &q, bool active, CodesWave &w, B &&under) {
    if (!active) {
        under();
        return;
    }
    const int l = lane_anew(), h = q.h0 + (l & 15), g = l >> 4;
    const int64_t row = q.row + (h < a.H ? h : a.H - 1);
    const __bf16 *qa = (const __bf16 *)a.qabs + row * kPL, *qr = (const __bf16 *)a.qrope + row * (kPD - kPL);
#pragma unroll
    for (int i = 0; i < 18; i++) w.w[i] = *(const pu32x4 *)((i < 16 ? qa + 32 * (i & ~1) : qr) + 16 * g + 8 * (i & 1));
    under();
    const float c = a.scale * kLog2e;
    w.lat = __fmul_rn(query_digits<0, 16>(w.w), c);
    w.rope = __fmul_rn(query_digits<16, 18>(w.w), c);
    // whole, and here: not in the loop at their first use
#pragma unroll
    for (int i = 0; i < 18; i++) asm volatile("" : "+v"(w.w[i]));
    w.m = 0.0f;
    w.l = 0.0f;
    w.ups = false;
#pragma unroll
    for (int mt = 0; mt < 32; mt++) w.o[mt] = pf32x4{0.0f, 0.0f, 0.0f, 0.0f};
}
// A unit's context, or a range's part of it.
template <int KIND>
__device__ __forceinline__ void finish(const PagedMfmaArgs &p, const Range &rg, int r, int grp, bool active, const Seg &q, CodesWave &w, uint32_t U) {
    const PagedArgs &a = p.a;
    const float sum = col_sum(w.l);
    const int up = active && w.ups ? *column_up(U) : 0;
    const int l = lane_anew(), g = l >> 4, col = l & 15, h = q.h0 + col;
    if (active && ((KIND == kListed && p.whole) || (q.b0 == 0 && q.b1 == q.tiles))) {
        const float inv = sum == 0.0f ? 0.0f : 1.0f / sum;
        __bf16 *out = (__bf16 *)a.out + (q.row + h) * kPL + 4 * g;
        if (h < a.H)
#pragma unroll
            for (int mt = 0; mt < 32; mt++) {
                pbf16x4 v;
#pragma unroll
                for (int i = 0; i < 4; i++) v[i] = (__bf16)ldexpf(__fmul_rn(w.o[mt][i], inv), -up);  // (apart: both may be tiny)
                *(pbf16x4 *)(out + 16 * mt) = v;
            }
    } else if (active) {
        // a part's context in f16, which is 1/8 of what the output's own rounding to
        // bf16 may take, times a power of two of the column that puts the largest at
        // 2^13 to 2^14; what that leaves of its size, and the sum's, apart: the join
        // must not lose one to the other
        float top = 0.0f;
#pragma unroll
        for (int mt = 0; mt < 32; mt++)
#pragma unroll
            for (int i = 0; i < 4; i++) top = fmaxf(top, fabsf(w.o[mt][i]));
        top = col_max(top);
        const int e = (int)(__float_as_uint(top) >> 23) - 127, by = top > 0.0f && top < INFINITY ? (13 - e < 120 ? 13 - e : 120) : 0;
        const float f = ldexpf(1.0f, by);
        const int64_t slot = plan_slot(r, rg.s <= q.first) * p.groups + grp;
        pf16x4 *po = (pf16x4 *)p.part_o + slot * 128 * kCols + g * kCols + col;
#pragma unroll
        for (int mt = 0; mt < 32; mt++) {
            pf16x4 v;
#pragma unroll
            for (int i = 0; i < 4; i++) v[i] = (_Float16)__fmul_rn(w.o[mt][i], f);
            po[mt * 4 * kCols] = v;
        }
        const int z = __builtin_amdgcn_frexp_expf(sum);
        const float k = top == 0.0f ? kLow : w.m - (float)(by + up);
        if (g == 0) *(float4 *)(p.part_ml + (slot * kCols + col) * 4) = make_float4(sum == 0.0f ? kLow : w.m + (float)z, ldexpf(sum, -z), k, 0.0f);
    }
}

// As k_paged_mfma: a workgroup's waves have a column group each, over the same
// tiles.  While a tile is worked on the next one is on its way; the one after it
// takes its place as soon as its scores and values are made.
template <int KIND, bool OWN>
__global__ __launch_bounds__(kCW * 64, kCodesPerCu * kCW / 4) void k_paged_codes(PagedMfmaArgs p) {
    constexpr bool SPARSE = KIND == kListed;
    __shared__ __attribute__((aligned(1024))) uint8_t stage[kCLds];
    const PagedArgs &a = p.a;
    const int w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    int r, chunk;
    const int id = place<OWN>(p.chunks, r, chunk);
    // units without positions: zeros
    const int64_t vec = (int64_t)(SPARSE ? 1 : a.M) * a.H * kPL * 2 / 16;
    for (int u = id; u < p.units; u += gridDim.x)
        if (unit_tiles<KIND>(a, u) == 0)
            for (int64_t i = threadIdx.x; i < vec; i += kCW * 64) ((pu32x4 *)a.out)[u * vec + i] = pu32x4{0, 0, 0, 0};
    Range rg;
    if (r >= p.most || !find_range<KIND, kCW>(p, r, p.most > 1 && r == 0 && chunk == 0, rg)) return;
    const int grp = chunk * p.per + w;
    const bool active = w < p.per && grp < p.groups;
    const int gr = active ? grp : 0;
    const uint32_t stage0 = (uint32_t)(uintptr_t)(lds_u8 *)stage;
    const uint32_t ups0 = __builtin_amdgcn_readfirstlane(stage0 + kCUps + w * 64);
    CodesWave wv;
    bool bad = false;
    int32_t entry = 0;  // the next copy's, of this wave's eight rows
    auto copy = [&](const Seg &q, int32_t x) {
        const int l = lane_anew(), row = (l >> 3) & 7, row4 = (l >> 2) & 7, n = x - q.b0;
        const int32_t phys = plan_page(entry, a.n_pages, bad);
        const int32_t at = (phys << a.shift) + ((tile_at<KIND>(q.lk, x) + 8 * w) & ((1 << a.shift) - 1));
        const uint8_t *src = (const uint8_t *)uniform((int64_t)a.pages + (int64_t)at * kPD);
        const uint32_t T = stage0 + (n & 1) * kCTile;
        copy_blocks<0, 4>(row * kPD + (((l & 7) ^ tile_swz(row)) << 4), src, __builtin_amdgcn_readfirstlane(T + w * kCBlocks * 1024));
        if (l < 32) copy_block<0>(row4 * kPD + kPL + (((l & 3) ^ rope_swz(8 * w + row4)) << 4), src, __builtin_amdgcn_readfirstlane(T + kCRope + w * 512));
        if (l < 4) copy_block<0>(l * 16, (const uint8_t *)uniform((int64_t)(a.scales + at)), __builtin_amdgcn_readfirstlane(stage0 + kCScales + (n & 3) * 256 + w * 64));
    };
    auto entry_of = [&](const Seg &q, int32_t x) { return page_entry<KIND>(q.lk, page_of<KIND>(q.lk, tile_at<KIND>(q.lk, x) + 8 * w)); };
    auto start = [&](const Seg &q) {
        for (int32_t x = q.b0; x < q.b1 && x < q.b0 + kCStages; x++) {
            entry = entry_of(q, x);
            copy(q, x);
        }
        entry = entry_of(q, q.b0 + kCStages);
    };
    Walk<KIND, OWN> walk = walk_of<KIND, OWN>(p, rg, chunk);
    Seg q;
    if (!walk.next(p, rg, gr, q)) return;
    bool begun = false;
    while (true) {
        load_queries(a, q, active, wv, [&]() {
            if (!begun) start(q);
            begun = true;
        });
        bool fresh = true;
        for (int32_t x = q.b0; x < q.b1; x++) {
            const uint32_t n = x - q.b0, T = stage0 + (n & 1) * kCTile, V = stage0 + kCValues;
            const uint32_t seen = visible<KIND>(q.lk, tile_at<KIND>(q.lk, x), q.n);
            // tile x's copies have landed, and the values before it are not needed any more
            if (x + 1 < q.b1) meet<kCCopies>();
            else meet<0>();
            convert_tile(T, V, w);
            float t[8], s[8];
            const bool some = active && seen;
            if (some) tile_scores(wv, T, stage0 + kCScales + (n & 3) * 256, wv.m, t, s);
            meet<-1>();
            // the wave that is through with its scores goes first, so that the other of its SIMD
            // is at its own scores under these products (512 prompt rows over 8192 positions 1296
            // us without, 1222 with; at the scores 1276, at the context's products 1246)
            __builtin_amdgcn_s_setprio(1);
            if (x + kCStages < q.b1) {
                copy(q, x + kCStages);
                entry = entry_of(q, x + kCStages + 1);
            }
            if (some) tile_context(wv, tile_weights(wv, ups0, stage0 + kCScales + (n & 3) * 256, seen, fresh, t, s), V);
            __builtin_amdgcn_s_setprio(0);
        }
        __syncthreads();  // the stages may be filled again: with the next part's first tiles
        Seg nx;
        const bool more = walk.next(p, rg, gr, nx);
        if (more) start(nx);
        finish<KIND>(p, rg, r, grp, active, q, wv, ups0);
        if (!more) break;
        q = nx;
    }
    if (bad && (threadIdx.x & 63) == 0) *a.err = 1;
}

void launch_codes(ut_ctx *ctx, const PagedMfmaArgs &p, int kind, bool own, unsigned wgs) {
    with_kind(kind, own, [&](auto k, auto o) {
        hipLaunchKernelGGL((k_paged_codes<decltype(k)::value, decltype(o)::value>), dim3(wgs), dim3(kCW * 64), 0, ctx->stream, p);
    });
}

}  // namespace ut
