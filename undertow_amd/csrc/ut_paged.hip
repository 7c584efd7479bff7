// ut_paged.hip -- the paged MLA latent cache: appending a step's rows, the
// score that selects pages, and attention for any latent width.
#include "ut_paged.h"

namespace ut {

struct Bf16 {
    static constexpr int kPlanes = 1;
    typedef __bf16 q_t;
    typedef float code_t;
    __device__ static float value(const uint16_t *row, int D, int d) {
        return __uint_as_float((uint32_t)row[d] << 16);
    }
    // four values as a row holds them, and back
    __device__ static void store(const float (&x)[4], uint2 (&h)[1]) {
        __bf16 v[4];
#pragma unroll
        for (int i = 0; i < 4; i++) v[i] = (__bf16)x[i];
        h[0] = *(const uint2 *)v;
    }
    __device__ static float stored(const uint2 (&h)[1], int i) {
        const uint32_t w = i < 2 ? h[0].x : h[0].y;
        return __uint_as_float(i & 1 ? w & 0xffff0000u : w << 16);
    }
};
struct F16x2 {
    static constexpr int kPlanes = 2;
    typedef float q_t;
    typedef double code_t;
    __device__ static float value(const uint16_t *row, int D, int d) {
        const _Float16 *h = (const _Float16 *)row;
        return __fadd_rn((float)h[d], __fmul_rn((float)h[D + d], 1.0f / kF16x2Step));
    }
    __device__ static void store(const float (&x)[4], uint2 (&h)[2]) {
        _Float16 v[2][4];
#pragma unroll
        for (int i = 0; i < 4; i++) f16x2_split(x[i], v[0][i], v[1][i]);
        h[0] = *(const uint2 *)v[0];
        h[1] = *(const uint2 *)v[1];
    }
    __device__ static float stored(const uint2 (&h)[2], int i) {
        const _Float16 *hi = (const _Float16 *)&h[0], *lo = (const _Float16 *)&h[1];
        return __fadd_rn((float)hi[i], __fmul_rn((float)lo[i], 1.0f / kF16x2Step));
    }
};

// -------------------------------------------------------------- append ---
// A workgroup takes one page that a sequence's new rows fall into: it writes
// the new rows and, where summaries are kept, adds the page's rows up dim by
// dim in 64 bits (sums of values of 8 or 22 bits: exact but for extreme
// ranges), the older ones read back and the new ones as stored:
//   S_d = sum x_d, A = max_d |S_d|, code = rint(S_d 127 / A),
//   scale = A / (127 n)   (code * scale is the mean row to 1/254 of its max).
// A thread holds four dims of every fourth position.  Latency bounds it: the
// length, the table's entry and the rows are loads that follow on one another.
// 48 rows into pages of 64, summaries anew: 6.3 us (1.9 MB); 3 x 777 rows in
// f16x2 12.4 us (10.9 MB, 0.9 TB/s): some 40 pages are as many workgroups.
// 16 new rows of a thread under way at a time change nothing there; the dims
// cut over workgroups, sums and then codes in two launches, took 10.8 us, but
// the call 18.2 against 16.2.
template <class F>
__global__ __launch_bounds__(576) void k_paged_append(PagedArgs a, uint16_t *__restrict__ pages,
                                                      const float *__restrict__ latent,
                                                      const float *__restrict__ krot,
                                                      int8_t *__restrict__ mean,
                                                      float *__restrict__ mean_scale) {
    extern __shared__ double sum[];  // [4][D]
    __shared__ double red[16];
    const int b = blockIdx.y, tid = threadIdx.x, D = a.L + a.P, nq = D / 4;
    bool bad = false;
    const int32_t len = plan_len(((const_i32 *)a.lens)[b], (int64_t)a.max_pages << a.shift, bad);
    if (bad) {  // cut to the table's end, the new rows would take the place of older ones
        *a.err = 1;
        return;
    }
    const int32_t from = len > a.M ? len - a.M : 0;  // the first new position
    const int k = (from >> a.shift) + (int)blockIdx.x;
    const int32_t page = 1 << a.shift;
    const int64_t p0 = (int64_t)k << a.shift;
    if (p0 >= len) return;
    const int32_t phys = paged_phys(a, b, k, bad);
    if (bad) return;
    const int live = len - p0 < page ? (int)(len - p0) : page;
    const int first = from > p0 ? (int)(from - p0) : 0;  // the page's first new row
    const int64_t row16 = (int64_t)D * F::kPlanes;
    uint16_t *base = pages + ((int64_t)phys << a.shift) * row16;
    for (int u = tid; u < 4 * nq; u += blockDim.x) {
        const int s = u / nq, d = (u - s * nq) * 4;
        double t[4] = {0.0, 0.0, 0.0, 0.0};
        // kOld (kNew) rows at a time, so that as many loads are under way
        constexpr int kOld = 16, kNew = 8;
        if (mean)
            for (int o0 = s; o0 < first; o0 += 4 * kOld) {
                uint2 v[kOld][F::kPlanes];
#pragma unroll
                for (int k = 0; k < kOld; k++) {
                    const int o = o0 + 4 * k < first ? o0 + 4 * k : o0;
#pragma unroll
                    for (int i = 0; i < F::kPlanes; i++) v[k][i] = *(const uint2 *)(base + o * row16 + i * D + d);
                }
#pragma unroll
                for (int k = 0; k < kOld; k++)
                    if (o0 + 4 * k < first) {
#pragma unroll
                        for (int i = 0; i < 4; i++) t[i] += (double)F::stored(v[k], i);
                    }
            }
        const float *src = d < a.L ? latent + d : krot + (d - a.L);
        const int64_t width = d < a.L ? a.L : a.P, r0 = (int64_t)b * a.M + (p0 - (len - a.M));
        for (int o0 = first + ((s - first) & 3); o0 < live; o0 += 4 * kNew) {
            float4 v[kNew];
#pragma unroll
            for (int k = 0; k < kNew; k++) v[k] = *(const float4 *)(src + (r0 + (o0 + 4 * k < live ? o0 + 4 * k : o0)) * width);
#pragma unroll
            for (int k = 0; k < kNew; k++)
                if (o0 + 4 * k < live) {
                    const float x[4] = {v[k].x, v[k].y, v[k].z, v[k].w};
                    uint2 h[F::kPlanes];
                    F::store(x, h);
#pragma unroll
                    for (int i = 0; i < F::kPlanes; i++) *(uint2 *)(base + (o0 + 4 * k) * row16 + i * D + d) = h[i];
#pragma unroll
                    for (int i = 0; i < 4; i++) t[i] += (double)F::stored(h, i);
                }
        }
        if (mean)
#pragma unroll
            for (int i = 0; i < 4; i++) sum[s * D + d + i] = t[i];
    }
    if (!mean) return;
    __syncthreads();
    double top = 0.0;
    for (int d = tid; d < D; d += blockDim.x) {
        const double t = (sum[d] + sum[D + d]) + (sum[2 * D + d] + sum[3 * D + d]);
        sum[d] = t;
        top = fmax(top, fabs(t));
    }
    for (int off = 32; off >= 1; off >>= 1) top = fmax(top, __shfl_xor(top, off, 64));
    if ((tid & 63) == 0) red[tid >> 6] = top;
    __syncthreads();
    for (int w = 0; w < (int)(blockDim.x >> 6); w++) top = fmax(top, red[w]);
    for (int d = tid; d < D; d += blockDim.x) {
        const double c = top > 0.0 ? rint(sum[d] * 127.0 / top) : 0.0;
        mean[(int64_t)phys * D + d] = (int8_t)(c >= -127.0 && c <= 127.0 ? (int)c : 0);
    }
    if (tid == 0) mean_scale[phys] = (float)(top / (127.0 * live));
}

// ----------------------------------------------------------- attention ---
// Any latent width and page, in f32: a workgroup takes four heads of one row
// and a slice of its positions, 64 at a time.  Scores: four lanes to a
// position, which is read once for the four heads; then a wave to a head for
// the maximum and the weights (one exponential each); context: a lane to a
// dim, or 2 or 4 of them with part of the positions each where the latent has
// at most 128 or 64 (with one, 3 lanes of 4 would idle at 64).  Only visible
// positions are read.
//
// The chains of dependent loads bound it, not bytes: so a row is cut into
// slices until four workgroups a CU run, and k_paged_generic_join joins them.
// 1 row of 4 heads over 1459 positions of 64 + 16 takes 22 us a call, and
// 337 with a whole row to a workgroup; 50 x 4 such rows in f16x2 48 and 431.
constexpr int kGenChunk = 64, kGenHeads = 4, kGenSlices = 32;
constexpr float kGenLow = -3.402823466e38f;  // the maximum before any score

// Virtual positions of a row and how they are cut.
struct GenCut {
    int64_t total;
    int32_t chunks, per;  // chunks of a slice
};
__device__ __forceinline__ GenCut gen_cut(const PagedArgs &a, int32_t n, int slices) {
    GenCut c;
    c.total = n <= 0 ? 0 : a.sel ? (int64_t)a.top_k << a.shift : n;
    c.chunks = (int32_t)((c.total + kGenChunk - 1) / kGenChunk);
    c.per = (c.chunks + slices - 1) / slices;
    return c;
}

// part_ml [row][head][slice][2], part_o [row][head][slice][L]
template <class F>
__global__ __launch_bounds__(256) void k_paged_generic(PagedArgs a, int slices, float *__restrict__ part_ml,
                                                       float *__restrict__ part_o) {
    extern __shared__ float sm[];
    constexpr int HG = kGenHeads;
    const int h0 = blockIdx.x * HG, j = blockIdx.y / slices, sl = blockIdx.y - j * slices, b = blockIdx.z;
    const int tid = threadIdx.x, w = tid >> 6, lane = tid & 63, D = a.L + a.P;
    float *q = sm;                                     // [HG][D], then the lanes' contexts
    __shared__ alignas(16) float p[kGenChunk][HG];
    __shared__ float s_m[HG], s_f[HG];
    __shared__ int64_t at[kGenChunk];
    const int64_t r = (int64_t)b * a.M + j;
    const int32_t n = paged_len(a, b) - a.M + j + 1;
    const GenCut cut = gen_cut(a, n, slices);
    const int32_t c0 = sl * cut.per, c1 = c0 + cut.per < cut.chunks ? c0 + cut.per : cut.chunks;
    if (sl > 0 && c0 >= c1) return;  // slice 0 writes a row without positions
    for (int i = tid; i < HG * D; i += 256) {
        const int h = h0 + i / D < a.H ? h0 + i / D : a.H - 1, d = i % D;
        q[i] = d < a.L ? (float)((const typename F::q_t *)a.qabs)[(r * a.H + h) * a.L + d]
                       : (float)((const typename F::q_t *)a.qrope)[(r * a.H + h) * a.P + (d - a.L)];
    }
    // lanes of a dim: `ways`, over positions way, way + ways, ..
    const int ways = a.L <= 64 ? 4 : a.L <= 128 ? 2 : 1, width = 256 / ways, way = tid / width, d0 = tid - way * width;
    float o[HG][4];
#pragma unroll
    for (int h = 0; h < HG; h++)
#pragma unroll
        for (int i = 0; i < 4; i++) o[h][i] = 0.0f;
    float m = kGenLow, l = 0.0f;  // wave w: of head w
    const int64_t row16 = (int64_t)D * F::kPlanes;
    for (int32_t c = c0; c < c1; c++) {
        if (tid < kGenChunk) {
            const int64_t t = (int64_t)c * kGenChunk + tid;
            int64_t row = -1;
            if (t < cut.total) {
                int64_t k = t >> a.shift;
                if (a.sel) k = a.sel[r * a.top_k + k];
                const int64_t in = t & ((1 << a.shift) - 1);
                if (k >= 0 && (k << a.shift) + in < n) row = ((int64_t)paged_phys(a, b, (int)k) << a.shift) + in;
            }
            at[tid] = row;
        }
        __syncthreads();
        {
            const int t = tid >> 2, s = tid & 3;
            float acc[HG] = {0.0f, 0.0f, 0.0f, 0.0f};
            if (at[t] >= 0) {
                const uint16_t *src = (const uint16_t *)a.pages + at[t] * row16;
#pragma unroll 4
                for (int d = 4 * s; d < D; d += 16) {
                    uint2 v[F::kPlanes];
#pragma unroll
                    for (int i = 0; i < F::kPlanes; i++) v[i] = *(const uint2 *)(src + i * D + d);
#pragma unroll
                    for (int h = 0; h < HG; h++) {
                        const float4 x = *(const float4 *)(q + h * D + d);
                        acc[h] = __builtin_fmaf(x.x, F::stored(v, 0), acc[h]);
                        acc[h] = __builtin_fmaf(x.y, F::stored(v, 1), acc[h]);
                        acc[h] = __builtin_fmaf(x.z, F::stored(v, 2), acc[h]);
                        acc[h] = __builtin_fmaf(x.w, F::stored(v, 3), acc[h]);
                    }
                }
            }
#pragma unroll
            for (int h = 0; h < HG; h++) {
                acc[h] += __shfl_xor(acc[h], 1, 64);
                acc[h] += __shfl_xor(acc[h], 2, 64);
            }
            p[t][s] = s == 0 ? acc[0] : s == 1 ? acc[1] : s == 2 ? acc[2] : acc[3];
        }
        __syncthreads();
        {
            // a maximum that skips NaN; the weight of a NaN score is NaN
            const bool live = at[lane] >= 0;
            const float v = live ? __fmul_rn(p[lane][w], a.scale) : -INFINITY;
            float top = v;
            for (int off = 32; off >= 1; off >>= 1) top = fmaxf(top, __shfl_xor(top, off, 64));
            const float mn = fmaxf(m, top), f = expf(m - mn), e = live ? expf(v - mn) : 0.0f;
            float sum = e;
            for (int off = 32; off >= 1; off >>= 1) sum += __shfl_xor(sum, off, 64);
            l = l * f + sum;
            m = mn;
            p[lane][w] = e;
            if (lane == 0) s_f[w] = f;
        }
        __syncthreads();
        float f[HG];
#pragma unroll
        for (int h = 0; h < HG; h++) f[h] = s_f[h];
#pragma unroll
        for (int i = 0; i < 4; i++) {
            const int d = d0 + width * i;
            if (d >= a.L) break;
            float x[HG];
#pragma unroll
            for (int h = 0; h < HG; h++) x[h] = o[h][i] * f[h];
#pragma unroll 8
            for (int t = way; t < kGenChunk; t += ways)
                if (at[t] >= 0) {
                    const float v = F::value((const uint16_t *)a.pages + at[t] * row16, D, d);
                    const float4 e = *(const float4 *)p[t];
                    x[0] = __builtin_fmaf(e.x, v, x[0]);
                    x[1] = __builtin_fmaf(e.y, v, x[1]);
                    x[2] = __builtin_fmaf(e.z, v, x[2]);
                    x[3] = __builtin_fmaf(e.w, v, x[3]);
                }
#pragma unroll
            for (int h = 0; h < HG; h++) o[h][i] = x[h];
        }
        __syncthreads();
    }
    if (lane == 0) {
        s_m[w] = m;
        s_f[w] = l;
    }
    if (ways > 1) {  // the lanes of a dim: one dim each (i = 0)
        __syncthreads();
#pragma unroll
        for (int h = 0; h < HG; h++) sm[h * 256 + tid] = o[h][0];
        __syncthreads();
        if (way == 0)
#pragma unroll
            for (int h = 0; h < HG; h++)
                for (int y = 1; y < ways; y++) o[h][0] += sm[h * 256 + y * width + d0];
    }
    __syncthreads();
#pragma unroll
    for (int h = 0; h < HG; h++) {
        if (h0 + h >= a.H) break;
        const int64_t rh = r * a.H + h0 + h;
        const float sum = s_f[h], inv = sum != 0.0f ? 1.0f / sum : 0.0f;
        if (slices > 1 && tid == 0) {
            part_ml[(rh * slices + sl) * 2] = s_m[h];
            part_ml[(rh * slices + sl) * 2 + 1] = sum;
        }
#pragma unroll
        for (int i = 0; i < 4; i++) {
            const int d = d0 + width * i;
            if (way > 0 || d >= a.L) break;
            if (slices > 1) part_o[(rh * slices + sl) * a.L + d] = o[h][i];
            else ((typename F::q_t *)a.out)[rh * a.L + d] = (typename F::q_t)(o[h][i] * inv);
        }
    }
}

// out = sum_s o_s e^(m_s - M) / sum_s l_s e^(m_s - M) over a row's slices.
template <class F>
__global__ __launch_bounds__(256) void k_paged_generic_join(PagedArgs a, int slices, const float *__restrict__ part_ml,
                                                            const float *__restrict__ part_o) {
    const int64_t rh = blockIdx.x;
    const int row = (int)(rh / a.H), b = row / a.M;
    const GenCut cut = gen_cut(a, paged_len(a, b) - a.M + (row - b * a.M) + 1, slices);
    const int used = cut.chunks > 0 ? (cut.chunks + cut.per - 1) / cut.per : 1;
    float M = kGenLow, sum = 0.0f, w[kGenSlices];
#pragma unroll
    for (int s = 0; s < kGenSlices; s++)
        if (s < used) M = fmaxf(M, part_ml[(rh * slices + s) * 2]);
#pragma unroll
    for (int s = 0; s < kGenSlices; s++)
        if (s < used) {
            w[s] = expf(part_ml[(rh * slices + s) * 2] - M);
            sum = __builtin_fmaf(part_ml[(rh * slices + s) * 2 + 1], w[s], sum);
        }
    const float inv = sum != 0.0f ? 1.0f / sum : 0.0f;
    for (int d = threadIdx.x; d < a.L; d += 256) {
        float v = 0.0f;
#pragma unroll
        for (int s = 0; s < kGenSlices; s++)
            if (s < used) v = __builtin_fmaf(part_o[(rh * slices + s) * a.L + d], w[s], v);
        ((typename F::q_t *)a.out)[rh * a.L + d] = (typename F::q_t)(v * inv);
    }
}

// -------------------------------------------------------------- select ---
// A head's query in 8 bits: code = rint(q 127 / max|q|) of the real quotient;
// its share of a score is weight max|q| / 127.  A head with a value that is
// not finite has none.  c = rint(q (127 / max)) may miss by one next to a
// half; q 127 - c max is exact and tells: a bf16 query's numbers fit f32 (15
// bits), a f32 one's take 64 bits.
constexpr int kCodeStep = 64;
__host__ __device__ inline int64_t code_row(int64_t D) { return (D + kCodeStep - 1) / kCodeStep * kCodeStep; }
__device__ __forceinline__ float exact_fma(float x, float y, float z) { return __builtin_fmaf(x, y, z); }
__device__ __forceinline__ double exact_fma(double x, double y, double z) { return __builtin_fma(x, y, z); }
template <class T> __device__ __forceinline__ int code8(T q, T top, T f) {
    const T c = rint(q * f), e = exact_fma(c, -2 * top, q * 254);  // twice the rest
    const int k = (int)c;
    const bool next = e > top || -e > top || ((e == top || -e == top) && (k & 1));
    return next ? (e > 0 ? k + 1 : k - 1) : k;
}
// Head r's query (none from `end` on), over a wave: eight dims a lane, a
// single one behind them, and (D is at most 1024) up to seven more, which are
// read where they are used.
template <class F> struct HeadQuery {
    typedef typename F::q_t q_t;
    typedef q_t q8 __attribute__((ext_vector_type(8)));
    const q_t *qa, *qr;
    q8 q;
    q_t one;
    float weight;
    bool any;
    __device__ __forceinline__ HeadQuery(const PagedArgs &a, int64_t r, int64_t end, const float *weights) {
        const int lane = threadIdx.x & 63, D = a.L + a.P;
        any = r < end;
        if (!any) r = end - 1;
        qa = (const q_t *)a.qabs + r * a.L;
        qr = (const q_t *)a.qrope + r * a.P;
        q = q8{0, 0, 0, 0, 0, 0, 0, 0};
        if (8 * lane < D) q = *(const q8 *)(8 * lane < a.L ? qa + 8 * lane : qr + (8 * lane - a.L));
        one = 0;
        if (512 + lane < D) one = 512 + lane < a.L ? qa[512 + lane] : qr[512 + lane - a.L];
        weight = weights ? weights[r] : 1.0f;
    }
};
// Its codes: code_row(D) bytes, zeros behind the D; its share.
template <class F>
__device__ __forceinline__ void head_codes(const PagedArgs &a, const HeadQuery<F> &x, int8_t *codes, double *share) {
    const int lane = threadIdx.x & 63, D = a.L + a.P, Dp = (int)code_row(D);
    typedef typename F::code_t T;
    auto at = [&](int d) { return (float)(d < a.L ? x.qa[d] : x.qr[d - a.L]); };
    auto bits = [](float x) { return __float_as_uint(x) & 0x7fffffffu; };  // NaN lies above infinity
    const auto q = x.q;
    const float one = (float)x.one, weight = x.weight;
    const bool any = x.any;
    uint32_t top = bits(one);
#pragma unroll
    for (int k = 0; k < 8; k++) {
        const uint32_t v = bits((float)q[k]);
        top = v > top ? v : top;
    }
#pragma unroll 1
    for (int d = 576 + lane; d < D; d += 64) {
        const uint32_t v = bits(at(d));
        top = v > top ? v : top;
    }
    for (int off = 32; off >= 1; off >>= 1) {
        const uint32_t v = __shfl_xor(top, off, 64);
        top = v > top ? v : top;
    }
    const bool live = any && top > 0 && top < 0x7f800000u;
    const float m = __uint_as_float(top);
    // a power of two keeps the numbers within f32's normal range
    const T up = m < 1e-30f ? (T)0x1p90f : m > 1e30f ? (T)0x1p-30f : (T)1, mt = (T)m * up, f = live ? (T)127 / mt : (T)0;
    auto code = [&](float x) { return live ? code8<T>((T)x * up, mt, f) : 0; };
    uint32_t c[2] = {0, 0};
#pragma unroll
    for (int k = 0; k < 8; k++) c[k >> 2] |= (uint32_t)(code((float)q[k]) & 255) << (8 * (k & 3));
    if (8 * lane < Dp) *(uint2 *)(codes + 8 * lane) = make_uint2(c[0], c[1]);
    if (512 + lane < Dp) codes[512 + lane] = (int8_t)code(one);
#pragma unroll 1
    for (int d = 576 + lane; d < Dp; d += 64) codes[d] = d < D ? (int8_t)code(at(d)) : 0;
    if (lane == 0) *share = live ? (double)weight * ((double)m / 127.0) : 0.0;
}

// A score's order as an unsigned number; NaN below everything.
__device__ __forceinline__ uint64_t score_key(double s) {
    if (!(s == s)) return 0;
    const uint64_t u = (uint64_t)__double_as_longlong(s + 0.0);  // -0 counts as 0
    return u >> 63 ? ~u : u | (1ull << 63);
}
template <int CTRL> __device__ __forceinline__ double dpp_double(double v) {
    const uint64_t u = (uint64_t)__double_as_longlong(v);
    const uint32_t lo = __builtin_amdgcn_update_dpp(0u, (uint32_t)u, CTRL, 0xf, 0xf, true);
    const uint32_t hi = __builtin_amdgcn_update_dpp(0u, (uint32_t)(u >> 32), CTRL, 0xf, 0xf, true);
    return __longlong_as_double((long long)((uint64_t)hi << 32 | lo));
}

// score = (sum_h share_h max(0, code_h . mean)) mean_scale; the products are
// v_mfma_i32_16x16x64_i8 (pages x heads, exact), the sums over heads run in 64
// bits in an order that is the same for every page.  Two ways to the sums:
//
// many rows: a launch makes all codes; then a workgroup takes 32 pages of a
// row, its waves every fourth tile of 16 heads, so that a page's mean is read
// once for all heads (48 rows of up to 625 pages: 27.3 us a call, with 16 pages
// 28.5, with 64 29.8);
// few rows (and rows of nine whole steps of 64): one launch, a workgroup takes
// 16 heads, whose codes its waves make first, and 256 pages or more, and
// leaves its heads' part of each sum.
// The one launch reads the means again for every 16 heads.  Whole calls over
// 512 pages, 128 heads: one row 14.4 us (two launches 16.4), 8 rows 15.0
// (16.5), 16 rows 15.3 (17.3), 48 rows 28.3 (26.2); 32 rows of 64 heads 16.5
// (19.2).  So one launch up to as many tiles of 16 heads as CUs.
typedef int si32x4 __attribute__((ext_vector_type(4)));
// The sum over a row of 16 lanes, in all of them: lanes ^ 1, ^ 2, then each
// eight and sixteen mirrored (a quad agrees by then).
__device__ __forceinline__ double sum16(double v) {
    v += dpp_double<0xB1>(v);   // quad_perm [1, 0, 3, 2]
    v += dpp_double<0x4E>(v);   // quad_perm [2, 3, 0, 1]
    v += dpp_double<0x141>(v);  // row_half_mirror
    v += dpp_double<0x140>(v);  // row_mirror
    return v;
}

template <class F>
__global__ __launch_bounds__(256) void k_select_codes(PagedArgs a, const float *__restrict__ weights, int64_t r0,
                                                      int64_t heads, int8_t *__restrict__ codes,
                                                      double *__restrict__ share) {
    const int64_t i = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6);
    if (i < heads) head_codes<F>(a, HeadQuery<F>(a, r0 + i, r0 + heads, weights), codes + i * code_row(a.L + a.P), share + i);
}

constexpr int kScorePages = 32, kScoreTiles = kScorePages / 16;
template <bool FULL>
__global__ __launch_bounds__(256) void k_select_score(PagedArgs a, const int8_t *__restrict__ codes,
                                                      const double *__restrict__ share,
                                                      const int8_t *__restrict__ mean, int row0,
                                                      double *__restrict__ part) {
    constexpr int STEPS = FULL ? 9 : 16;  // at most 1024 dims
    __shared__ double wave_part[4][kScorePages];
    const int row = row0 + blockIdx.y, b = row / a.M, j = row - b * a.M;
    const int w = threadIdx.x >> 6, l = threadIdx.x & 63, g = l >> 4;
    const int D = a.L + a.P, Dp = (int)code_row(D), steps = Dp / kCodeStep;
    const int32_t n = paged_len(a, b) - a.M + j + 1;
    const int np = n > 0 ? ((n - 1) >> a.shift) + 1 : 0, k0 = blockIdx.x * kScorePages;
    if (k0 >= np) return;
    // a tile of heads is loaded under the products of the one before, the first
    // beside the look-ups of the pages
    si32x4 B[STEPS];
    double sh = 0.0;
    auto load = [&](int h0) {
        const int h = h0 + (l & 15);
        const int64_t r = (int64_t)blockIdx.y * a.H + (h < a.H ? h : a.H - 1);
        sh = h < a.H ? share[r] : 0.0;
#pragma unroll
        for (int s = 0; s < STEPS; s++)
            if (FULL || s < steps) B[s] = *(const si32x4 *)(codes + r * Dp + kCodeStep * s + 16 * g);
    };
    if (16 * w < a.H) load(16 * w);
    si32x4 A[kScoreTiles][STEPS];
#pragma unroll
    for (int t = 0; t < kScoreTiles; t++) {
        const int k = k0 + 16 * t + (l & 15);
        const int8_t *src = mean + (int64_t)paged_phys(a, b, k < np ? k : np - 1) * D;
#pragma unroll
        for (int s = 0; s < STEPS; s++) {
            const int d = kCodeStep * s + 16 * g;
            if (FULL) {
                A[t][s] = *(const si32x4 *)(src + d);
            } else {  // rows of a multiple of 8 bytes, zeros behind them
                const int2 z = make_int2(0, 0), x = d + 8 <= D ? *(const int2 *)(src + d) : z;
                const int2 y = d + 16 <= D ? *(const int2 *)(src + d + 8) : z;
                A[t][s] = si32x4{x.x, x.y, y.x, y.y};
            }
        }
    }
    double sum[4 * kScoreTiles] = {};
    for (int h0 = 16 * w; h0 < a.H; h0 += 64) {
        si32x4 c[kScoreTiles] = {};
        const double share_h = sh;
#pragma unroll
        for (int s = 0; s < STEPS; s++)
            if (FULL || s < steps)
#pragma unroll
                for (int t = 0; t < kScoreTiles; t++)
                    c[t] = __builtin_amdgcn_mfma_i32_16x16x64_i8(A[t][s], B[s], c[t], 0, 0, 0);
        if (h0 + 64 < a.H) load(h0 + 64);
#pragma unroll
        for (int i = 0; i < 4 * kScoreTiles; i++) {
            const int v = c[i >> 2][i & 3];
            sum[i] += share_h * (double)(v > 0 ? v : 0);
        }
    }
    // lane l: pages 16 (i >> 2) + 4 g + (i & 3) for its head column
#pragma unroll
    for (int i = 0; i < 4 * kScoreTiles; i++) sum[i] = sum16(sum[i]);
    if ((l & 15) == 0)
#pragma unroll
        for (int i = 0; i < 4 * kScoreTiles; i++) wave_part[w][16 * (i >> 2) + 4 * g + (i & 3)] = sum[i];
    __syncthreads();
    const int t = threadIdx.x;
    if (t < kScorePages && k0 + t < np)
        part[(int64_t)blockIdx.y * a.max_pages + k0 + t] = (wave_part[0][t] + wave_part[1][t]) + (wave_part[2][t] + wave_part[3][t]);
}

constexpr int kFusedHeads = 16, kFusedThreads = 64 * kFusedHeads, kFusedPages = 16 * kFusedHeads;
template <class F>
__global__ __launch_bounds__(kFusedThreads) void k_select_fused(PagedArgs a, const float *__restrict__ weights,
                                                                const int8_t *__restrict__ mean, int row0,
                                                                double *__restrict__ part) {
    constexpr int STEPS = 9, D = STEPS * kCodeStep;
    __shared__ __attribute__((aligned(16))) int8_t codes[kFusedHeads][D + 16];  // 16 bytes more: other banks
    __shared__ double share[kFusedHeads];
    const int row = row0 + blockIdx.z, b = row / a.M, j = row - b * a.M, h0 = blockIdx.y * kFusedHeads;
    const int w = threadIdx.x >> 6, l = threadIdx.x & 63, g = l >> 4;
    // the query is read beside the length and the table
    const HeadQuery<F> query(a, (int64_t)row * a.H + h0 + w, (int64_t)(row + 1) * a.H, weights);
    const int32_t n = paged_len(a, b) - a.M + j + 1;
    const int np = n > 0 ? ((n - 1) >> a.shift) + 1 : 0;
    if ((int)blockIdx.x * kFusedPages >= np) return;
    // a wave's 16 pages: their means come in while the codes are made
    const int k0 = blockIdx.x * kFusedPages + 16 * w, k = k0 + (l & 15);
    const int8_t *src = mean + (int64_t)paged_phys(a, b, k < np ? k : np - 1) * D;
    si32x4 A[STEPS];
#pragma unroll
    for (int s = 0; s < STEPS; s++) A[s] = *(const si32x4 *)(src + kCodeStep * s + 16 * g);
    head_codes<F>(a, query, codes[w], &share[w]);
    __syncthreads();
    si32x4 c = {0, 0, 0, 0};
#pragma unroll
    for (int s = 0; s < STEPS; s++)
        c = __builtin_amdgcn_mfma_i32_16x16x64_i8(A[s], *(const si32x4 *)&codes[l & 15][kCodeStep * s + 16 * g], c, 0, 0, 0);
    const double sh = share[l & 15];
    double sum[4];
#pragma unroll
    for (int i = 0; i < 4; i++) sum[i] = sum16(sh * (double)(c[i] > 0 ? c[i] : 0));
    const int i = l & 3;  // lane l: pages 4 g + i
    const double mine = i == 0 ? sum[0] : i == 1 ? sum[1] : i == 2 ? sum[2] : sum[3];
    if ((l & 15) < 4 && k0 + 4 * g + i < np)
        part[((int64_t)blockIdx.z * gridDim.y + blockIdx.y) * a.max_pages + k0 + 4 * g + i] = mine;
}

// The top_k pages of a row: the first keep_first, the last keep_last, then by
// score, ties to the lower page; ascending, -1 behind them.  A workgroup per
// row adds the head groups' parts to the scores' keys and looks for the key of
// the last page to be taken: keys between the least and the largest that are
// left fall into 256 bins by the first eight bits in which those two differ;
// the bin that holds the one sought is looked into further, until its keys are
// equal or at most 64, which one wave then ranks.  One more pass writes the
// pages above that key and the first of those equal to it.  Passes over a few
// hundred keys, each a barrier apart: 512 pages 6.2 us, 48 rows of up to 625
// pages 8.0 (codes 9.0 and scores 11.7 before it).
constexpr int kPickThreads = 512;
__global__ __launch_bounds__(kPickThreads) void k_select_pick(PagedArgs a, const double *__restrict__ part,
                                                              int tiles, const float *__restrict__ mean_scale,
                                                              int row0, uint64_t *keys, int keep_first,
                                                              int keep_last, int32_t *__restrict__ out) {
    constexpr int NW = kPickThreads / 64;
    __shared__ int hist[256], few_n, s_bin, s_above;
    __shared__ uint64_t ends[2][NW], few[64], s_key;
    __shared__ int scan[2][NW];
    const int row = row0 + blockIdx.x, b = row / a.M, j = row - b * a.M, tid = threadIdx.x;
    const int lane = tid & 63, w = tid >> 6;
    const int32_t n = paged_len(a, b) - a.M + j + 1;
    const int np = n > 0 ? ((n - 1) >> a.shift) + 1 : 0;
    out += (int64_t)row * a.top_k;
    if (np <= a.top_k) {
        for (int i = tid; i < a.top_k; i += kPickThreads) out[i] = i < np ? i : -1;
        return;
    }
    // thread tid makes and reads the keys of pages tid, tid + kPickThreads, ..
    keys += (int64_t)blockIdx.x * a.max_pages;
    part += (int64_t)blockIdx.x * tiles * a.max_pages;
    for (int k = tid; k < np; k += kPickThreads) {
        const float scale = mean_scale[paged_phys(a, b, k)];
        double t = 0.0;
#pragma unroll 8
        for (int i = 0; i < tiles; i++) t += part[(int64_t)i * a.max_pages + k];
        keys[k] = score_key(t * (double)scale);
    }
    const int kept = keep_first + keep_last;  // of np > top_k >= kept pages
    auto scored = [&](int k) { return k >= keep_first && k < np - keep_last; };
    int need = a.top_k - kept;  // of the scored pages
    uint64_t cut = ~0ull;       // pages of larger keys are taken, of equal ones `need`
    if (need > 0) {
        // the keys in question: lo <= key <= hi, `need` of them from above
        uint64_t lo = 0, hi = ~0ull;
        for (;;) {
            uint64_t mn = ~0ull, mx = 0;
            for (int k = tid; k < np; k += kPickThreads)
                if (scored(k)) {
                    const uint64_t v = keys[k];
                    if (v >= lo && v <= hi) {
                        mn = v < mn ? v : mn;
                        mx = v > mx ? v : mx;
                    }
                }
            for (int off = 32; off >= 1; off >>= 1) {
                const uint64_t x = __shfl_xor(mn, off, 64), y = __shfl_xor(mx, off, 64);
                mn = x < mn ? x : mn;
                mx = y > mx ? y : mx;
            }
            if (lane == 0) {
                ends[0][w] = mn;
                ends[1][w] = mx;
            }
            if (tid < 256) hist[tid] = 0;
            if (tid == 0) few_n = 0;
            __syncthreads();
            for (int i = 0; i < NW; i++) {
                mn = ends[0][i] < mn ? ends[0][i] : mn;
                mx = ends[1][i] > mx ? ends[1][i] : mx;
            }
            if (mn == mx) {
                cut = mn;
                break;
            }
            // the highest bit that differs is the bins' highest
            const int top = 63 - __builtin_clzll(mn ^ mx), sh = top > 7 ? top - 7 : 0;
            const uint64_t base = mn >> sh & ~255ull;
            for (int k = tid; k < np; k += kPickThreads)
                if (scored(k)) {
                    const uint64_t v = keys[k];
                    if (v >= mn && v <= mx) atomicAdd(&hist[(int)((v >> sh) - base)], 1);
                }
            __syncthreads();
            if (w == 0) {
                // lane l: bins 255 - 4 l - [0, 4), summed from the top
                int c[4], s = 0;
#pragma unroll
                for (int i = 0; i < 4; i++) s += c[i] = hist[255 - 4 * lane - i];
                int x = s;
                for (int off = 1; off < 64; off <<= 1) {
                    const int y = __shfl_up(x, off, 64);
                    if (lane >= off) x += y;
                }
                int above = x - s;
                if (above < need && need <= x) {
                    int i = 0;
                    while (above + c[i] < need) above += c[i++];
                    s_bin = 255 - 4 * lane - i;
                    s_above = above;
                }
            }
            __syncthreads();
            need -= s_above;
            lo = (base + (uint64_t)s_bin) << sh;
            hi = lo | ((1ull << sh) - 1);
            const int left = hist[s_bin];
            if (left <= 64) {
                for (int k = tid; k < np; k += kPickThreads)
                    if (scored(k)) {
                        const uint64_t v = keys[k];
                        if (v >= lo && v <= hi) few[atomicAdd(&few_n, 1)] = v;
                    }
                __syncthreads();
                if (w == 0) {
                    const uint64_t v = lane < left ? few[lane] : 0;
                    int more = 0, same = 0;
                    for (int i = 0; i < left; i++) {
                        more += few[i] > v;
                        same += few[i] == v;
                    }
                    // the key that holds the place sought
                    if (lane < left && more < need && need <= more + same) {
                        s_key = v;
                        s_above = more;
                    }
                }
                __syncthreads();
                cut = s_key;
                need -= s_above;
                break;
            }
            __syncthreads();  // hist and few_n are set anew
        }
    }
    // of the pages equal to the cut `need` are taken, the lowest first
    int done = 0, equal = 0;
    for (int k0 = 0; k0 < np; k0 += kPickThreads) {
        const int k = k0 + tid;
        const bool in = k < np && scored(k);
        const uint64_t v = in ? keys[k] : 0;
        const bool eq = in && need > 0 && v == cut;
        const uint64_t be = __ballot(eq), before = (1ull << lane) - 1;
        __syncthreads();
        if (lane == 0) scan[0][w] = __popcll(be);
        __syncthreads();
        int e = equal + __popcll(be & before), te = equal;
        for (int i = 0; i < NW; i++) {
            if (i < w) e += scan[0][i];
            te += scan[0][i];
        }
        equal = te;
        const bool take = (k < np && !in) || (in && v > cut) || (eq && e < need);
        const uint64_t bt = __ballot(take);
        if (lane == 0) scan[1][w] = __popcll(bt);
        __syncthreads();
        int at = done + __popcll(bt & before), td = done;
        for (int i = 0; i < NW; i++) {
            if (i < w) at += scan[1][i];
            td += scan[1][i];
        }
        if (take) out[at] = k;
        done = td;
    }
}

// ------------------------------------------------------------ the calls ---
// The context's device while a call runs: its allocations and launches go
// there whichever device the caller has current.
struct DeviceScope {
    int before = -1;
    hipError_t err;
    explicit DeviceScope(int device) {
        int d = -1;
        err = hipGetDevice(&d);
        if (err == hipSuccess && d != device) {
            before = d;
            err = hipSetDevice(device);
        }
    }
    ~DeviceScope() {
        if (before >= 0) (void)hipSetDevice(before);
    }
};

constexpr int64_t kMostRows = 65535;         // query rows of a call
constexpr int64_t kMostGroups = 1ll << 22;   // workgroups along a grid's first axis, where pages set them
static int32_t paged_args(ut_ctx *ctx, const DeviceScope &dev, const char *what, const ut_mla_pages *kv,
                          const int32_t *table, int64_t stride, int64_t max_pages,
                          const int32_t *lens, int64_t B, int64_t M, int64_t H, int64_t most_rows,
                          PagedArgs &a) {
    auto bad = [&](const char *why) {
        set_error(ctx, "%s: %s", what, why);
        return UT_ERR_ARG;
    };
    if (!kv || !kv->pages || !table || !lens) return bad("null pointer");
    if (kv->fmt != UT_KV_BF16 && kv->fmt != UT_KV_F16X2) return bad("unknown cache format");
    if (kv->n_pages <= 0 || max_pages <= 0 || B <= 0 || M <= 0 || H <= 0 || stride < max_pages)
        return bad("sizes must be positive and the table's stride cover its pages");
    if (((uintptr_t)kv->pages & 15) != 0) return bad("pages must be 16-byte aligned");
    UT_CHECK_HIP(ctx, dev.err);
    const int64_t page = kv->page, L = kv->latent, P = kv->rope;
    auto shape = [&](const char *why) {
        set_error(ctx, "%s: %s (page %lld, latent %lld, rope %lld, sequences %lld, rows %lld, heads %lld)",
                  what, why, (long long)page, (long long)L, (long long)P, (long long)B, (long long)M,
                  (long long)H);
        return UT_ERR_SHAPE;
    };
    if (page < 1 || page > 1024 || (page & (page - 1)) != 0)
        return shape("a page is a power of two of at most 1024 positions");
    if (L <= 0 || P <= 0 || L % 8 != 0 || P % 8 != 0 || L + P > 1024)
        return shape("latent and rope must be multiples of 8 that add up to at most 1024");
    if (kv->n_pages > INT32_MAX / page || max_pages > kMostPositions / page)
        return shape("a pool holds fewer than 2^31 positions, a sequence at most 2^31 - 1024");
    if (B > 65535 || H > 65535 || M > INT32_MAX / B / H || B * M > most_rows)
        return shape("too many sequences, rows or heads");
    a = PagedArgs{};
    a.pages = kv->pages;
    a.table = table;
    a.stride = stride;
    a.lens = lens;
    UT_TRY(device_error_flag(ctx, &a.err));
    a.err += 1;  // the page word
    a.n_pages = (int32_t)kv->n_pages;
    a.max_pages = (int32_t)max_pages;
    a.shift = __builtin_ctzll((uint64_t)page);
    a.B = (int32_t)B;
    a.M = (int32_t)M;
    a.H = (int32_t)H;
    a.L = (int32_t)L;
    a.P = (int32_t)P;
    return UT_OK;
}

static int32_t launch_paged_generic(ut_ctx *ctx, const PagedArgs &a, int32_t fmt) {
    // slices: four workgroups a CU, partial results of 64 MB at most
    const int64_t groups = (a.H + kGenHeads - 1) / kGenHeads, R = (int64_t)a.B * a.M;
    const int64_t cap = (int64_t)(a.sel ? a.top_k : a.max_pages) << a.shift;
    int64_t slices = 4 * ctx->multiprocessors / (R * groups);
    const int64_t room = (int64_t(64) << 20) / (R * a.H * a.L * 4), chunks = (cap + kGenChunk - 1) / kGenChunk;
    slices = slices < room ? slices : room;
    slices = slices < chunks ? slices : chunks;
    slices = slices < 1 ? 1 : slices < kGenSlices ? slices : kGenSlices;
    float *ml = nullptr, *po = nullptr;
    if (slices > 1) {
        ScratchPlan plan;
        plan.add((size_t)(R * a.H * slices) * 8);
        plan.add((size_t)(R * a.H * slices * a.L) * 4);
        std::vector<void *> ptrs;
        UT_TRY(scratch_acquire(ctx, plan, ptrs));
        ml = (float *)ptrs[0];
        po = (float *)ptrs[1];
    }
    const size_t lds = (size_t)kGenHeads * (a.L + a.P < 256 ? 256 : a.L + a.P) * 4;
    int tok = timing_begin(ctx, "paged_generic");
    hipLaunchKernelGGL((fmt == UT_KV_BF16 ? k_paged_generic<Bf16> : k_paged_generic<F16x2>),
                       dim3((unsigned)groups, (unsigned)(a.M * slices), (unsigned)a.B), dim3(256), lds, ctx->stream, a,
                       (int)slices, ml, po);
    timing_end(ctx, tok);
    UT_TRY(launch_check(ctx, "k_paged_generic"));
    if (slices == 1) return UT_OK;
    tok = timing_begin(ctx, "paged_generic_join");
    hipLaunchKernelGGL((fmt == UT_KV_BF16 ? k_paged_generic_join<Bf16> : k_paged_generic_join<F16x2>),
                       dim3((unsigned)(R * a.H)), dim3(256), 0, ctx->stream, a, (int)slices, ml, po);
    timing_end(ctx, tok);
    return launch_check(ctx, "k_paged_generic_join");
}

static int32_t paged_attend(ut_ctx *ctx, const char *what, const ut_mla_pages *kv,
                            const int32_t *table, int64_t stride, int64_t max_pages,
                            const int32_t *lens, int64_t B, int64_t M, int64_t H, const void *qabs,
                            const void *qrope, float scale, const int32_t *sel, int64_t top_k,
                            void *out) {
    DeviceScope dev(ctx->device);
    PagedArgs a;
    UT_TRY(paged_args(ctx, dev, what, kv, table, stride, max_pages, lens, B, M, H, kMostRows, a));
    if (!qabs || !qrope || !out || ((uintptr_t)qabs & 15) != 0 || ((uintptr_t)qrope & 15) != 0 ||
        ((uintptr_t)out & 15) != 0) {
        set_error(ctx, "%s: queries and output must be 16-byte aligned device memory", what);
        return UT_ERR_ARG;
    }
    a.qabs = qabs;
    a.qrope = qrope;
    a.scale = scale;
    a.sel = sel;
    a.top_k = (int32_t)top_k;
    a.out = out;
    if (paged_mfma_ok(a)) return launch_paged_mfma(ctx, a, kv->fmt);
    return launch_paged_generic(ctx, a, kv->fmt);
}

}  // namespace ut

using namespace ut;

extern "C" int32_t ut_mla_paged_append(ut_ctx *ctx, const ut_mla_pages *kv,
                                       const int32_t *table_dev, int64_t table_stride,
                                       int64_t max_pages, const int32_t *lens_dev, int64_t batch,
                                       int64_t rows, const float *latent_dev,
                                       const float *krot_dev) {
    if (!ctx) return UT_ERR_ARG;
    DeviceScope dev(ctx->device);
    PagedArgs a;
    UT_TRY(paged_args(ctx, dev, "ut_mla_paged_append", kv, table_dev, table_stride, max_pages, lens_dev,
                      batch, rows, 1, INT32_MAX, a));
    if (!latent_dev || !krot_dev || ((uintptr_t)latent_dev & 15) != 0 ||
        ((uintptr_t)krot_dev & 15) != 0 || !kv->mean != !kv->mean_scale) {
        set_error(ctx, "ut_mla_paged_append: rows must be 16-byte aligned device memory, and mean "
                       "and mean_scale be given together");
        return UT_ERR_ARG;
    }
    // pages that `rows` positions can fall into
    const int64_t page = kv->page, touched = (rows + page - 2) / page + 1;
    if (touched > kMostGroups && max_pages > kMostGroups) {
        set_error(ctx, "ut_mla_paged_append: rows of more than %lld pages in a call", (long long)kMostGroups);
        return UT_ERR_SHAPE;
    }
    const size_t lds = kv->mean ? (size_t)(a.L + a.P) * 4 * sizeof(double) : 0;
    const dim3 grid((unsigned)(touched < max_pages ? touched : max_pages), (unsigned)batch);
    int tok = timing_begin(ctx, "paged_append");
    if (kv->fmt == UT_KV_BF16)
        hipLaunchKernelGGL(k_paged_append<Bf16>, grid, dim3(576), lds, ctx->stream, a,
                           (uint16_t *)kv->pages, latent_dev, krot_dev, kv->mean, kv->mean_scale);
    else
        hipLaunchKernelGGL(k_paged_append<F16x2>, grid, dim3(576), lds, ctx->stream, a,
                           (uint16_t *)kv->pages, latent_dev, krot_dev, kv->mean, kv->mean_scale);
    timing_end(ctx, tok);
    return launch_check(ctx, "k_paged_append");
}

extern "C" int32_t ut_mla_paged_attend(ut_ctx *ctx, const ut_mla_pages *kv,
                                       const int32_t *table_dev, int64_t table_stride,
                                       int64_t max_pages, const int32_t *lens_dev, int64_t batch,
                                       int64_t rows, int64_t heads, const void *qabs_dev,
                                       const void *q_rope_dev, float scale, void *clat_dev) {
    if (!ctx) return UT_ERR_ARG;
    return paged_attend(ctx, "ut_mla_paged_attend", kv, table_dev, table_stride, max_pages,
                        lens_dev, batch, rows, heads, qabs_dev, q_rope_dev, scale, nullptr, 0,
                        clat_dev);
}

extern "C" int32_t ut_mla_sparse_attend(ut_ctx *ctx, const ut_mla_pages *kv,
                                        const int32_t *table_dev, int64_t table_stride,
                                        int64_t max_pages, const int32_t *lens_dev, int64_t batch,
                                        int64_t rows, int64_t heads, const void *qabs_dev,
                                        const void *q_rope_dev, float scale, const int32_t *sel_dev,
                                        int64_t top_k, void *clat_dev) {
    if (!ctx) return UT_ERR_ARG;
    if (!sel_dev || top_k <= 0 || (kv && kv->page > 0 && top_k > kMostPositions / kv->page)) {
        set_error(ctx, "ut_mla_sparse_attend: a selection of one page or more, 2^31 - 1024 positions at most, is needed");
        return UT_ERR_ARG;
    }
    return paged_attend(ctx, "ut_mla_sparse_attend", kv, table_dev, table_stride, max_pages,
                        lens_dev, batch, rows, heads, qabs_dev, q_rope_dev, scale, sel_dev, top_k,
                        clat_dev);
}

extern "C" int32_t ut_mla_page_select(ut_ctx *ctx, const ut_mla_pages *kv, const int32_t *table_dev,
                                      int64_t table_stride, int64_t max_pages,
                                      const int32_t *lens_dev, int64_t batch, int64_t rows,
                                      int64_t heads, const void *qabs_dev, const void *q_rope_dev,
                                      const float *weights_dev, int64_t keep_first,
                                      int64_t keep_last, int64_t top_k, int32_t *sel_dev) {
    if (!ctx) return UT_ERR_ARG;
    DeviceScope dev(ctx->device);
    PagedArgs a;
    UT_TRY(paged_args(ctx, dev, "ut_mla_page_select", kv, table_dev, table_stride, max_pages, lens_dev,
                      batch, rows, heads, kMostRows, a));
    if (!qabs_dev || !q_rope_dev || !sel_dev || !kv->mean || !kv->mean_scale ||
        ((uintptr_t)qabs_dev & 15) != 0 || ((uintptr_t)q_rope_dev & 15) != 0 ||
        ((uintptr_t)kv->mean & 15) != 0) {
        set_error(ctx, "ut_mla_page_select: queries and page means must be 16-byte aligned device "
                       "memory");
        return UT_ERR_ARG;
    }
    if (keep_first < 0 || keep_last < 0 || top_k <= 0 || top_k > INT32_MAX / 2 ||
        keep_first > top_k || keep_last > top_k - keep_first) {
        set_error(ctx, "ut_mla_page_select: top_k %lld must hold the %lld first and %lld last pages",
                  (long long)top_k, (long long)keep_first, (long long)keep_last);
        return UT_ERR_ARG;
    }
    if (max_pages > kMostGroups * kScorePages) {
        set_error(ctx, "ut_mla_page_select: a row chooses among at most %lld pages, the table holds %lld",
                  (long long)(kMostGroups * kScorePages), (long long)max_pages);
        return UT_ERR_SHAPE;
    }
    a.qabs = qabs_dev;
    a.qrope = q_rope_dev;
    a.top_k = (int32_t)top_k;
    const int64_t R = batch * rows, D = a.L + a.P, tiles = (heads + kFusedHeads - 1) / kFusedHeads;
    const bool fused = D == 9 * kCodeStep && R * tiles <= ctx->multiprocessors;
    // slices of rows whose codes and parts take 64 MB at most
    const int64_t parts = fused ? tiles : 1, row_bytes = parts * max_pages * 8 + (fused ? 0 : heads * code_row(D));
    int64_t slice = (int64_t(64) << 20) / row_bytes;
    slice = slice < 1 ? 1 : slice < R ? slice : R;
    ScratchPlan plan;
    plan.add((size_t)(slice * parts * max_pages) * 8);
    plan.add((size_t)(slice * max_pages) * 8);
    plan.add(fused ? 0 : (size_t)(slice * heads * code_row(D)));
    plan.add(fused ? 0 : (size_t)(slice * heads) * 8);
    std::vector<void *> ptrs;
    UT_TRY(scratch_acquire(ctx, plan, ptrs));
    double *part = (double *)ptrs[0], *share = (double *)ptrs[3];
    uint64_t *keys = (uint64_t *)ptrs[1];
    int8_t *codes = (int8_t *)ptrs[2];
    const bool bf16 = kv->fmt == UT_KV_BF16;
    for (int64_t r0 = 0; r0 < R; r0 += slice) {
        const int64_t n = R - r0 < slice ? R - r0 : slice;
        if (fused) {
            int tok = timing_begin(ctx, "select_fused");
            hipLaunchKernelGGL((bf16 ? k_select_fused<Bf16> : k_select_fused<F16x2>),
                               dim3((unsigned)((max_pages + kFusedPages - 1) / kFusedPages), (unsigned)tiles, (unsigned)n),
                               dim3(kFusedThreads), 0, ctx->stream, a, weights_dev, kv->mean, (int)r0, part);
            timing_end(ctx, tok);
            UT_TRY(launch_check(ctx, "k_select_fused"));
        } else {
            int tok = timing_begin(ctx, "select_codes");
            hipLaunchKernelGGL((bf16 ? k_select_codes<Bf16> : k_select_codes<F16x2>), dim3((unsigned)((n * heads + 3) / 4)),
                               dim3(256), 0, ctx->stream, a, weights_dev, r0 * heads, n * heads, codes, share);
            timing_end(ctx, tok);
            UT_TRY(launch_check(ctx, "k_select_codes"));
            tok = timing_begin(ctx, "select_score");
            hipLaunchKernelGGL((D == 9 * kCodeStep ? k_select_score<true> : k_select_score<false>),
                               dim3((unsigned)((max_pages + kScorePages - 1) / kScorePages), (unsigned)n), dim3(256), 0,
                               ctx->stream, a, codes, share, kv->mean, (int)r0, part);
            timing_end(ctx, tok);
            UT_TRY(launch_check(ctx, "k_select_score"));
        }
        int tok = timing_begin(ctx, "select_pick");
        hipLaunchKernelGGL(k_select_pick, dim3((unsigned)n), dim3(kPickThreads), 0, ctx->stream, a, part, (int)parts,
                           kv->mean_scale, (int)r0, keys, (int)keep_first, (int)keep_last, sel_dev);
        timing_end(ctx, tok);
        UT_TRY(launch_check(ctx, "k_select_pick"));
    }
    return UT_OK;
}
