// ut_paged.h -- internal interface of the paged MLA latent cache.
#pragma once

#include "ut_internal.h"
#include "ut_paged_plan.h"

namespace ut {

// What the kernels read of a paged cache and a batch over it.
struct PagedArgs {
    const void *pages;     // [n_pages][page][row]
    const int32_t *table;  // [B][stride]: physical page of a sequence's k-th page
    int64_t stride;        // entries from one sequence's row of the table to the next
    const int32_t *lens;   // [B]
    int32_t *err;          // the context's page error word
    int32_t n_pages, max_pages, shift;  // page = 1 << shift positions
    int32_t B, M, H, L, P;
    const int32_t *sel;    // [B][M][top_k] pages of the sequence, or nullptr: all
    int32_t top_k;
    float scale;
    const void *qabs, *qrope;
    void *out;
};

// Lengths and tables do not change while a kernel runs: read as constants,
// through the scalar cache where the index is the same for a wave.
typedef const __attribute__((address_space(4))) int32_t const_i32;

// Positions of sequence b, bounded by what its row of the table can hold.
__device__ __forceinline__ int32_t paged_len(const PagedArgs &a, int b) {
    bool bad = false;
    const int32_t n = plan_len(((const_i32 *)a.lens)[b], (int64_t)a.max_pages << a.shift, bad);
    if (bad) *a.err = 1;
    return n;
}
// The physical page of a sequence's k-th page (k < max_pages); an id outside
// the pool is reported and page 0 stands in for it.
__device__ __forceinline__ int32_t paged_phys(const PagedArgs &a, int b, int k, bool &bad) {
    const int32_t p = plan_page(((const_i32 *)a.table)[(int64_t)b * a.stride + k], a.n_pages, bad);
    if (bad) *a.err = 1;
    return p;
}
__device__ __forceinline__ int32_t paged_phys(const PagedArgs &a, int b, int k) {
    bool bad = false;
    return paged_phys(a, b, k, bad);
}

// f16x2: x = hi + lo / 2^11.  hi carries 11 bits and lo the next 11, so the
// pair is off by at most 2^-23 |x| (by 2^-36 below f16's normal range).
constexpr float kF16x2Step = 2048.0f;
__device__ __forceinline__ void f16x2_split(float x, _Float16 &hi, _Float16 &lo) {
    // a finite value past f16's range takes the range's end
    const float c = fabsf(x) < INFINITY ? fminf(fmaxf(x, -65504.0f), 65504.0f) : x;
    hi = (_Float16)c;
    lo = fabsf(c) < INFINITY ? (_Float16)__fmul_rn(__fsub_rn(c, (float)hi), kF16x2Step)
                             : (_Float16)0.0f;
}

// The matrix-core attention (latent 512 + rope 64, pages of 8 and more).
bool paged_mfma_ok(const PagedArgs &a);
int32_t launch_paged_mfma(ut_ctx *ctx, const PagedArgs &a, int32_t fmt);

}  // namespace ut
