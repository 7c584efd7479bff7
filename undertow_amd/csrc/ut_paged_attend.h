// ut_paged_attend.h -- what the matrix-core attention kernels over the paged
// latent cache share: how a workgroup finds its range of the batch's tiles and
// goes over the parts of it, which positions a row sees, how positions are looked
// up, and copies straight to LDS.
#pragma once

#include <type_traits>

#include "ut_paged.h"

namespace ut {

typedef __bf16 pbf16x8 __attribute__((ext_vector_type(8)));
typedef __bf16 pbf16x4 __attribute__((ext_vector_type(4)));
typedef __bf16 pbf16x2 __attribute__((ext_vector_type(2)));
typedef _Float16 pf16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 pf16x4 __attribute__((ext_vector_type(4)));
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
    void *part_o;     // [slot][group][128 quads][16 columns][4], f32 or (8-bit pages) f16
    float *part_ml;   // [slot][group][16 columns][2], offset and sum; with f16 [4], the third part_o's own offset
    int64_t *plan;    // [units] first tile of each, then W (where there is more than one range)
    int32_t lead;     // empty tiles before every unit with tiles but the first
};

// What a call's rows see: all positions up to their own, the listed pages, or
// the first ones and a window.
enum { kAll, kListed, kNear };

__device__ __forceinline__ NearCut near_cut(const PagedArgs &a, int32_t n) { return near_cut(n, a.M, a.window, a.sinks, kPT); }

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

// What a wave needs to look positions up: unit u's sequence and row.
struct Lookup {
    const_i32 *table, *sel;  // the sequence's row of the table, the row's pages
    int32_t n, top_k, shift;
    int32_t window, sinks;  // with a window
    NearCut cut;
};
// The first position of the unit's tile x.
template <int KIND> __device__ __forceinline__ int32_t tile_at(const Lookup &k, int32_t x) {
    return KIND == kNear ? near_tile(k.cut, x, kPT) : x * kPT;
}
// The page of the sequence that holds the unit's position v0; one that it
// does have, where there is none or it lies behind the end.
template <int KIND> __device__ __forceinline__ int32_t page_of(const Lookup &k, int32_t v0) {
    if (KIND == kListed) {
        const int32_t i = v0 >> k.shift;
        return i < k.top_k ? k.sel[i] : 0;
    }
    // (eight positions that no row sees: their page need not be named)
    if (KIND == kNear && near_hidden(k.cut, k.sinks, v0, 8)) return -1;
    return (v0 < k.n ? v0 : k.n - 1) >> k.shift;
}
template <int KIND> __device__ __forceinline__ int32_t page_entry(const Lookup &k, int32_t page) {
    // the pool's first page stands in for one that is not listed or not seen: the
    // table need not name any but the listed ones
    const bool none = KIND == kNear ? page < 0 : KIND == kListed && (page < 0 || ((int64_t)page << k.shift) >= k.n);
    const int32_t entry = k.table[none ? 0 : page];
    return none ? 0 : entry;
}
// The visible positions of the tile at v0 for a row that sees n.
template <int KIND>
__device__ __forceinline__ uint32_t visible(const Lookup &k, int32_t v0, int32_t n) {
    if (KIND == kAll) return low_bits(n - v0);
    if (KIND == kNear) return near_seen(v0, n, k.window, k.sinks);
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
template <int KIND> __device__ __forceinline__ uint32_t some_see(const Lookup &k, int32_t x, int32_t len) {
    const int32_t v0 = tile_at<KIND>(k, x);
    return KIND == kNear ? near_some(k.cut, v0, len, k.sinks) : low_bits(len - v0);
}
template <int KIND> __device__ __forceinline__ uint32_t all_see(const Lookup &k, int32_t x, int32_t len, int32_t M) {
    const int32_t v0 = tile_at<KIND>(k, x);
    return KIND == kNear ? near_every(v0, len, M, k.window, k.sinks) : low_bits(len - M + 1 - v0);
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

// s_waitcnt of at most n vector memory operations under way
constexpr int wait_vm(int n) { return 0x0f70 | n; }

// The part of a range that lies in one unit.
struct Seg {
    int32_t u, j, h0, b0, b1, tiles, n;
    int32_t base, len, rows;  // row j sees the positions before base + j; the workgroup's rows end at len, so many
    int64_t first, row;
    Lookup lk;
};
// Goes over a range's parts.  OWN (prompts, where there are no parts to join): the
// tiles of a unit are those that the workgroup's rows j0 .. j1 see, from the first
// to the last.
template <int KIND, bool OWN> struct Walk {
    int32_t u;
    int64_t first, at;
    int32_t j0, j1;
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
        q.base = q.len - a.M + 1;
        q.rows = a.M;
        q.n = q.len - a.M + q.j + 1;
        if (OWN) {
            q.len = q.base + j1 > 1 ? q.base + j1 : 1;  // (rows that see nothing go over one tile)
            q.rows = j1 - j0 + 1;
        }
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
            q.lk.cut = near_cut(q.len, q.rows, a.window, a.sinks, kPT);
        }
        if (OWN) q.tiles = q.b1 = (q.len - 1) / kPT + 1 - (KIND == kNear ? q.lk.cut.skip : 0);
        first += tiles + p.lead;
        at = first;
        u++;
        return true;
    }
};

// Which range and which of its workgroups this one is.  Neighbours are on one XCD;
// prompts' rows, whose ends differ, go from the last one to the first, over all XCDs.
template <bool OWN> __device__ __forceinline__ int place(int chunks, int &r, int &chunk) {
    const int id = OWN ? blockIdx.x : (blockIdx.x & 7) * (gridDim.x >> 3) + (blockIdx.x >> 3);
    r = id / chunks;
    chunk = id - r * chunks;
    if (OWN) chunk = chunks - 1 - chunk;
    return id;
}
template <int KIND, bool OWN> __device__ __forceinline__ Walk<KIND, OWN> walk_of(const PagedMfmaArgs &p, const Range &rg, int chunk) {
    if (!OWN) return {rg.u, rg.first, rg.s, 0, 0};
    const int per_row = (p.a.H + kCols - 1) / kCols, g0 = chunk * p.per, g1 = g0 + p.per < p.groups ? g0 + p.per : p.groups;
    return {rg.u, rg.first, rg.s, g0 / per_row, (g1 - 1) / per_row};
}
// A call's kernel: f(KIND, OWN).
template <class F> void with_kind(int kind, bool own, F &&f) {
    typedef std::integral_constant<bool, true> yes;
    typedef std::integral_constant<bool, false> no;
    if (kind == kListed) f(std::integral_constant<int, kListed>(), no());
    else if (kind == kAll) own ? f(std::integral_constant<int, kAll>(), yes()) : f(std::integral_constant<int, kAll>(), no());
    else own ? f(std::integral_constant<int, kNear>(), yes()) : f(std::integral_constant<int, kNear>(), no());
}

// The kernel of 8-bit pages (ut_paged_codes.hip), `wgs` workgroups.
struct CodesI8 {
    static constexpr bool kCodes = true;
    static constexpr PlanCostsMany kCosts = kCostsI8;
    typedef __bf16 out_t;
    typedef _Float16 part_t;
};
void launch_codes(ut_ctx *ctx, const PagedMfmaArgs &p, int kind, bool own, unsigned wgs);

}  // namespace ut
