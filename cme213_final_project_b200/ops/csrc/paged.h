// Paged cache of keys and values: what its kernels share.
#pragma once
#include "common.h"
#include "paged_desc.h"

#include <cuda.h>

// The kernel and the division of the keys that a call takes.
struct PagedPlan {
    int kernel;          // PAGED_*
    int row_tile;        // rows (tokens x query heads of one key head) of a CTA
    int tiles;           // row tiles of all sequences at the most
    int splits;          // parts that the keys of a row tile are divided into; stream: CTAs
    int split_keys;      // keys of a part (multiple of the key tile; rows and tc)
};
enum PagedKernel : int {
    PAGED_CLUSTER = 0,   // up to 16 rows a tile; the parts are one cluster's CTAs, which join them through shared memory
    PAGED_STREAM = 1,    // up to 16 rows a tile; all tiles' keys in a row, divided among the CTAs; joined through `ws`
    PAGED_ROWS = 2,      // 64 rows; joined through `ws`, as are the next one's
    PAGED_TC = 3,        // tcgen05, 128 rows (head size 128: 256)
};

int paged_make_map(CUtensorMap* out, const CmePaged* a, const void* base, long long page_stride, long long head_stride,
                   long long slot_stride, int box_cols, int box_rows, CUtensorMapSwizzle swizzle);
// Q as (column, head, token, -): a box of `group` heads and `tokens` tokens, so that its rows lie token by token.
int paged_make_q_map(CUtensorMap* out, const CmePaged* a, int group, int tokens);
int paged_attention_mma(const CmePaged* a, const PagedPlan& plan, cudaStream_t st);
int paged_attention_tc(const CmePaged* a, const PagedPlan& plan, cudaStream_t st);
int paged_join(const CmePaged* a, int splits, cudaStream_t st);      // the parts in a->ws to a->o and a->lse
// Keys of the tiles that the kernels walk in.
int paged_mma_key_tile(int dtype, int head_dim);
int paged_mma_ctas(int dtype, int head_dim);               // of the kernels for up to 16 rows, on an SM
constexpr int PAGED_TC_KEYS = 64;

// Division by a number that the host knows, for 0 <= x < 2^31: x / d = (x * m) >> s with m = ceil(2^s / d) and s = 31 + ceil(log2 d)
// (Granlund and Montgomery, Division by Invariant Integers using Multiplication, 1994).
struct PagedDiv {
    unsigned long long m;
    int s, d;
    __host__ __device__ int div(int x) const { return (int)(((unsigned long long)(unsigned)x * m) >> s); }
};
inline PagedDiv paged_div(int d) {
    PagedDiv p;
    int lg = 0;
    while ((1ll << lg) < d) ++lg;
    p.d = d;
    p.s = 31 + lg;
    p.m = ((1ull << p.s) + d - 1) / d;
    return p;
}

// Whether paged_find_tile_by_keys takes the call.
inline bool paged_by_keys(const CmePaged* a, int group) { return a->seqs <= 32 && (long long)a->rows * group < (1ll << 30); }

#ifdef __CUDACC__

// What a CTA works on: rows [first, first + rows) of a sequence's tokens x group, for one key head.
struct PagedTile {
    int seq, first, rows;        // rows == 0: the tile does not exist
    int token0, n, length;       // the sequence's first row of q, its new tokens, its tokens
};

// The length of a sequence with n new tokens.  Where it passes max_len (here no more than the table holds), the new tokens keep their positions
// (cache_append writes those that have a place): each sees the keys below max_len up to its own.  Where none of them has a place, the length counts as max_len.
__device__ __forceinline__ int paged_length(const CmePaged& a, int len, int n) {
    len = max(0, len);
    return len - n >= a.max_len ? a.max_len : len;
}

// Finds row tile `tile`, counting ceil(new tokens x group / row_tile) tiles per sequence.  Whole warps call it; every warp gets
// the answer.  offsets and lengths that make no sense cannot lead outside of the buffers: they are cut to them.
__device__ __forceinline__ PagedTile paged_find_tile(const CmePaged& a, int tile, int group, int row_tile) {
    const int lane = threadIdx.x & 31;
    PagedTile t{};
    int base = 0;
    for (int b0 = 0; b0 < a.seqs; b0 += 32) {
        const int b = b0 + lane;
        int lo = 0, hi = 0, len = 0;
        if (b < a.seqs) { lo = a.offsets[b]; hi = a.offsets[b + 1]; len = a.lengths[b]; }
        lo = max(0, min(lo, a.rows));
        hi = max(lo, min(hi, a.rows));
        const int n = hi - lo;
        const int own = (int)(((long long)n * group + row_tile - 1) / row_tile);
        int upto = own;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const int v = __shfl_up_sync(0xffffffffu, upto, o);
            if (lane >= o) upto += v;
        }
        const unsigned found = __ballot_sync(0xffffffffu, tile < base + upto);
        if (found) {
            const int src = __ffs(found) - 1;
            const int first = (tile - base - __shfl_sync(0xffffffffu, upto - own, src)) * row_tile;
            t.seq = b0 + src;
            t.token0 = __shfl_sync(0xffffffffu, lo, src);
            t.n = __shfl_sync(0xffffffffu, n, src);
            t.length = paged_length(a, __shfl_sync(0xffffffffu, len, src), t.n);
            t.first = first;
            t.rows = (int)min((long long)row_tile, (long long)t.n * group - first);
            return t;
        }
        base += __shfl_sync(0xffffffffu, upto, 31);
    }
    return t;
}

// As paged_find_tile, counting the tiles by what they see: most key tiles of `keys` keys first, equal ones by sequence.  Up to 32 sequences
// and 2^30 rows.
__device__ __forceinline__ PagedTile paged_find_tile_by_keys(const CmePaged& a, int tile, int group, int row_tile, int keys) {
    const int b = threadIdx.x & 31;
    PagedTile t{};
    int lo = 0, hi = 0, len = 0;
    if (b < a.seqs) {
        lo = a.offsets[b];
        hi = a.offsets[b + 1];
        len = a.lengths[b];
    }
    lo = max(0, min(lo, a.rows));
    hi = max(lo, min(hi, a.rows));
    const int n = hi - lo, length = paged_length(a, len, n), held = min(length, a.max_len);
    const int own = (n * group + row_tile - 1) / row_tile;
    // tiles of the sequence that see x key tiles at least; they are its last ones
    auto count = [&](int x) {
        const long long need = (long long)(x - 1) * keys + 1;          // keys
        if (x <= 0) return own;
        if (held < need) return 0;
        const int more = (int)max(1ll, need - length + n);             // of the new tokens (<= n)
        return own - ((more - 1) * group + row_tile) / row_tile + 1;   // without those that end before the first row of token more - 1
    };
    if (tile >= (int)__reduce_add_sync(0xffffffffu, own)) return t;
    int x = 0, most = __reduce_max_sync(0xffffffffu, n > 0 ? held / keys + 1 : 0);      // the tile sees between x and `most` key tiles
    while (x < most) {
        const int mid = (x + most + 1) >> 1;
        if ((int)__reduce_add_sync(0xffffffffu, count(mid)) > tile) x = mid;
        else most = mid - 1;
    }
    const int above = count(x + 1), same = count(x) - above;
    tile -= (int)__reduce_add_sync(0xffffffffu, above);
    int upto = same;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const int v = __shfl_up_sync(0xffffffffu, upto, o);
        if (b >= o) upto += v;
    }
    const int src = __ffs(__ballot_sync(0xffffffffu, tile < upto)) - 1;
    t.seq = src;
    t.first = __shfl_sync(0xffffffffu, (own - above - 1 - (tile - (upto - same))) * row_tile, src);
    t.token0 = __shfl_sync(0xffffffffu, lo, src);
    t.n = __shfl_sync(0xffffffffu, n, src);
    t.length = __shfl_sync(0xffffffffu, length, src);
    t.rows = (int)min((long long)row_tile, (long long)t.n * group - t.first);
    return t;
}

#endif  // __CUDACC__
