// A paged cache of keys and values: what goes into it, and the host side of the attention that reads it.
#include "paged.h"

#include <algorithm>
#include <mutex>

namespace {

// ------------------------------------------------------------------------------------------------------
// Append
// ------------------------------------------------------------------------------------------------------
// Token i of a sequence's n new ones goes to position length - n + i.  A copy, so bytes bound it (read once, written once); one warp per
// token, whose loads are on their way before it looks up where they go: offsets -> length -> page is a chain of three.
// 16 prompts of 500 to 1024 tokens, 12 heads of 64: 14.6 us, 5.1 TB/s of 75 MB.  16 tokens: 2.3 us, a launch and the chain.
constexpr int APPEND_WARPS = 4;
constexpr int APPEND_UNROLL = 4;           // 16-byte pieces per lane of keys, and as many of values, at a time

template <bool WIDE>                       // whether a token has more pieces than one round of a warp takes
__global__ void __launch_bounds__(APPEND_WARPS * 32) paged_append_kernel(const CmePaged a, PagedDiv page_div, int elem, int head_log) {
    pdl_release();
    pdl_wait();
    const int token = blockIdx.x * APPEND_WARPS + (threadIdx.x >> 5), lane = threadIdx.x & 31;
    if (token >= a.rows) return;
    const int pieces = a.kv_heads << head_log;             // of 16 bytes, keys
    const char* k = static_cast<const char*>(a.q) + token * a.q_token * elem;
    const char* v = static_cast<const char*>(a.nv) + token * a.v_token * elem;
    uint4 kr[APPEND_UNROLL], vr[APPEND_UNROLL];
    auto load = [&](int c0) {
#pragma unroll
        for (int u = 0; u < APPEND_UNROLL; ++u) {
            const int c = c0 + u * 32 + lane, h = c >> head_log, d = (c - (h << head_log)) * 16;
            if (c < pieces) {
                kr[u] = *reinterpret_cast<const uint4*>(k + h * a.q_head * elem + d);
                vr[u] = *reinterpret_cast<const uint4*>(v + h * a.v_head * elem + d);
            }
        }
    };
    load(0);
    // the sequence whose rows hold the token: the last b with offsets[b] <= token, a 32nd of the range at a time
    int lo = 0, n = a.seqs;                                // it lies in [lo, lo + n)
    while (n > 1) {
        const int step = (n + 31) >> 5, b = lo + lane * step;
        const unsigned le = __ballot_sync(0xffffffffu, lane * step < n && a.offsets[b] <= token);
        const int last = le ? 31 - __clz(le) : 0;
        n = min(step, n - last * step);
        lo += last * step;
    }
    const int first = a.offsets[lo], next = a.offsets[lo + 1];
    const int length = a.lengths[lo];
    if (token < first || token >= next || next > a.rows) return;
    const long long pos = (long long)length - next + token;
    if (pos < 0 || pos >= min((long long)a.width * a.page, (long long)a.max_len)) return;
    const int col = page_div.div((int)pos), slot = (int)pos - col * a.page;
    const int page = a.pages[lo * a.pages_ld + col];
    if (page < 0 || page >= a.num_pages) return;
    char* dk = static_cast<char*>(a.k) + (page * a.k_page_stride + slot * a.k_slot_stride) * elem;
    char* dv = static_cast<char*>(a.v) + (page * a.v_page_stride + slot * a.v_slot_stride) * elem;
    for (int c0 = 0; c0 < pieces; c0 += APPEND_UNROLL * 32) {
        if (WIDE && c0) load(c0);
#pragma unroll
        for (int u = 0; u < APPEND_UNROLL; ++u) {
            const int c = c0 + u * 32 + lane, h = c >> head_log, d = (c - (h << head_log)) * 16;
            if (c < pieces) {
                *reinterpret_cast<uint4*>(dk + h * a.k_head_stride * elem + d) = kr[u];
                *reinterpret_cast<uint4*>(dv + h * a.v_head_stride * elem + d) = vr[u];
            }
        }
    }
}

// ------------------------------------------------------------------------------------------------------
// Checks, and the choice of a kernel
// ------------------------------------------------------------------------------------------------------
int check_cache(const CmePaged* a, const char* what) {
    CME_REQUIRE(a->dtype == CME_F32 || a->dtype == CME_BF16, CME_ERR_UNSUPPORTED, "%s: unsupported dtype", what);
    CME_REQUIRE(a->head_dim == 32 || a->head_dim == 64 || a->head_dim == 128, CME_ERR_SHAPE, "%s: head size %d is not 32, 64 or 128",
                what, a->head_dim);
    CME_REQUIRE(a->page >= 8 && a->page % 8 == 0, CME_ERR_SHAPE, "%s: pages of %d slots (a multiple of 8 is needed)", what, a->page);
    CME_REQUIRE(a->seqs >= 0 && a->rows >= 0 && a->kv_heads > 0 && a->kv_heads <= 65535 && a->width >= 0 && a->num_pages >= 0 &&
                a->max_len >= 0, CME_ERR_SHAPE, "%s: bad sizes", what);
    const int per16 = a->dtype == CME_F32 ? 4 : 8;
    auto ok = [&](const void* p, long long s0, long long s1, long long s2) {
        return (reinterpret_cast<uintptr_t>(p) & 15) == 0 && s0 % per16 == 0 && s1 % per16 == 0 && s2 % per16 == 0;
    };
    CME_REQUIRE(ok(a->k, a->k_page_stride, a->k_head_stride, a->k_slot_stride) && ok(a->v, a->v_page_stride, a->v_head_stride, a->v_slot_stride),
                CME_ERR_SHAPE, "%s: the cache has to start, and its strides have to be, at multiples of 16 bytes", what);
    CME_REQUIRE(ok(a->q, a->q_token, a->q_head, 0) && ok(a->nv, a->v_token, a->v_head, 0), CME_ERR_SHAPE,
                "%s: new rows have to start, and their strides have to be, at multiples of 16 bytes", what);
    return CME_OK;
}

constexpr int MAX_SPLITS = 128;

// Estimated time of a form, in us: turns of its CTAs on the GPU, key tiles of a turn (two more where there are several: starts and ends), time
// of a key tile (of its own size and rows, measured with
// the keys in L2 and all SMs busy), and what its parts cost that are joined through scratch (written and read once more, at 3 TB/s,
// and a launch).  The host does not know the sequences: they are taken to be as long as the longest, and to share the new tokens evenly.
// Measured / estimated: 12 heads of 64, 128 tokens over 4096 in 4 sequences: tc in 1, 4, 8 parts 72 / 79, 32 / 32, 31 / 27, stream 62 / 72;
// 4 heads of 128 in fp32, 256 over 512 in 8: rows 56 / 53, stream 97 / 107; 12 heads of 64 in fp32, 256 over 512 in 8: rows 72 / 98, stream 109 / 113.
struct Form {
    int keys;                // of a tile
    int slots;               // CTAs that run at a time
    float tile_us;
};
Form form_of(const CmePaged* a, int backend, int sms) {
    const bool f32 = a->dtype == CME_F32;
    const int d = a->head_dim;
    if (backend == 3) return {PAGED_TC_KEYS, sms * (d == 128 ? 1 : 3), d == 128 ? 1.0f : 1.15f};
    const int keys = paged_mma_key_tile(a->dtype, d);
    if (backend == 1) return {keys, sms * paged_mma_ctas(a->dtype, d), f32 ? (d == 128 ? 2.8f : d == 64 ? 2.0f : 1.4f) : d == 64 ? 1.4f : 1.2f};
    return {keys, sms * (d == 32 ? (f32 ? 2 : 3) : 1), f32 ? (d == 128 ? 6.0f : d == 64 ? 3.0f : 4.5f) : d == 128 ? 2.6f : 1.8f};
}
float estimate(const CmePaged* a, const Form& f, long long tiles, int key_tiles, int parts) {
    const long long ctas = tiles * a->kv_heads * parts;
    const double turns = ctas <= f.slots ? 1.0 : (double)ctas / f.slots + 0.5;         // (the shortest last: half a turn at the end)
    const double joined = parts > 1 ? 4.0 + (double)a->rows * a->heads * parts * (a->head_dim + 2) * 8 / 3e6 : 0.0;
    return (float)(5.0 + turns * (cme_cdiv(key_tiles, parts) + 2 * (turns > 1)) * f.tile_us + joined);
}

// backend: 0 by the rule, 1 up to 16 rows a tile, 2 rows, 3 tc.  splits: 0 by the rule; up to 16 rows: a cluster of so many CTAs (1, 2, 4
// or 8), negative: the stream; others: parts of the keys.
int make_plan(const CmePaged* a, int backend, int splits, int sms, PagedPlan* plan) {
    const int group = a->heads / a->kv_heads;
    const long long rows = (long long)a->rows * group;     // of one key head
    const bool tc = a->dtype == CME_BF16 && group <= 128;
    CME_REQUIRE(backend >= 0 && backend <= 3, CME_ERR_UNSUPPORTED, "paged attention: unknown backend");
    CME_REQUIRE(backend != 3 || tc, CME_ERR_UNSUPPORTED,
                "paged attention: the tcgen05 kernel takes bf16 and up to 128 query heads per key head");
    auto row_tile = [&](int b) { return b == 1 ? 16 : b == 2 ? 64 : (a->head_dim == 128 ? 2 : 1) * (128 / group * group); };
    auto tiles_of = [&](int b) { return rows / row_tile(b) + std::min(a->seqs, a->rows); };      // at the most: each sequence adds less than one
    auto even_tiles = [&](int b) { return a->seqs ? a->seqs * ((rows + (long long)a->seqs * row_tile(b) - 1) / ((long long)a->seqs * row_tile(b))) : 0; };
    const int longest = (int)std::min((long long)a->max_len, (long long)a->width * a->page);
    auto key_tiles_of = [&](const Form& f) { return std::max(1, cme_cdiv(longest, f.keys)); };
    auto best_parts = [&](int b, float* us) {              // of rows and tc
        const Form f = form_of(a, b, sms);
        const int n = key_tiles_of(f);
        int best = 1;
        *us = estimate(a, f, even_tiles(b), n, 1);
        for (int parts = 2; parts <= std::min(n, MAX_SPLITS); parts += (parts + 3) / 4) {
            const float t = estimate(a, f, even_tiles(b), n, parts);
            if (t < *us) { *us = t; best = parts; }
        }
        return best;
    };
    // Up to 16 rows a tile: as many CTAs of a cluster as let all run at once; the stream from where a CTA would have more than eight key
    // tiles in its turns (head size 64, lengths from half of the longest on, us, cluster / stream: 96 items of up to 1024 keys 8.5 /
    // 10.1, of 4096 21.9 / 20.5; 384 items of 256 9.9 / 11.2, of 1024 23.0 / 21.4.  128: 32 items of 4096 14.1 / 17.7, 8 of 16384 33.6 / 21.8).
    const Form one = form_of(a, 1, sms);
    const int one_keys = key_tiles_of(one);
    auto cluster_of = [&](long long items, int* c) {       // the cluster's size, and the key tiles of a CTA's turns
        for (*c = 1; *c < 8 && *c < one_keys && items * *c * 2 <= one.slots;) *c *= 2;
        return (items * *c + one.slots - 1) / one.slots * cme_cdiv(one_keys, *c);
    };
    if (!backend) {
        backend = 1;
        if (rows > 16ll * a->seqs) {                       // (else a row tile has all rows of a sequence: its keys are read once)
            int many = tc ? 3 : 2;
            // (a sequence's last tile of rows is half full on average)
            const long long items = (rows / 16 + a->seqs / 2) * a->kv_heads;
            int c;
            const long long turns = cluster_of(items, &c);
            float us;
            best_parts(many, &us);
            // head size 32 wins less on the tensor cores (us, 12 heads, rows / tc: 64 tokens over 256 in 32 sequences 9.5 / 13.6, 512 over 8192
            // in one 45 / 36, 1100 over 4166 in 5 184 / 141)
            float rows_us;
            if (tc && a->head_dim == 32 && (best_parts(2, &rows_us), rows_us < us)) { many = 2; us = rows_us; }
            // (two more tiles an item of the stream, as its kernel reckons)
            const float tiles = turns <= 8 ? (float)((items * c + one.slots - 1) / one.slots) * (float)longest / (float)(one.keys * c)
                                           : (float)((items * (one_keys + 2) + one.slots - 1) / one.slots);
            const float few = (turns <= 8 ? 4.5f : 6.f) + tiles * one.tile_us;
            if (us < few) backend = many;
        }
    }
    const Form f = form_of(a, backend, sms);
    const long long tiles = tiles_of(backend), ctas = tiles * a->kv_heads;
    const int key_tiles = key_tiles_of(f);
    plan->row_tile = row_tile(backend);
    int parts = std::min(splits < 0 ? -splits : splits, MAX_SPLITS);
    if (backend == 1) {
        int c;
        const bool cluster = cluster_of(ctas, &c) <= 8 ? splits >= 0 : splits > 0;
        plan->kernel = cluster ? PAGED_CLUSTER : PAGED_STREAM;
        if (cluster) {
            const int want = splits ? parts : c;
            parts = 1;
            while (parts < want && parts < 8) parts *= 2;
        } else {
            CME_REQUIRE(ctas * (key_tiles + 8ll) < (1ll << 31), CME_ERR_LIMIT, "paged attention: too many keys");
            parts = (int)std::min((long long)f.slots, std::max(1ll, ctas * key_tiles));
        }
    } else {
        plan->kernel = backend == 2 ? PAGED_ROWS : PAGED_TC;
        float us;
        if (!parts) parts = best_parts(backend, &us);
    }
    parts = std::max(1, parts);
    plan->splits = parts;
    plan->split_keys = cme_cdiv(key_tiles, parts) * f.keys;
    CME_REQUIRE(tiles * parts * a->kv_heads < (1ll << 31), CME_ERR_LIMIT, "paged attention: too many rows");
    plan->tiles = (int)tiles;
    return CME_OK;
}

long long ws_bytes(const CmePaged* a, const PagedPlan& p) {
    if (p.kernel == PAGED_CLUSTER || (p.kernel != PAGED_STREAM && p.splits == 1)) return 0;
    const long long parts = p.kernel == PAGED_STREAM ? p.splits * 32ll : (long long)a->rows * a->heads * p.splits;
    return ((parts * 2 + 3) / 4 * 4 + parts * a->head_dim + (p.kernel == PAGED_STREAM ? p.splits * 8ll : 0)) * 4;
}

int check_attention(const CmePaged* a) {
    const int rc = check_cache(a, "paged attention");
    if (rc) return rc;
    CME_REQUIRE(a->heads > 0 && a->heads % a->kv_heads == 0, CME_ERR_SHAPE, "paged attention: %d heads do not share %d key heads evenly",
                a->heads, a->kv_heads);
    CME_REQUIRE(a->scale > 0.f && a->scale < INFINITY, CME_ERR_SHAPE, "paged attention: the scale has to be positive and finite");
    return CME_OK;
}

typedef CUresult (*EncodeTiledFn)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*,
                                  const cuuint64_t*, const cuuint32_t*, const cuuint32_t*, CUtensorMapInterleave,
                                  CUtensorMapSwizzle, CUtensorMapL2promotion, CUtensorMapFloatOOBfill);
EncodeTiledFn encoder() {
    static EncodeTiledFn fn = nullptr;
    static std::once_flag once;
    std::call_once(once, [] {
        void* sym = nullptr;
        cudaDriverEntryPointQueryResult q;
        if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &sym, cudaEnableDefault, &q) == cudaSuccess &&
            q == cudaDriverEntryPointSuccess)
            fn = reinterpret_cast<EncodeTiledFn>(sym);
    });
    return fn;
}

}  // namespace

// Map over (column, slot, head, page) with box (box_cols, box_rows, 1, 1).  Page num_pages lies behind it: such a box is filled with zeros.
int paged_make_map(CUtensorMap* out, const CmePaged* a, const void* base, long long page_stride, long long head_stride,
                   long long slot_stride, int box_cols, int box_rows, CUtensorMapSwizzle swizzle) {
    EncodeTiledFn enc = encoder();
    CME_REQUIRE(enc != nullptr, CME_ERR_CUDA, "cuTensorMapEncodeTiled is not available from the driver");
    const long long e = a->dtype == CME_F32 ? 4 : 2;
    cuuint64_t dims[4] = {(cuuint64_t)a->head_dim, (cuuint64_t)a->page, (cuuint64_t)a->kv_heads, (cuuint64_t)std::max(1, a->num_pages)};
    // the stride along a dimension of one entry leads nowhere
    cuuint64_t strides[3] = {(cuuint64_t)(slot_stride * e), (cuuint64_t)((a->kv_heads > 1 ? head_stride : a->head_dim) * e),
                             (cuuint64_t)((a->num_pages > 1 ? page_stride : a->head_dim) * e)};
    cuuint32_t box[4] = {(cuuint32_t)box_cols, (cuuint32_t)box_rows, 1, 1};
    cuuint32_t estr[4] = {1, 1, 1, 1};
    CUresult r = enc(out, a->dtype == CME_F32 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT32 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 4,
                     const_cast<void*>(base), dims, strides, box, estr, CU_TENSOR_MAP_INTERLEAVE_NONE, swizzle,
                     CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    CME_REQUIRE(r == CUDA_SUCCESS, CME_ERR_CUDA, "paged cache: cuTensorMapEncodeTiled failed (%d): strides %lld %lld %lld", (int)r,
                page_stride, head_stride, slot_stride);
    return CME_OK;
}

int paged_make_q_map(CUtensorMap* out, const CmePaged* a, int group, int tokens) {
    EncodeTiledFn enc = encoder();
    CME_REQUIRE(enc != nullptr, CME_ERR_CUDA, "cuTensorMapEncodeTiled is not available from the driver");
    cuuint64_t dims[4] = {(cuuint64_t)a->head_dim, (cuuint64_t)a->heads, (cuuint64_t)a->rows, 1};
    cuuint64_t strides[3] = {(cuuint64_t)(a->heads > 1 ? a->q_head : a->head_dim) * 2, (cuuint64_t)(a->rows > 1 ? a->q_token : a->head_dim) * 2,
                             (cuuint64_t)a->head_dim * 2};
    cuuint32_t box[4] = {64, (cuuint32_t)group, (cuuint32_t)tokens, 1};
    cuuint32_t estr[4] = {1, 1, 1, 1};
    CUresult r = enc(out, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 4, const_cast<void*>(a->q), dims, strides, box, estr,
                     CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                     CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    CME_REQUIRE(r == CUDA_SUCCESS, CME_ERR_CUDA, "paged attention: the map of q failed (%d): strides %lld %lld", (int)r, a->q_token, a->q_head);
    return CME_OK;
}

CME_API int cme_paged_append(const CmePaged* a, void* stream) {
    const int rc = check_cache(a, "cache append");
    if (rc) return rc;
    if (a->rows == 0 || a->seqs == 0 || a->num_pages == 0 || a->width == 0) return CME_OK;
    const int elem = a->dtype == CME_F32 ? 4 : 2;
    int head_log = 0;
    while ((16 << head_log) < a->head_dim * elem) ++head_log;
    const bool wide = (a->kv_heads << head_log) > APPEND_UNROLL * 32;
    const dim3 grid(cme_cdiv(a->rows, APPEND_WARPS));
    auto* kernel = wide ? paged_append_kernel<true> : paged_append_kernel<false>;
    CME_CUDA(cme_launch_dependent(kernel, grid, dim3(APPEND_WARPS * 32), 0, (cudaStream_t)stream, *a, paged_div(a->page), elem, head_log));
    CME_LAUNCH_CHECK();
    return CME_OK;
}

// What a call will take: {kernel, row tile, row tiles, parts, keys of a part}.
CME_API int cme_paged_attention_plan(const CmePaged* a, int backend, int splits, int sms, int* out) {
    PagedPlan p{};
    int rc = check_attention(a);
    if (rc || (rc = make_plan(a, backend, splits, sms, &p))) return rc;
    out[0] = p.kernel; out[1] = p.row_tile; out[2] = p.tiles; out[3] = p.splits; out[4] = p.split_keys;
    return CME_OK;
}

// Scratch of a call, in bytes.
CME_API int cme_paged_attention_ws_bytes(const CmePaged* a, int backend, int splits, long long* out) {
    PagedPlan p{};
    int rc, sms;
    if ((rc = check_attention(a)) || (rc = cme_num_sms(&sms)) || (rc = make_plan(a, backend, splits, sms, &p))) return rc;
    *out = ws_bytes(a, p);
    return CME_OK;
}

CME_API int cme_paged_attention(const CmePaged* a, int backend, int splits, void* stream) {
    PagedPlan p{};
    int rc, sms;
    if ((rc = check_attention(a)) || (rc = cme_num_sms(&sms)) || (rc = make_plan(a, backend, splits, sms, &p))) return rc;
    if (a->rows == 0 || a->seqs == 0) return CME_OK;
    CmePaged held = *a;
    held.max_len = (int)std::min((long long)a->max_len, (long long)a->width * a->page);
    if (a->num_pages == 0) {                               // a cache without memory: no key is there, and nothing is loaded
        held.max_len = 0;
        held.k = held.v = const_cast<void*>(a->q);
    }
    a = &held;
    CME_REQUIRE(ws_bytes(a, p) <= a->ws_bytes, CME_ERR_SHAPE, "paged attention: %lld bytes of scratch, %lld are needed", a->ws_bytes,
                ws_bytes(a, p));
    cudaStream_t st = (cudaStream_t)stream;
    if ((rc = p.kernel == PAGED_TC ? paged_attention_tc(a, p, st) : paged_attention_mma(a, p, st))) return rc;
    return p.splits > 1 && p.kernel >= PAGED_ROWS ? paged_join(a, p.splits, st) : CME_OK;
}
