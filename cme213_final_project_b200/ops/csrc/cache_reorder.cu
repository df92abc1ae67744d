// A paged cache after a step of a search with beams: sequence i of a group goes on from its parent p.
//
// Pages that are full are never written again, so the beams share them: of those the table takes p's entries.  The last, partly filled page is
// written by each beam for itself: where p is not i, its filled slots are copied to i's spare page, which takes the old one's place in the table, and
// the old one, which others may be copying from, becomes the spare page of the next step.  Tables and spare pages are written to new memory, so
// that no order among the CTAs is needed.
//
// What bounds it: the bytes of the last pages of all layers, read and written once; with few beams a launch and the chain parent, length ->
// page -> rows.  A warp copies the filled slots of one layer, head and tensor at a time.  8 groups of 8 beams, 24 layers, 16 heads of 64, pages of
// 16, 57 MB: 16.4 us on inputs that are not in L2, 3.5 TB/s, 20.5 with L2 cleared before each call, 11.2 replayed on one input (20.8 and more then with
// a division for each piece's row and a CTA for four items; two items of a warp at a time 12.3, cleared 22.5); 4 beams of 12 layers 2.8 us.
#include "paged.h"
#include "beam_desc.h"

#include <algorithm>

namespace {

constexpr int WARPS = 4;

// n pieces of type V, of which `pieces` make up a row; 0: all lie in a row (as the rows of a head do where slots are one behind the other).
template <typename V> __device__ __forceinline__ void copy_rows(const char* src, char* dst, long long stride, int n, const PagedDiv& pieces, int lane) {
    constexpr int AHEAD = 4;
    for (int i0 = lane; i0 < n; i0 += 32 * AHEAD) {
        V v[AHEAD];
        long long at[AHEAD];
#pragma unroll
        for (int u = 0; u < AHEAD; ++u) {
            const int i = i0 + u * 32;
            if (pieces.d) {
                const int r = pieces.div(i);
                at[u] = r * stride + (i - r * pieces.d) * (int)sizeof(V);
            } else {
                at[u] = i * (int)sizeof(V);
            }
            if (i < n) v[u] = *reinterpret_cast<const V*>(src + at[u]);
        }
#pragma unroll
        for (int u = 0; u < AHEAD; ++u) if (i0 + u * 32 < n) *reinterpret_cast<V*>(dst + at[u]) = v[u];
    }
}

struct Divisors { PagedDiv sequence, beams, heads[4], pieces[4]; };

__global__ void __launch_bounds__(WARPS * 32) cache_reorder_kernel(const CmeReorder a, const Divisors by, int chunks) {
    pdl_release();
    pdl_wait();
    const int seq = by.sequence.div(blockIdx.x), chunk = blockIdx.x - seq * chunks, group = by.beams.div(seq), own = seq - group * a.beams;
    int parent = a.parents[seq];
    const int length = max(0, a.lengths[group]), spare = a.spare[seq];
    if (parent < 0 || parent >= a.beams) parent = own;
    const int* from = a.pages + (long long)(group * a.beams + parent) * a.pages_ld;
    const int* mine = a.pages + (long long)seq * a.pages_ld;
    const int full = min(a.width, length / a.slots), rest = full < a.width ? length - full * a.slots : 0;
    const bool moved = rest > 0 && parent != own;
    const int src = moved ? from[full] : -1;
    const bool there = src >= 0 && src < a.num_pages, copied = moved && there && spare >= 0 && spare < a.num_pages;
    if (chunk == 0) {
        int* to = a.new_pages + (long long)seq * a.width;
        for (int c = threadIdx.x; c < a.width; c += WARPS * 32) {
            int v = c < full ? from[c] : mine[c];
            if (c == full && moved) v = copied ? spare : there ? -1 : src;
            to[c] = v;
        }
        if (threadIdx.x == 0) a.new_spare[seq] = copied ? mine[full] : spare;
    }
    if (!copied) return;
    const int lane = threadIdx.x & 31;
    int base = 0;                          // items (tensor, layer, head) of the tensors before
    int item = chunk * WARPS + (threadIdx.x >> 5);
    for (int k = 0; k < a.tensors; ++k) {
        const CmePages& t = a.t[k];
        const int n = a.layers * t.heads, rows = (rest + t.per - 1) / t.per;
        for (; item < base + n; item += chunks * WARPS) {
            const int layer = by.heads[k].div(item - base), head = (item - base) - layer * t.heads;
            const char* p = t.base + layer * t.layer + head * t.head;
            char* q = t.base + layer * t.layer + head * t.head + spare * t.page;
            p += src * t.page;
            if (t.row_bytes & 15) copy_rows<int>(p, q, t.row, rows * t.row_bytes >> 2, by.pieces[k], lane);
            else copy_rows<uint4>(p, q, t.row, rows * t.row_bytes >> 4, by.pieces[k], lane);
        }
        base += n;
    }
}

}  // namespace

CME_API int cme_cache_reorder(const CmeReorder* a, void* stream) {
    CME_REQUIRE(a->groups >= 0 && a->beams > 0 && a->width >= 0 && a->slots > 0 && a->layers >= 0 && a->num_pages >= 0 && a->tensors >= 0 &&
                a->tensors <= 4, CME_ERR_SHAPE, "cache reorder: bad sizes");
    long long items = 0;
    Divisors by{};
    for (int k = 0; k < a->tensors; ++k) {
        const CmePages& t = a->t[k];
        CME_REQUIRE(t.heads > 0 && t.per > 0 && t.row_bytes > 0, CME_ERR_SHAPE, "cache reorder: bad sizes");
        const int n = t.row_bytes & 15 ? 4 : 16;
        CME_REQUIRE(t.row_bytes % n == 0 && reinterpret_cast<uintptr_t>(t.base) % n == 0 && t.layer % n == 0 && t.page % n == 0 && t.head % n == 0 &&
                    t.row % n == 0, CME_ERR_SHAPE, "cache reorder: the cache has to start, and its strides have to be, at multiples of 16 bytes (scales: 4)");
        CME_REQUIRE((long long)a->slots * t.row_bytes < (1ll << 31), CME_ERR_LIMIT, "cache reorder: too large pages");
        items += (long long)a->layers * t.heads;
        by.heads[k] = paged_div(t.heads);
        if (t.row != t.row_bytes) by.pieces[k] = paged_div(t.row_bytes / n);
    }
    const long long seqs = (long long)a->groups * a->beams;
    if (seqs == 0) return CME_OK;
    CME_REQUIRE(items < (1ll << 30) && seqs < (1ll << 24), CME_ERR_LIMIT, "cache reorder: too many sequences or layers");
    // Sixteen CTAs for each SM (some of which find nothing to copy), and a warp for each item at the most.  64 an SM 14.9 us, 32 11.5, 8 11.9.
    int sms;
    if (const int rc = cme_num_sms(&sms)) return rc;
    const long long most = std::max(1ll, (items + WARPS - 1) / WARPS), wanted = (sms * 16ll + seqs - 1) / seqs;
    const int chunks = (int)std::max(1ll, std::min(most, std::min(wanted, ((1ll << 31) - 1) / seqs)));
    by.sequence = paged_div(chunks);
    by.beams = paged_div(a->beams);
    CME_CUDA(cme_launch_dependent(cache_reorder_kernel, dim3((unsigned)(seqs * chunks)), dim3(WARPS * 32), 0, (cudaStream_t)stream, *a, by, chunks));
    CME_LAUNCH_CHECK();
    return CME_OK;
}
