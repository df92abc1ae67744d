// New tokens' keys and values into a paged cache of 8-bit integers with a scale for each block of tokens and head.
//
//     s' = max(s, max |x| (1 / 127)) over the block's new numbers x, s the scale of what it holds already (0 if its first slot is new);   below 2^-100: 0
//     q  = round(x / s'), as x times the rounded 1 / s';     where s' > s, what was held becomes round(q (s / s'))
// Each step is one rounded operation in 32 bits.  A number that stays is off by s' / 2 at most, and by half of every scale that it had before.
// A NaN or an infinity makes the scale a NaN, and with it the block.
//
// What bounds it: bytes (new rows read once, a byte a number written); with few tokens the chain offsets -> length -> page -> scale.  One warp has
// a block and head of keys or of values, so nobody else touches its scale; its rows are on their way before it knows where they go, and with
// them, once it does, what the block holds.  16 prompts of 500 to 777 tokens, 12 heads of 64, blocks of 16, 47 MB: 14.4 us where the new rows are
// not in L2, 3.3 TB/s (fp32, 78 MB: 17.4), 11.1 replayed on one input, of which L2 holds all (16.1 then with a block and head a warp and no
// more, which looks up its place for two KB); 16 tokens 2.6 us.
#include "paged.h"

#include <algorithm>

namespace {

constexpr int WARPS = 4;
constexpr int RESIDENT = 12;                // CTAs of an SM

// Rounds 16 bytes' numbers, the bytes in the order of the numbers.  |x inverse| < 2^22: 1.5 * 2^23 more leaves the nearest integer (the even one of two)
// in the low bits.
__device__ __forceinline__ unsigned round4(float a, float b, float c, float d, float f) {
    constexpr float UP = 12582912.f;
    const unsigned x = __float_as_uint(__fadd_rn(__fmul_rn(a, f), UP)), y = __float_as_uint(__fadd_rn(__fmul_rn(b, f), UP));
    const unsigned z = __float_as_uint(__fadd_rn(__fmul_rn(c, f), UP)), w = __float_as_uint(__fadd_rn(__fmul_rn(d, f), UP));
    return __byte_perm(__byte_perm(x, y, 0x0040), __byte_perm(z, w, 0x0040), 0x5410);
}
__device__ __forceinline__ unsigned again4(unsigned w, float f) {
    auto at = [&](int i) { return (float)(signed char)(w >> (8 * i)); };
    return round4(at(0), at(1), at(2), at(3), f);
}
template <typename T> __device__ __forceinline__ unsigned largest(const uint4& v) {        // magnitude, as the bits of a float (a NaN is above all)
    unsigned m = 0;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const unsigned w = (&v.x)[i];
        m = sizeof(T) == 4 ? max(m, w & 0x7fffffffu) : max(m, max(w & 0x7fff0000u, (w << 16) & 0x7fff0000u));
    }
    return m;
}

// KEPT: 16-byte pieces of a lane that stay in registers between the maximum and the rounding.
template <typename T, int D, int KEPT>
__global__ void __launch_bounds__(WARPS * 32) paged_append8_kernel(const CmePaged a, const CmePagedScales s, PagedDiv page_div, PagedDiv block_div) {
    constexpr int LANES = D * (int)sizeof(T) / 16, ROWS = 32 / LANES;      // of a row; rows of a warp at a time
    pdl_release();
    pdl_wait();
    const int lane = threadIdx.x & 31;
    int item = blockIdx.y * WARPS + (threadIdx.x >> 5);    // head, keys or values; then the next one of this warp's
    if (item >= 2 * a.kv_heads) return;
    // the sequence of unit blockIdx.x, counting the blocks that each sequence's new tokens touch
    int unit = blockIdx.x, seq = -1, row = 0, first = 0, last = 0, blk = 0;
    const int places = (int)min((long long)a.width * a.page, (long long)a.max_len);
    for (int b0 = 0; b0 < a.seqs && seq < 0; b0 += 128) {
        int lo[4], hi[4], len[4];
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            const int b = b0 + k * 32 + lane;
            const bool in = b < a.seqs;
            lo[k] = in ? a.offsets[b] : 0;
            hi[k] = in ? a.offsets[b + 1] : 0;
            len[k] = in ? a.lengths[b] : 0;
        }
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            lo[k] = max(0, min(lo[k], a.rows));
            hi[k] = max(lo[k], min(hi[k], a.rows));
            const long long start = (long long)len[k] - (hi[k] - lo[k]);   // position of the first new token
            const int p0 = (int)max(0ll, min(start, (long long)places)), p1 = max(p0, min(len[k], places));
            const int b_first = block_div.div(p0), own = p1 > p0 ? block_div.div(p1 - 1) - b_first + 1 : 0;
            int upto = own;
#pragma unroll
            for (int o = 1; o < 32; o <<= 1) {
                const int v = __shfl_up_sync(0xffffffffu, upto, o);
                if (lane >= o) upto += v;
            }
            const unsigned found = __ballot_sync(0xffffffffu, unit < upto);
            if (found) {
                const int src = __ffs(found) - 1;
                seq = b0 + k * 32 + src;
                blk = __shfl_sync(0xffffffffu, b_first - (upto - own), src) + unit;
                first = (int)max((long long)__shfl_sync(0xffffffffu, p0, src), (long long)blk * s.block);
                last = (int)min((long long)__shfl_sync(0xffffffffu, p1, src), (blk + 1ll) * s.block);
                row = __shfl_sync(0xffffffffu, (int)(lo[k] - start), src) + first;
                break;
            }
            unit -= __shfl_sync(0xffffffffu, upto, 31);
        }
    }
    if (seq < 0 || blk < 0 || first >= last) return;       // (offsets out of order can lead past the sums, not out of the buffers)
    // this warp's rows
    const int of = lane / LANES, piece = lane % LANES, n = last - first;
    uint4 v[KEPT];
    auto load = [&](int r0) {
        const bool values = item & 1;
        const T* x = static_cast<const T*>(values ? a.nv : a.q) + row * (values ? a.v_token : a.q_token) + (item >> 1) * (values ? a.v_head : a.q_head) +
                     piece * (16 / (int)sizeof(T));
        const long long step = values ? a.v_token : a.q_token;
#pragma unroll
        for (int u = 0; u < KEPT; ++u) {
            const int r = r0 + u * ROWS + of;
            v[u] = r < n ? *reinterpret_cast<const uint4*>(x + r * step) : make_uint4(0, 0, 0, 0);
        }
    };
    load(0);
    const int col = page_div.div(first), slot = first - col * a.page, held = first - blk * s.block;
    const int page = a.pages[seq * a.pages_ld + col];
    if (page < 0 || page >= a.num_pages) return;
    for (;;) {
        const int head = item >> 1;
        const bool values = item & 1;
        char* cache = values ? static_cast<char*>(a.v) + page * a.v_page_stride + head * a.v_head_stride
                             : static_cast<char*>(a.k) + page * a.k_page_stride + head * a.k_head_stride;
        const long long slot_stride = values ? a.v_slot_stride : a.k_slot_stride;
        float* scale = (values ? s.v + page * s.v_page + head * s.v_head : s.k + page * s.k_page + head * s.k_head) + block_div.div(slot);
        const float before = held ? *scale : 0.f;
        constexpr int PIECES = D / 16;         // of a held row
        char* const begun = cache + (slot - held) * slot_stride;
        uint4 h = make_uint4(0, 0, 0, 0);
        if (lane < held * PIECES) h = *reinterpret_cast<const uint4*>(begun + lane / PIECES * slot_stride + lane % PIECES * 16);
        unsigned m = 0;
#pragma unroll
        for (int u = 0; u < KEPT; ++u) m = max(m, largest<T>(v[u]));
        for (int r0 = KEPT * ROWS; r0 < n; r0 += KEPT * ROWS) {
            load(r0);
#pragma unroll
            for (int u = 0; u < KEPT; ++u) m = max(m, largest<T>(v[u]));
        }
        const float top = __uint_as_float(__reduce_max_sync(0xffffffffu, m)) * (1.f / 127.f);
        float after = before > top || before != before ? before : top;
        if (after < PAGED_SMALLEST_SCALE) after = 0.f;
        if (!(after < INFINITY)) after = __uint_as_float(0x7fffffffu);
        const float inverse = after > 0.f ? __frcp_rn(after) : 0.f;
        if (lane == 0) *scale = after;
        if (held && after != before) {
            const float f = after > 0.f ? __fdiv_rn(before, after) : 0.f;
            for (int i = lane; i < held * PIECES; i += 32) {
                uint4* at = reinterpret_cast<uint4*>(begun + i / PIECES * slot_stride + i % PIECES * 16);
                if (i != lane) h = *at;
                *at = make_uint4(again4(h.x, f), again4(h.y, f), again4(h.z, f), again4(h.w, f));
            }
        }
        for (int r0 = 0; r0 < n; r0 += KEPT * ROWS) {
            if (n > KEPT * ROWS) load(r0);     // (else they are there)
#pragma unroll
            for (int u = 0; u < KEPT; ++u) {
                const int r = r0 + u * ROWS + of;
                if (r >= n) continue;
                char* to = cache + (slot + r) * slot_stride + piece * (16 / (int)sizeof(T));
                if constexpr (sizeof(T) == 4) {
                    *reinterpret_cast<unsigned*>(to) = round4(__uint_as_float(v[u].x), __uint_as_float(v[u].y), __uint_as_float(v[u].z),
                                                              __uint_as_float(v[u].w), inverse);
                } else {
                    float f[8];
                    unpack8(v[u], f);
                    *reinterpret_cast<uint2*>(to) = make_uint2(round4(f[0], f[1], f[2], f[3], inverse), round4(f[4], f[5], f[6], f[7], inverse));
                }
            }
        }
        item += gridDim.y * WARPS;
        if (item >= 2 * a.kv_heads) return;
        load(0);
    }
}

template <typename T> int launch(const CmePaged* a, const CmePagedScales* s, cudaStream_t st) {
    // a sequence with n new tokens touches no more than n blocks and no more than n / block + 2
    const long long units = std::min((long long)a->rows, (long long)a->rows / s->block + 2ll * std::min(a->seqs, a->rows));
    // Where there are more warps than run at a time, one has several heads of its block, and looks it up once.
    int sms;
    if (const int rc = cme_num_sms(&sms)) return rc;
    const int most = cme_cdiv(2ll * a->kv_heads, WARPS);
    int across = most;
    while (across > 1 && units * across > sms * RESIDENT) across = (across + 1) / 2;
    const dim3 grid((unsigned)units, across);
    // (rows of up to 256 bytes in blocks of 16 tokens or fewer: half as many registers, more warps on an SM)
    const bool small = (long long)s->block * a->head_dim * sizeof(T) <= 4 * 512;
    auto* kernel = a->head_dim == 32   ? (small ? paged_append8_kernel<T, 32, 4> : paged_append8_kernel<T, 32, 8>)
                   : a->head_dim == 64 ? (small ? paged_append8_kernel<T, 64, 4> : paged_append8_kernel<T, 64, 8>)
                                       : (small ? paged_append8_kernel<T, 128, 4> : paged_append8_kernel<T, 128, 8>);
    CME_CUDA(cme_launch_dependent(kernel, grid, dim3(WARPS * 32), 0, st, *a, *s, paged_div(a->page), paged_div(s->block)));
    CME_LAUNCH_CHECK();
    return CME_OK;
}

}  // namespace

CME_API int cme_paged_append8(const CmePaged* a, const CmePagedScales* scales, void* stream) {
    const int rc = paged_check_cache(a, scales, "cache append");
    if (rc) return rc;
    if (a->rows == 0 || a->seqs == 0 || a->num_pages == 0 || a->width == 0) return CME_OK;
    return a->dtype == CME_F32 ? launch<float>(a, scales, (cudaStream_t)stream) : launch<__nv_bfloat16>(a, scales, (cudaStream_t)stream);
}
