// Attention of new tokens over a paged cache on warp-level matrix instructions: any of the head sizes, bf16 and fp32.
//
//     s_t = scale q . k_t,   out = sum_t exp(s_t - m) v_t / l,   m = max s_t,   l = sum exp(s_t - m),   lse = m + log l
//
// over the keys t up to the token's own position whose page is in the cache.  The query heads that share a key head are rows of one
// tile, so that a key is read once for all of them.  Two forms:
//   single  up to 16 rows a CTA, each of four warps takes a quarter of every key tile and keeps its own m, l and sums; they are
//           joined at the end.  For single tokens, which are bound by the bytes of the cache.
//   rows    64 rows a CTA, 16 a warp, every warp takes all keys.  For chunks that the tcgen05 kernel does not take.
// The fifth warp looks up the pages and loads key tiles by TMA, one box per page (or key tile), several tiles ahead.
// fp32 operands are split into two tf32 numbers each (x = hi + lo, 11 bits each) and multiplied as hi hi + hi lo + lo hi: what is
// left out is below 2^-22 of a product.  The tensor core's sums are kept short (one key tile, added up in fp32 registers), since it cuts
// what it shifts out.
// Long axes: the keys of a tile of rows are divided among up to eight CTAs of a cluster, which join their parts through each other's shared
// memory, or among any number of CTAs that leave them in scratch for a second kernel.
// Every wait is bounded; on expiry the CTA flags the status word and returns.
#include "paged.h"
#include "sm100_ptx.cuh"

#include <algorithm>
#include <cooperative_groups.h>
#include <mutex>

using namespace sm100;
namespace cg = cooperative_groups;

int* cme_attn_status_ptr();

namespace {

constexpr float LOG2E = 1.4426950408889634f;
constexpr int THREADS = 160;               // four warps that compute, one that loads

template <typename T, int D, bool ROWS> struct Cfg {
    static constexpr int ROW = D * (int)sizeof(T);                    // bytes of a key
    static constexpr int SLAB = ROW < 128 ? ROW : 128;                // bytes of a key in one swizzled slab
    static constexpr int SLABS = ROW / SLAB;
    static constexpr int WARP_KEYS = ROW <= 128 ? 32 : 16;            // keys that a warp takes at a time
    static constexpr int KEYS = 4 * WARP_KEYS;                        // key tile
    static constexpr int TILE = KEYS * ROW;                           // bytes of its keys (and of its values)
    static constexpr int STAGES = ROW == 64 ? 4 : ROWS && ROW == 512 ? 2 : 3;      // (the rows' fragments take 64 KB then)
    static constexpr bool F32 = sizeof(T) == 4;
    static_assert(STAGES <= 4, "words kept for the stages");
};

struct MmaParams {
    CmePaged a;
    PagedDiv page;
    int group, box, box_log, splits, cluster, split_keys;
    float scale_log2;
    float* part_o;                         // [rows, heads, splits, head_dim] sums of a part
    float2* part_ml;                       // [rows, heads, splits] its m (log2 units) and l
    int* status;
};

// Address of 16-byte chunk `c` of key `r`, as TMA's 128-byte (64-byte for 64-byte keys) swizzle lays it down.
template <typename C> __device__ __forceinline__ uint32_t chunk_at(int r, int c) {
    if (C::SLAB == 64) return (uint32_t)(r * 64 + ((c ^ ((r >> 1) & 3)) << 4));
    return (uint32_t)((c >> 3) * (C::KEYS * 128) + r * 128 + (((c & 7) ^ (r & 7)) << 4));
}
__device__ __forceinline__ void tma_load_4d(uint32_t dst, const CUtensorMap* m, uint64_t* bar, int c0, int c1, int c2, int c3) {
    asm volatile(
        "cp.async.bulk.tensor.4d.shared::cta.global.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4, %5, %6}], [%2];"
        ::"r"(dst), "l"(reinterpret_cast<uint64_t>(m)), "r"(smem_u32(bar)), "r"(c0), "r"(c1), "r"(c2), "r"(c3)
        : "memory");
}
__device__ __forceinline__ void ldsm4(uint32_t addr, uint32_t* r) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0, %1, %2, %3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr) : "memory");
}
__device__ __forceinline__ void ldsm4_t(uint32_t addr, uint32_t* r) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0, %1, %2, %3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr) : "memory");
}
__device__ __forceinline__ uint32_t lds32(uint32_t addr) {
    uint32_t v;
    asm volatile("ld.shared.b32 %0, [%1];" : "=r"(v) : "r"(addr) : "memory");
    return v;
}
__device__ __forceinline__ void mma_bf16(float* c, const uint32_t* a, uint32_t b0, uint32_t b1) {
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3]) : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ void mma_tf32(float* c, const uint32_t* a, uint32_t b0, uint32_t b1) {
    asm volatile("mma.sync.aligned.m16n8k8.row.col.f32.tf32.tf32.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3]) : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
// x as the sum of two tf32 numbers.  An infinity has no low part (its difference to itself would be NaN).
__device__ __forceinline__ void split_tf32(float x, uint32_t& hi, uint32_t& lo) {
    asm("cvt.rna.tf32.f32 %0, %1;" : "=r"(hi) : "f"(x));
    const float d = x - __uint_as_float(hi);
    asm("cvt.rna.tf32.f32 %0, %1;" : "=r"(lo) : "f"(d));
    if (fabsf(x) >= 3.4e38f) { hi = __float_as_uint(x); lo = 0; }
}

// ROWS: 16 rows per warp and all keys, else 16 rows per CTA and a quarter of the keys per warp.
// Four finished columns of a row.
template <typename T> __device__ __forceinline__ void store4(T* dst, float4 v, float f) {
    if constexpr (sizeof(T) == 4) *reinterpret_cast<float4*>(dst) = make_float4(v.x * f, v.y * f, v.z * f, v.w * f);
    else *reinterpret_cast<uint2*>(dst) = make_uint2(f2_to_bf2(v.x * f, v.y * f), f2_to_bf2(v.z * f, v.w * f));
}
// What the sums of a row are multiplied by, and its log-sum-exp.  Nothing seen: zeros and -inf; a NaN goes through.
__device__ __forceinline__ float inverse(float l) { return l == 0.f ? 0.f : 1.f / l; }
__device__ __forceinline__ float log_sum(float m, float l) {
    return l == 0.f ? -INFINITY : (m == -INFINITY ? l : (m + log2f(l)) / LOG2E);
}
// Factor of a part whose maximum is m where the largest is mm.
__device__ __forceinline__ float part_factor(float m, float mm) { return ex2_approx(m - (mm == -INFINITY ? 0.f : mm)); }
__device__ __forceinline__ void add4(float4& v, float f, const float4& x) {
    v.x = fmaf(f, x.x, v.x); v.y = fmaf(f, x.y, v.y); v.z = fmaf(f, x.z, v.z); v.w = fmaf(f, x.w, v.w);
}

template <typename T, int D, bool ROWS>
__global__ void __launch_bounds__(THREADS, Cfg<T, D, ROWS>::STAGES * Cfg<T, D, ROWS>::TILE * 2 > 100 * 1024 || ROWS ? 1 : 2)
paged_attn_mma_kernel(const __grid_constant__ CUtensorMap tmK, const __grid_constant__ CUtensorMap tmV, const MmaParams p) {
    using C = Cfg<T, D, ROWS>;
    constexpr int KS = D / (C::F32 ? 8 : 16);              // steps of the score product along the head
    constexpr int NT = D / 8;                              // column tiles of the output
    extern __shared__ __align__(1024) uint8_t smem[];
    uint8_t* sK = smem;
    uint8_t* sV = sK + C::STAGES * C::TILE;
    uint8_t* sQ = sV + C::STAGES * C::TILE;                // fp32: the rows' fragments, high and low parts
    constexpr int QWARPS = ROWS ? 4 : 1;
    constexpr int QBYTES = C::F32 ? QWARPS * KS * 32 * 32 : 0;
    uint64_t* full = reinterpret_cast<uint64_t*>(sQ + QBYTES);
    uint64_t* empty = full + C::STAGES;
    uint32_t* there = reinterpret_cast<uint32_t*>(empty + C::STAGES);      // [stage] which of its boxes' pages are in the cache
    volatile int* abort_flag = reinterpret_cast<volatile int*>(there + 7);
    float* sML = reinterpret_cast<float*>(there + 8);   // [4 warps, then the CTA][16 rows][2]: m and l

    const int warp = __shfl_sync(0xffffffffu, threadIdx.x >> 5, 0), lane = threadIdx.x & 31;
    const CmePaged& a = p.a;
    const int split = blockIdx.x % p.splits, head = blockIdx.y;
    if (threadIdx.x == 0) {
        *abort_flag = 0;
        for (int s = 0; s < C::STAGES; ++s) { mbar_init(&full[s], 1); mbar_init(&empty[s], 4); }
        fence_barrier_init();
        prefetch_tmap(&tmK);
        prefetch_tmap(&tmV);
    }
    pdl_wait();
    const PagedTile t = paged_find_tile(a, blockIdx.x / p.splits, p.group, ROWS ? 64 : 16);
    __syncthreads();
    if (t.rows == 0) return;                               // all CTAs of a cluster
    // keys [0, limit) are seen by the last row; this CTA takes [begin, end)
    const int limit = max(0, min(t.length, t.length - t.n + (t.first + t.rows - 1) / p.group + 1));
    int span = p.split_keys;
    if (p.cluster) span = cme_cdiv_dev(cme_cdiv_dev(limit, C::KEYS), p.splits) * C::KEYS;
    const int begin = (int)min((long long)limit, (long long)split * span), end = (int)min((long long)limit, (long long)begin + span);
    const int tiles = cme_cdiv_dev(end - begin, C::KEYS);

    // what a computing warp ends with
    float m[2] = {-INFINITY, -INFINITY}, l[2] = {0.f, 0.f};
    float o[NT][4];
#pragma unroll
    for (int j = 0; j < NT; ++j) { o[j][0] = o[j][1] = o[j][2] = o[j][3] = 0.f; }
    const int g = lane >> 2, tq = lane & 3;
    const int row0 = (ROWS ? warp * 16 : 0) + g;           // this thread's rows of the tile: row0, row0 + 8

    if (warp == 4) {
        // lanes 0-15 load keys, 16-31 values, a lane one box (of up to 16) of each tile
        const int b = lane & 15;
        const CUtensorMap* map = lane < 16 ? &tmK : &tmV;
        const uint32_t base = smem_u32(lane < 16 ? sK : sV) + b * p.box * C::SLAB;
        bool ok = true;
        for (int j = 0; j < tiles; ++j) {
            const int s = j % C::STAGES, k0 = begin + j * C::KEYS;
            if (j >= C::STAGES) ok = mbar_wait(&empty[s], (j / C::STAGES - 1) & 1, abort_flag);
            ok = __all_sync(0xffffffffu, ok);
            if (!ok) break;
            const int boxes = cme_cdiv_dev(min(C::KEYS, end - k0), p.box);
            int page = 0, slot = 0;
            if (b < boxes) {
                const int key = k0 + b * p.box, col = p.page.div(key);
                slot = key - col * p.page.d;
                page = a.pages[t.seq * a.pages_ld + col];
                if (page < 0 || page >= a.num_pages) page = a.num_pages;       // behind the cache: TMA fills the box with zeros
            }
            const uint32_t mask = __ballot_sync(0xffffffffu, page != a.num_pages);
            if (lane == 0) {
                there[s] = mask;
                mbar_arrive_expect_tx(&full[s], (uint32_t)(boxes * p.box * C::ROW * 2));
            }
            __syncwarp();
            if (b < boxes) {
#pragma unroll
                for (int c = 0; c < C::SLABS; ++c)
                    tma_load_4d(base + s * C::TILE + c * C::KEYS * 128, map, &full[s], c * (128 / (int)sizeof(T)), slot, head, page);
            }
        }
        if (!ok && lane == 0) for (int i = 0; i < 2000; ++i) __nanosleep(500);   // copies in flight end before the CTA does
    } else {
        // ---------------- the rows of Q, as A fragments ----------------
        uint32_t qf[C::F32 ? 1 : KS][4];
        const T* q = static_cast<const T*>(a.q);
        auto row_ptr = [&](int r) -> const T* {            // row r of the tile, or null
            if (r >= t.rows) return nullptr;
            const int rr = t.first + r, tok = rr / p.group;
            return q + (t.token0 + tok) * a.q_token + (head * p.group + rr - tok * p.group) * a.q_head;
        };
        const T* qa = row_ptr(row0);
        const T* qb = row_ptr(row0 + 8);
        if constexpr (C::F32) {
            float4* frag = reinterpret_cast<float4*>(sQ) + (ROWS ? warp * KS * 64 : 0);
            for (int ks = ROWS ? 0 : warp; ks < KS; ks += ROWS ? 1 : 4) {
                const int c = ks * 8 + tq;
                const float x[4] = {qa ? (float)qa[c] : 0.f, qb ? (float)qb[c] : 0.f, qa ? (float)qa[c + 4] : 0.f, qb ? (float)qb[c + 4] : 0.f};
                uint32_t hi[4], lo[4];
#pragma unroll
                for (int i = 0; i < 4; ++i) split_tf32(x[i], hi[i], lo[i]);
                frag[(ks * 2) * 32 + lane] = *reinterpret_cast<float4*>(hi);
                frag[(ks * 2 + 1) * 32 + lane] = *reinterpret_cast<float4*>(lo);
            }
            if (ROWS) __syncwarp();
            else named_bar_sync(1, 128);
        } else {
#pragma unroll
            for (int ks = 0; ks < KS; ++ks) {
                const int c = ks * 16 + tq * 2;
                qf[ks][0] = qa ? *reinterpret_cast<const uint32_t*>(qa + c) : 0u;
                qf[ks][1] = qb ? *reinterpret_cast<const uint32_t*>(qb + c) : 0u;
                qf[ks][2] = qa ? *reinterpret_cast<const uint32_t*>(qa + c + 8) : 0u;
                qf[ks][3] = qb ? *reinterpret_cast<const uint32_t*>(qb + c + 8) : 0u;
            }
        }
        // keys [0, see) are visible to a row; no row sees one at `end` or beyond
        const int see0 = min(end, t.length - t.n + (t.first + row0) / p.group + 1);
        const int see1 = min(end, t.length - t.n + (t.first + row0 + 8) / p.group + 1);
        const int see_first = t.length - t.n + (t.first + (ROWS ? warp * 16 : 0)) / p.group + 1;
        const uint32_t kbase = smem_u32(sK), vbase = smem_u32(sV);

        for (int j = 0; j < tiles; ++j) {
            const int s = j % C::STAGES, k0 = begin + j * C::KEYS;
            if (!mbar_wait(&full[s], (j / C::STAGES) & 1, abort_flag)) break;
            const uint32_t mask = there[s];
            const uint32_t kt = kbase + s * C::TILE, vt = vbase + s * C::TILE;
            if (k0 + C::KEYS > end) {
                // values behind the end may be anything, NaN too, which a probability of zero does not stop: zeros take their place.
                // A warp clears what it will read; warps that share keys write the same zeros.
                const int lo = ROWS ? 0 : warp * C::WARP_KEYS, hi = ROWS ? C::KEYS : lo + C::WARP_KEYS;
                for (int i = max(lo, end - k0) * (C::ROW / 16) + lane; i < hi * (C::ROW / 16); i += 32) {
                    const int r = i / (C::ROW / 16), c = i % (C::ROW / 16);
                    *reinterpret_cast<uint4*>(sV + s * C::TILE + chunk_at<C>(r, c)) = make_uint4(0, 0, 0, 0);
                }
                __syncwarp();
            }
#pragma unroll 1
            for (int part = 0; part < (ROWS ? 4 : 1); ++part) {
                const int key0 = (ROWS ? part : warp) * C::WARP_KEYS;      // first key of this part of the tile
                if (k0 + key0 >= end) break;
                constexpr int NK = C::WARP_KEYS / 8;
                float sc[NK][4];
#pragma unroll
                for (int n = 0; n < NK; ++n) { sc[n][0] = sc[n][1] = sc[n][2] = sc[n][3] = 0.f; }
                if constexpr (C::F32) {
                    const float4* frag = reinterpret_cast<const float4*>(sQ) + (ROWS ? warp * KS * 64 : 0);
                    float sl[NK][4];                       // the products with a low part
#pragma unroll
                    for (int n = 0; n < NK; ++n) { sl[n][0] = sl[n][1] = sl[n][2] = sl[n][3] = 0.f; }
#pragma unroll 2
                    for (int ks = 0; ks < KS; ks += 2) {
                        float4 f[4];
#pragma unroll
                        for (int i = 0; i < 4; ++i) f[i] = frag[(ks * 2 + i) * 32 + lane];
                        const uint32_t* qh0 = reinterpret_cast<const uint32_t*>(&f[0]);
                        const uint32_t* ql0 = reinterpret_cast<const uint32_t*>(&f[1]);
                        const uint32_t* qh1 = reinterpret_cast<const uint32_t*>(&f[2]);
                        const uint32_t* ql1 = reinterpret_cast<const uint32_t*>(&f[3]);
#pragma unroll
                        for (int n = 0; n < NK; ++n) {
                            uint32_t b[4], h[4], w[4];
                            ldsm4(kt + chunk_at<C>(key0 + n * 8 + (lane & 7), ks * 2 + (lane >> 3)), b);
#pragma unroll
                            for (int i = 0; i < 4; ++i) split_tf32(__uint_as_float(b[i]), h[i], w[i]);
                            mma_tf32(sc[n], qh0, h[0], h[1]);
                            mma_tf32(sl[n], qh0, w[0], w[1]);
                            mma_tf32(sl[n], ql0, h[0], h[1]);
                            mma_tf32(sc[n], qh1, h[2], h[3]);
                            mma_tf32(sl[n], qh1, w[2], w[3]);
                            mma_tf32(sl[n], ql1, h[2], h[3]);
                        }
                    }
#pragma unroll
                    for (int n = 0; n < NK; ++n)
#pragma unroll
                        for (int i = 0; i < 4; ++i) sc[n][i] += sl[n][i];
                } else {
#pragma unroll
                    for (int ks = 0; ks < KS; ++ks)
#pragma unroll
                        for (int n = 0; n < NK; n += 2) {
                            uint32_t b[4];
                            ldsm4(kt + chunk_at<C>(key0 + n * 8 + ((lane >> 4) << 3) + (lane & 7), ks * 2 + ((lane >> 3) & 1)), b);
                            mma_bf16(sc[n], qf[ks], b[0], b[1]);
                            mma_bf16(sc[n + 1], qf[ks], b[2], b[3]);
                        }
                }
                // what a row does not see
                if (mask != 0xffffffffu || k0 + key0 + C::WARP_KEYS > min(end, see_first)) {
#pragma unroll
                    for (int n = 0; n < NK; ++n)
#pragma unroll
                        for (int i = 0; i < 2; ++i) {
                            const int local = key0 + n * 8 + tq * 2 + i, key = k0 + local;
                            const bool in = (mask >> (local >> p.box_log)) & 1;
                            if (!in || key >= see0) sc[n][i] = -INFINITY;
                            if (!in || key >= see1) sc[n][2 + i] = -INFINITY;
                        }
                }
                float mx[2] = {-INFINITY, -INFINITY};
#pragma unroll
                for (int n = 0; n < NK; ++n)
#pragma unroll
                    for (int i = 0; i < 2; ++i) {
                        mx[0] = fmaxf(mx[0], sc[n][i]);
                        mx[1] = fmaxf(mx[1], sc[n][2 + i]);
                    }
                bool raise = false;
                float alpha[2], use[2];
#pragma unroll
                for (int r = 0; r < 2; ++r) {
                    mx[r] = fmaxf(mx[r], __shfl_xor_sync(0xffffffffu, mx[r], 1));
                    mx[r] = fmaxf(mx[r], __shfl_xor_sync(0xffffffffu, mx[r], 2));
                    mx[r] *= p.scale_log2;                 // scale > 0, so the maximum commutes with it
                    const bool up = mx[r] > m[r];
                    raise |= up;
                    alpha[r] = up ? (m[r] == -INFINITY ? 0.f : ex2_approx(m[r] - mx[r])) : 1.f;
                    if (up) m[r] = mx[r];
                    use[r] = m[r] == -INFINITY ? 0.f : m[r];
                }
                if (__any_sync(0xffffffffu, raise)) {
                    l[0] *= alpha[0];
                    l[1] *= alpha[1];
#pragma unroll
                    for (int n = 0; n < NT; ++n) { o[n][0] *= alpha[0]; o[n][1] *= alpha[0]; o[n][2] *= alpha[1]; o[n][3] *= alpha[1]; }
                }
#pragma unroll
                for (int n = 0; n < NK; ++n) {
#pragma unroll
                    for (int i = 0; i < 4; ++i) sc[n][i] = ex2_approx(fmaf(sc[n][i], p.scale_log2, -use[i >> 1]));
                    l[0] += sc[n][0] + sc[n][1];
                    l[1] += sc[n][2] + sc[n][3];
                }
                if constexpr (C::F32) {
                    // A step covers eight keys; slot t of it stands for key 2t and slot t + 4 for key 2t + 1, so that a thread's
                    // probabilities are its A fragment as they are, and the four rows of V that a warp reads at once lie in
                    // different banks.
                    uint32_t ph[NK][4], pl[NK][4];
#pragma unroll
                    for (int n = 0; n < NK; ++n) {
                        split_tf32(sc[n][0], ph[n][0], pl[n][0]);
                        split_tf32(sc[n][2], ph[n][1], pl[n][1]);
                        split_tf32(sc[n][1], ph[n][2], pl[n][2]);
                        split_tf32(sc[n][3], ph[n][3], pl[n][3]);
                    }
#pragma unroll
                    for (int d = 0; d < NT; ++d) {
                        float acc[4] = {0.f, 0.f, 0.f, 0.f}, low[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
                        for (int n = 0; n < NK; ++n) {
                            const int key = key0 + n * 8 + 2 * tq, c = d * 2 + (g >> 2);
                            uint32_t h0, w0, h1, w1;
                            split_tf32(__uint_as_float(lds32(vt + chunk_at<C>(key, c) + (g & 3) * 4)), h0, w0);
                            split_tf32(__uint_as_float(lds32(vt + chunk_at<C>(key + 1, c) + (g & 3) * 4)), h1, w1);
                            mma_tf32(acc, ph[n], h0, h1);
                            mma_tf32(low, ph[n], w0, w1);
                            mma_tf32(low, pl[n], h0, h1);
                        }
#pragma unroll
                        for (int i = 0; i < 4; ++i) o[d][i] += acc[i] + low[i];
                    }
                } else {
                    // probabilities as bf16, the operand's type; their sum l is of the unrounded ones
#pragma unroll
                    for (int n = 0; n < NK; n += 2) {
                        const uint32_t pa[4] = {f2_to_bf2(sc[n][0], sc[n][1]), f2_to_bf2(sc[n][2], sc[n][3]),
                                                f2_to_bf2(sc[n + 1][0], sc[n + 1][1]), f2_to_bf2(sc[n + 1][2], sc[n + 1][3])};
#pragma unroll
                        for (int d = 0; d < NT; d += 2) {
                            uint32_t b[4];
                            ldsm4_t(vt + chunk_at<C>(key0 + n * 8 + (((lane >> 3) & 1) << 3) + (lane & 7), d + (lane >> 4)), b);
                            mma_bf16(o[d], pa, b[0], b[1]);
                            mma_bf16(o[d + 1], pa, b[2], b[3]);
                        }
                    }
                }
            }
            __syncwarp();
            if (lane == 0) mbar_arrive(&empty[s]);
        }
#pragma unroll
        for (int r = 0; r < 2; ++r) {
            l[r] += __shfl_xor_sync(0xffffffffu, l[r], 1);
            l[r] += __shfl_xor_sync(0xffffffffu, l[r], 2);
        }
    }

    // ---------------- ends ----------------
    auto where = [&](int r, long long& row_head) {         // row r of the tile: index of (token, head)
        const int rr = t.first + r, tok = rr / p.group;
        row_head = (long long)(t.token0 + tok) * a.heads + head * p.group + rr - tok * p.group;
    };
    T* out = static_cast<T*>(a.o);
    if constexpr (ROWS) {
        if (warp < 4) {
#pragma unroll
            for (int r = 0; r < 2; ++r) {
                const int row = row0 + 8 * r;
                if (row >= t.rows) continue;
                long long at;
                where(row, at);
                if (p.splits == 1) {
                    const float inv = inverse(l[r]);
#pragma unroll
                    for (int d = 0; d < NT; ++d) {
                        T* dst = out + at * D + d * 8 + tq * 2;
                        if constexpr (C::F32) *reinterpret_cast<float2*>(dst) = make_float2(o[d][2 * r] * inv, o[d][2 * r + 1] * inv);
                        else *reinterpret_cast<uint32_t*>(dst) = f2_to_bf2(o[d][2 * r] * inv, o[d][2 * r + 1] * inv);
                    }
                    if (tq == 0) a.lse[at] = log_sum(m[r], l[r]);
                } else {
                    at = at * p.splits + split;
                    if (tiles > 0) {
#pragma unroll
                        for (int d = 0; d < NT; ++d)
                            *reinterpret_cast<float2*>(p.part_o + at * D + d * 8 + tq * 2) = make_float2(o[d][2 * r], o[d][2 * r + 1]);
                    }
                    if (tq == 0) p.part_ml[at] = make_float2(m[r], l[r]);
                }
            }
        }
    } else {
        // join the four warps: every load has been waited for, so the key tiles' memory is free
        float* part = reinterpret_cast<float*>(smem);      // [4][rows][D]
        float* own = part + 4 * 16 * D;                    // [rows][D]: this CTA's sums
        float* own_ml = sML + 4 * 32;                      // [rows][2]
        __syncthreads();
        if (warp < 4) {
#pragma unroll
            for (int r = 0; r < 2; ++r) {
                const int row = g + 8 * r;
                if (row >= t.rows) continue;
#pragma unroll
                for (int d = 0; d < NT; ++d)
                    *reinterpret_cast<float2*>(part + (warp * 16 + row) * D + d * 8 + tq * 2) = make_float2(o[d][2 * r], o[d][2 * r + 1]);
                if (tq == 0) { sML[(warp * 16 + row) * 2] = m[r]; sML[(warp * 16 + row) * 2 + 1] = l[r]; }
            }
        }
        __syncthreads();
        const bool cluster = p.cluster && p.splits > 1;
        for (int i = threadIdx.x; i < t.rows * (D / 4); i += THREADS) {
            const int row = i / (D / 4), c = i % (D / 4) * 4;
            float mm = -INFINITY, ll = 0.f;
#pragma unroll
            for (int w = 0; w < 4; ++w) mm = fmaxf(mm, sML[(w * 16 + row) * 2]);
            float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
            for (int w = 0; w < 4; ++w) {
                const float f = part_factor(sML[(w * 16 + row) * 2], mm);
                ll = fmaf(f, sML[(w * 16 + row) * 2 + 1], ll);
                add4(v, f, *reinterpret_cast<const float4*>(part + (w * 16 + row) * D + c));
            }
            long long at;
            where(row, at);
            if (p.splits == 1) {
                store4(out + at * D + c, v, inverse(ll));
                if (c == 0) a.lse[at] = log_sum(mm, ll);
            } else if (cluster) {
                *reinterpret_cast<float4*>(own + row * D + c) = v;
                if (c == 0) { own_ml[row * 2] = mm; own_ml[row * 2 + 1] = ll; }
            } else {
                at = at * p.splits + split;
                if (tiles > 0) *reinterpret_cast<float4*>(p.part_o + at * D + c) = v;
                if (c == 0) p.part_ml[at] = make_float2(mm, ll);
            }
        }
        if (cluster) {
            // the parts of the cluster's CTAs, each CTA joins its share of the elements
            cg::cluster_group cl = cg::this_cluster();
            cl.sync();
            for (int i = split * THREADS + threadIdx.x; i < t.rows * (D / 4); i += p.splits * THREADS) {
                const int row = i / (D / 4), c = i % (D / 4) * 4;
                float mm = -INFINITY, ll = 0.f;
                float2 ml[8];
#pragma unroll
                for (int k = 0; k < 8; ++k) {
                    ml[k] = make_float2(-INFINITY, 0.f);
                    if (k < p.splits) ml[k] = *reinterpret_cast<const float2*>(cl.map_shared_rank(own_ml + row * 2, k));
                    mm = fmaxf(mm, ml[k].x);
                }
                float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
                for (int k = 0; k < 8; ++k) {
                    if (k >= p.splits) break;
                    const float f = part_factor(ml[k].x, mm);
                    ll = fmaf(f, ml[k].y, ll);
                    add4(v, f, *reinterpret_cast<const float4*>(cl.map_shared_rank(own + row * D + c, k)));
                }
                long long at;
                where(row, at);
                store4(out + at * D + c, v, inverse(ll));
                if (c == 0) a.lse[at] = log_sum(mm, ll);
            }
            cl.sync();                                     // nobody's shared memory goes while it is read
        }
    }
    if (threadIdx.x == 0 && *abort_flag && p.status) atomicExch(p.status, CME_ERR_TIMEOUT);
}

// Joins the parts of a row that CTAs left in scratch: one warp per row.  A part that summed nothing has left no sums either.
template <typename T, int D>
__global__ void __launch_bounds__(128) paged_join_kernel(const float* __restrict__ part_o, const float2* __restrict__ part_ml, T* out,
                                                         float* lse, long long rows, int splits) {
    constexpr int VEC = D / 32;
    pdl_wait();
    const int lane = threadIdx.x & 31;
    const long long row = (long long)blockIdx.x * 4 + (threadIdx.x >> 5);
    if (row >= rows) return;
    const float2* ml = part_ml + row * splits;
    float mm = -INFINITY;
    for (int s = lane; s < splits; s += 32) mm = fmaxf(mm, ml[s].x);
    mm = warp_max(mm);
    float v[VEC] = {}, l = 0.f;
#pragma unroll 4
    for (int s = 0; s < splits; ++s) {
        const float2 part = ml[s];
        if (part.y == 0.f) continue;
        const float f = part_factor(part.x, mm);
        l = fmaf(f, part.y, l);
        const float* src = part_o + (row * splits + s) * D + lane * VEC;
#pragma unroll
        for (int i = 0; i < VEC; ++i) v[i] = fmaf(f, src[i], v[i]);
    }
    const float inv = inverse(l);
#pragma unroll
    for (int i = 0; i < VEC; ++i) out[row * D + lane * VEC + i] = from_f32<T>(v[i] * inv);
    if (lane == 0) lse[row] = log_sum(mm, l);
}

// ------------------------------------------------------------------------------------------------------
// Host side
// ------------------------------------------------------------------------------------------------------
template <typename T, int D, bool ROWS> constexpr int smem_bytes() {
    using C = Cfg<T, D, ROWS>;
    const int q = C::F32 ? (ROWS ? 4 : 1) * (D / 8) * 32 * 32 : 0;
    return C::STAGES * C::TILE * 2 + q + C::STAGES * 16 + 32 + (4 * 32 + 32) * 4;
}

template <typename T, int D, bool ROWS> int launch(const CmePaged* a, const PagedPlan& plan, const MmaParams& p, cudaStream_t st) {
    using C = Cfg<T, D, ROWS>;
    constexpr int SMEM = smem_bytes<T, D, ROWS>();
    static_assert(SMEM <= 227 * 1024, "shared memory of a CTA");
    auto* kernel = paged_attn_mma_kernel<T, D, ROWS>;
    static bool attr[CME_MAX_DEVICES] = {};               // function attributes are per device
    int dev = 0;
    CME_CUDA(cudaGetDevice(&dev));
    if (!attr[dev % CME_MAX_DEVICES]) {
        CME_CUDA(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, SMEM));
        attr[dev % CME_MAX_DEVICES] = true;
    }
    CUtensorMap mk, mv;
    const auto swizzle = C::SLAB == 64 ? CU_TENSOR_MAP_SWIZZLE_64B : CU_TENSOR_MAP_SWIZZLE_128B;
    int rc;
    if ((rc = paged_make_map(&mk, a, a->k, a->k_page_stride, a->k_head_stride, a->k_slot_stride, C::SLAB / (int)sizeof(T), p.box, swizzle))) return rc;
    if ((rc = paged_make_map(&mv, a, a->v, a->v_page_stride, a->v_head_stride, a->v_slot_stride, C::SLAB / (int)sizeof(T), p.box, swizzle))) return rc;
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = dim3(plan.tiles * plan.splits, a->kv_heads);
    cfg.blockDim = dim3(THREADS);
    cfg.dynamicSmemBytes = SMEM;
    cfg.stream = st;
    cudaLaunchAttribute at[2];
    at[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    at[0].val.programmaticStreamSerializationAllowed = 1;
    at[1].id = cudaLaunchAttributeClusterDimension;
    at[1].val.clusterDim.x = plan.cluster ? plan.splits : 1;
    at[1].val.clusterDim.y = at[1].val.clusterDim.z = 1;
    cfg.attrs = at;
    cfg.numAttrs = plan.cluster && plan.splits > 1 ? 2 : 1;
    CME_CUDA(cudaLaunchKernelEx(&cfg, kernel, mk, mv, p));
    CME_LAUNCH_CHECK();
    return CME_OK;
}

}  // namespace

int paged_mma_key_tile(int dtype, int head_dim) { return head_dim * (dtype == CME_F32 ? 4 : 2) <= 128 ? 128 : 64; }

// The parts in `ws`: log-sum-exp pairs first (16-byte aligned by their size), then the sums.
int paged_join(const CmePaged* a, int splits, cudaStream_t st) {
    const long long rows = (long long)a->rows * a->heads;
    const float2* ml = reinterpret_cast<const float2*>(a->ws);
    const float* o = a->ws + (rows * splits * 2 + 3) / 4 * 4;
    const dim3 grid((unsigned)((rows + 3) / 4));
    const bool f32 = a->dtype == CME_F32;
#define JOIN(T, D) \
    CME_CUDA(cme_launch_dependent(paged_join_kernel<T, D>, grid, dim3(128), 0, st, o, ml, (T*)a->o, a->lse, rows, splits))
    if (a->head_dim == 32) { if (f32) JOIN(float, 32); else JOIN(__nv_bfloat16, 32); }
    else if (a->head_dim == 64) { if (f32) JOIN(float, 64); else JOIN(__nv_bfloat16, 64); }
    else { if (f32) JOIN(float, 128); else JOIN(__nv_bfloat16, 128); }
#undef JOIN
    CME_LAUNCH_CHECK();
    return CME_OK;
}

int paged_attention_mma(const CmePaged* a, const PagedPlan& plan, cudaStream_t st) {
    MmaParams p;
    p.a = *a;
    p.page = paged_div(a->page);
    p.group = a->heads / a->kv_heads;
    const int tile = paged_mma_key_tile(a->dtype, a->head_dim);
    p.box = 1;
    p.box_log = 0;
    while (p.box < tile && a->page % (p.box * 2) == 0) { p.box *= 2; ++p.box_log; }
    p.splits = plan.splits;
    p.cluster = plan.cluster;
    p.split_keys = plan.split_keys;
    p.scale_log2 = a->scale * LOG2E;
    const long long parts = (long long)a->rows * a->heads * plan.splits;
    p.part_ml = reinterpret_cast<float2*>(a->ws);
    p.part_o = a->ws + (parts * 2 + 3) / 4 * 4;
    p.status = cme_attn_status_ptr();
    CME_REQUIRE(p.status != nullptr, CME_ERR_CUDA, "paged attention: device state unavailable");
    const bool rows = plan.kernel == PAGED_ROWS;
#define GO(T, D) return rows ? launch<T, D, true>(a, plan, p, st) : launch<T, D, false>(a, plan, p, st)
    if (a->dtype == CME_F32) {
        if (a->head_dim == 32) GO(float, 32);
        if (a->head_dim == 64) GO(float, 64);
        GO(float, 128);
    }
    if (a->head_dim == 32) GO(__nv_bfloat16, 32);
    if (a->head_dim == 64) GO(__nv_bfloat16, 64);
    GO(__nv_bfloat16, 128);
#undef GO
}
