// Attention of new tokens over a paged cache on warp-level matrix instructions: any of the head sizes, bf16 and fp32.
//
//     s_t = scale q . k_t,   out = sum_t exp(s_t - m) v_t / l,   m = max s_t,   l = sum exp(s_t - m),   lse = m + log l
//
// over the keys t up to the token's own position whose page is in the cache.  The query heads that share a key head are rows of one
// tile, so that a key is read once for all of them.  Two forms:
//   single  up to 16 rows a tile, each of four warps takes a quarter of every key tile and keeps its own m, l and sums; they are
//           joined at the end.  For single tokens, which are bound by the bytes of the cache.
//   rows    64 rows a CTA, 16 a warp; in fp32 and head sizes above 32 two warps share 16 rows and take every other 16 or 32 keys.  For chunks
//           that the tcgen05 kernel does not take.
// The last warp looks up the pages and loads key tiles by TMA, one box per page (or key tile), several tiles ahead.
// fp32 operands of the matrix instructions are split into two tf32 numbers each (x = hi + lo, 11 bits each) and multiplied as hi hi + hi lo + lo hi.  What is
// left out is 2^-21 of a product at the most: 2^-22 for lo lo, 2^-23 for what each operand's lo cuts off.  The tensor core's sums are kept short (one key tile, added up in fp32 registers), since it cuts
// what it shifts out.
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

template <typename T, int D, bool ROWS> struct Cfg {
    static constexpr bool F32 = sizeof(T) == 4;
    static constexpr int ROW = D * (int)sizeof(T);                    // bytes of a key
    static constexpr int SLAB = ROW < 128 ? ROW : 128;                // bytes of a key in one swizzled slab
    static constexpr int SLABS = ROW / SLAB;
    static constexpr int WARP_KEYS = ROW <= 128 || (ROWS && F32 && D == 64) ? 32 : 16;      // keys that a warp takes at a time
    static constexpr int KEYS = ROW <= 128 ? 128 : 64;                // key tile
    static constexpr int TILE = KEYS * ROW;                           // bytes of its keys (and of its values)
    static constexpr int STAGES = ROW == 64 ? 4 : ROWS && ROW == 512 ? 2 : 3;      // (the rows' fragments take 64 KB then)
    static constexpr int FRAGS = F32 ? D * 128 : 0;                   // bytes of 16 rows' fragments in shared memory
    // CTAs of an SM, and groups of four warps, which take every other key tile (rows: every other WARP_KEYS keys of each).  Two CTAs' or two groups'
    // chains of products and softmax run at a time; 64 KB tiles, or 64 rows' fragments of fp32, leave room for one CTA.  Rows, fp32, one
    // group / two, us: 16 heads of 64, 512 tokens over 2048 in 4 sequences 469 / 384; 32 heads of 128 on 8, 500 over 2000 in 2 864 / 701;
    // 12 heads of 64, 64 over 128 in one 11.9 / 11.4.  (Head size 32 has room for two CTAs.)
    static constexpr int CTAS = ROWS ? (D == 32 ? 2 : 1) : ROW == 512 ? 1 : 2;
    static constexpr int GROUPS = (ROWS ? F32 && D > 32 : ROW == 512) ? 2 : 1, WARPS = 4 * GROUPS;
    static constexpr int JOIN_ROWS = 32 / WARPS;                      // joined at a time (up to 16 rows)
    static_assert(STAGES <= 4, "words kept for the stages");
};

struct MmaParams {
    CmePaged a;
    PagedDiv page, heads, parts;           // slots of a page; key heads and splits (rows)
    int group, box, box_log, splits, split_keys, tiles, by_keys;
    float scale_log2;
    float* part_o;                         // [rows, heads, splits, head_dim] sums of a part; stream: [CTA, 2, 16, head_dim]
    float2* part_ml;                       // [rows, heads, splits] its m (log2 units) and l; stream: [CTA, 2, 16]
    int* records;                          // stream: [CTA]
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
__device__ __forceinline__ float4 lds128(uint32_t addr) {
    float4 v;
    asm volatile("ld.shared.v4.f32 {%0, %1, %2, %3}, [%4];" : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w) : "r"(addr) : "memory");
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
// x as the sum of two tf32 numbers: the nearest one (half away from zero), and what is left, up to 2^-11 of x, cut off to its 11 upper bits.
// That is a multiple of x's last place of 13 bits at the most, which loses one last place, 2^-23 of x.  On the integer
// pipe: the conversion instruction runs at an eighth of its rate.  NaN stays (in the low part, if its bits overflow).
__device__ __forceinline__ void split_tf32(float x, uint32_t& hi, uint32_t& lo) {
    hi = (__float_as_uint(x) + 0x1000u) & 0xffffe000u;
    lo = __float_as_uint(x - __uint_as_float(hi)) & 0xffffe000u;
}

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

// ------------------------------------------------------------------------------------------------------
// One warp: 16 rows and WARP_KEYS keys of a tile in shared memory
// ------------------------------------------------------------------------------------------------------
template <typename C, int D> struct WarpState {
    static constexpr int NT = D / 8;                       // column tiles of the output
    float m[2], l[2], o[NT][4];                            // of rows lane / 4 and lane / 4 + 8; l of this lane's keys only
    __device__ __forceinline__ void clear() {
        m[0] = m[1] = -INFINITY;
        l[0] = l[1] = 0.f;
#pragma unroll
        for (int j = 0; j < NT; ++j) o[j][0] = o[j][1] = o[j][2] = o[j][3] = 0.f;
    }
    __device__ __forceinline__ void finish() {             // l of the whole row
#pragma unroll
        for (int r = 0; r < 2; ++r) {
            l[r] += __shfl_xor_sync(0xffffffffu, l[r], 1);
            l[r] += __shfl_xor_sync(0xffffffffu, l[r], 2);
        }
    }
};

// The rows' A fragments: bf16 in registers, fp32 in shared memory (high and low parts), made from PARTS warps' share of the elements.
template <typename T, typename C, int D, int PARTS> struct Rows {
    static constexpr int KS = D / (C::F32 ? 8 : 16);       // steps of the score product along the head
    uint32_t raw[C::F32 ? KS / PARTS : KS][4];             // bf16: the fragments
    const float4* frag;

    // On their way from memory; rows that are not there are zeros.
    __device__ __forceinline__ void load(const T* qa, const T* qb, int part) {
        const int tq = threadIdx.x & 3;
#pragma unroll
        for (int i = 0; i < (C::F32 ? KS / PARTS : KS); ++i) {
            const int c = C::F32 ? (i * PARTS + part) * 8 + tq : i * 16 + tq * 2, half = C::F32 ? 4 : 8;
            raw[i][0] = qa ? *reinterpret_cast<const uint32_t*>(qa + c) : 0u;
            raw[i][1] = qb ? *reinterpret_cast<const uint32_t*>(qb + c) : 0u;
            raw[i][2] = qa ? *reinterpret_cast<const uint32_t*>(qa + c + half) : 0u;
            raw[i][3] = qb ? *reinterpret_cast<const uint32_t*>(qb + c + half) : 0u;
        }
    }
    // fp32: into shared memory, for all who have their share there.
    __device__ __forceinline__ void publish(uint8_t* to, int part) {
        if constexpr (C::F32) {
            float4* f = reinterpret_cast<float4*>(to) + (threadIdx.x & 31);
            frag = reinterpret_cast<const float4*>(to);
#pragma unroll
            for (int i = 0; i < KS / PARTS; ++i) {
                uint32_t hi[4], lo[4];
#pragma unroll
                for (int e = 0; e < 4; ++e) split_tf32(__uint_as_float(raw[i][e]), hi[e], lo[e]);
                f[(i * PARTS + part) * 64] = *reinterpret_cast<float4*>(hi);
                f[(i * PARTS + part) * 64 + 32] = *reinterpret_cast<float4*>(lo);
            }
            if (PARTS > 1) named_bar_sync(1, PARTS * 32);
            else __syncwarp();
        }
    }
    // fp32: the first `rows` rows as they are.
    __device__ __forceinline__ void publish_rows(float* to, int part, int rows) {
        const int g = (threadIdx.x & 31) >> 2, tq = threadIdx.x & 3;
        if (g < rows) {
#pragma unroll
            for (int i = 0; i < KS / PARTS; ++i) {
                to[g * D + (i * PARTS + part) * 8 + tq] = __uint_as_float(raw[i][0]);
                to[g * D + (i * PARTS + part) * 8 + tq + 4] = __uint_as_float(raw[i][2]);
            }
        }
        named_bar_sync(1, PARTS * 32);
    }
};

// Keys [key0, key0 + WARP_KEYS) of the tile at kt / vt, whose first key is k0.  Keys [0, see0) are visible to this lane's first row, [0,
// see1) to its second; `masked` where some key of them is not visible to a row.
template <typename C, int D, typename R>
__device__ __forceinline__ void attend(WarpState<C, D>& w, const R& q, uint32_t kt, uint32_t vt, int key0, int k0, int see0,
                                       int see1, bool masked, uint32_t there, int box_log, float scale_log2) {
    constexpr int NK = C::WARP_KEYS / 8, NT = D / 8, KS = R::KS;
    const int lane = threadIdx.x & 31, g = lane >> 2, tq = lane & 3;
    float sc[NK][4];
#pragma unroll
    for (int n = 0; n < NK; ++n) sc[n][0] = sc[n][1] = sc[n][2] = sc[n][3] = 0.f;
    if constexpr (C::F32) {
        float sl[NK][4];                                   // the products with a low part
#pragma unroll
        for (int n = 0; n < NK; ++n) sl[n][0] = sl[n][1] = sl[n][2] = sl[n][3] = 0.f;
#pragma unroll
        for (int ks = 0; ks < KS; ks += 2) {
            float4 f[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) f[i] = q.frag[(ks * 2 + i) * 32 + lane];
            const uint32_t* qh0 = reinterpret_cast<const uint32_t*>(&f[0]);
            const uint32_t* ql0 = reinterpret_cast<const uint32_t*>(&f[1]);
            const uint32_t* qh1 = reinterpret_cast<const uint32_t*>(&f[2]);
            const uint32_t* ql1 = reinterpret_cast<const uint32_t*>(&f[3]);
#pragma unroll
            for (int n = 0; n < NK; ++n) {
                uint32_t b[4], h[4], lo[4];
                ldsm4(kt + chunk_at<C>(key0 + n * 8 + (lane & 7), ks * 2 + (lane >> 3)), b);
#pragma unroll
                for (int i = 0; i < 4; ++i) split_tf32(__uint_as_float(b[i]), h[i], lo[i]);
                mma_tf32(sc[n], qh0, h[0], h[1]);
                mma_tf32(sl[n], qh0, lo[0], lo[1]);
                mma_tf32(sl[n], ql0, h[0], h[1]);
                mma_tf32(sc[n], qh1, h[2], h[3]);
                mma_tf32(sl[n], qh1, lo[2], lo[3]);
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
                mma_bf16(sc[n], q.raw[ks], b[0], b[1]);
                mma_bf16(sc[n + 1], q.raw[ks], b[2], b[3]);
            }
    }
    if (masked) {
#pragma unroll
        for (int n = 0; n < NK; ++n)
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                const int local = key0 + n * 8 + tq * 2 + i, key = k0 + local;
                const bool in = (there >> (local >> box_log)) & 1;
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
        mx[r] *= scale_log2;                               // scale > 0, so the maximum commutes with it
        const bool up = mx[r] > w.m[r];
        raise |= up;
        alpha[r] = up ? (w.m[r] == -INFINITY ? 0.f : ex2_approx(w.m[r] - mx[r])) : 1.f;
        if (up) w.m[r] = mx[r];
        use[r] = w.m[r] == -INFINITY ? 0.f : w.m[r];
    }
    if (__any_sync(0xffffffffu, raise)) {
        w.l[0] *= alpha[0];
        w.l[1] *= alpha[1];
#pragma unroll
        for (int n = 0; n < NT; ++n) { w.o[n][0] *= alpha[0]; w.o[n][1] *= alpha[0]; w.o[n][2] *= alpha[1]; w.o[n][3] *= alpha[1]; }
    }
#pragma unroll
    for (int n = 0; n < NK; ++n) {
#pragma unroll
        for (int i = 0; i < 4; ++i) sc[n][i] = ex2_approx(fmaf(sc[n][i], scale_log2, -use[i >> 1]));
        w.l[0] += sc[n][0] + sc[n][1];
        w.l[1] += sc[n][2] + sc[n][3];
    }
    if constexpr (C::F32) {
        // A step covers eight keys; slot t of it stands for key 2t and slot t + 4 for key 2t + 1, so that a thread's probabilities are its
        // A fragment as they are, and the four rows of V that a warp reads at once lie in different banks.
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
            for (int i = 0; i < 4; ++i) w.o[d][i] += acc[i] + low[i];
        }
    } else {
        // Probabilities as bf16, the type of the other operand, V; their sum l is of the unrounded ones.  Errors against 64 bits are 0.0013 to 0.0022
        // of a result's size, 0.0011 to 0.0017 with probabilities in 32 bits (the result's own rounding).
#pragma unroll
        for (int n = 0; n < NK; n += 2) {
            const uint32_t pa[4] = {f2_to_bf2(sc[n][0], sc[n][1]), f2_to_bf2(sc[n][2], sc[n][3]),
                                    f2_to_bf2(sc[n + 1][0], sc[n + 1][1]), f2_to_bf2(sc[n + 1][2], sc[n + 1][3])};
#pragma unroll
            for (int d = 0; d < NT; d += 2) {
                uint32_t b[4];
                ldsm4_t(vt + chunk_at<C>(key0 + n * 8 + (((lane >> 3) & 1) << 3) + (lane & 7), d + (lane >> 4)), b);
                mma_bf16(w.o[d], pa, b[0], b[1]);
                mma_bf16(w.o[d + 1], pa, b[2], b[3]);
            }
        }
    }
}

// fp32 with R <= 4 rows on the CUDA cores: sixteen rows' worth of tf32 products would take longer than the tile's bytes (a 64 KB tile 2.1 us
// on the tensor cores for 1.5 us of memory; here 0.3 us a row).  Scores: a lane has a key (and, with 16 keys a warp, half of the columns).
// Sums: a lane has four columns, and with head sizes below 128 every second or fourth key.
template <typename C, int D, int R> struct SimtState {
    static constexpr int PER_KEY = 32 / C::WARP_KEYS, CL = D / 4, SUBSETS = 32 / CL;
    float m[R], l[R];
    float4 o[R];
    __device__ __forceinline__ void clear() {
#pragma unroll
        for (int r = 0; r < R; ++r) { m[r] = -INFINITY; l[r] = 0.f; o[r] = make_float4(0.f, 0.f, 0.f, 0.f); }
    }
    // As attend(); `see`: keys that a row sees, `q`: the rows in shared memory.
    __device__ __forceinline__ void attend(const float* q, uint32_t kt, uint32_t vt, int key0, int k0, const int* see, bool masked,
                                           uint32_t there, int box_log, float scale_log2) {
        const int lane = threadIdx.x & 31, key = key0 + lane % C::WARP_KEYS, c0 = lane / C::WARP_KEYS * (D / 4 / PER_KEY);
        float s[R];
#pragma unroll
        for (int r = 0; r < R; ++r) s[r] = 0.f;
#pragma unroll 8
        for (int c = c0; c < c0 + D / 4 / PER_KEY; ++c) {
            const float4 k = lds128(kt + chunk_at<C>(key, c));
#pragma unroll
            for (int r = 0; r < R; ++r) {
                const float4 x = *reinterpret_cast<const float4*>(q + r * D + c * 4);
                s[r] = fmaf(k.x, x.x, fmaf(k.y, x.y, fmaf(k.z, x.z, fmaf(k.w, x.w, s[r]))));
            }
        }
        bool raise = false;
        float alpha[R];
#pragma unroll
        for (int r = 0; r < R; ++r) {
            if (PER_KEY > 1) s[r] += __shfl_xor_sync(0xffffffffu, s[r], 16);
            if (masked && (!((there >> (key >> box_log)) & 1) || k0 + key >= see[r])) s[r] = -INFINITY;
            const float mx = warp_max(s[r]) * scale_log2;  // scale > 0, so the maximum commutes with it
            const bool up = mx > m[r];
            raise |= up;
            alpha[r] = up ? (m[r] == -INFINITY ? 0.f : ex2_approx(m[r] - mx)) : 1.f;
            if (up) m[r] = mx;
            s[r] = ex2_approx(fmaf(s[r], scale_log2, m[r] == -INFINITY ? 0.f : -m[r]));
            l[r] = fmaf(l[r], alpha[r], s[r]);
        }
        if (raise) {                                       // (the same in all lanes)
#pragma unroll
            for (int r = 0; r < R; ++r) { o[r].x *= alpha[r]; o[r].y *= alpha[r]; o[r].z *= alpha[r]; o[r].w *= alpha[r]; }
        }
#pragma unroll 8
        for (int i = 0; i < C::WARP_KEYS; i += SUBSETS) {
            const int k = i + lane / CL;
            const float4 v = lds128(vt + chunk_at<C>(key0 + k, lane % CL));
#pragma unroll
            for (int r = 0; r < R; ++r) add4(o[r], __shfl_sync(0xffffffffu, s[r], k), v);
        }
    }
    __device__ __forceinline__ void finish() {
#pragma unroll
        for (int r = 0; r < R; ++r) {
#pragma unroll
            for (int x = C::WARP_KEYS / 2; x; x >>= 1) l[r] += __shfl_xor_sync(0xffffffffu, l[r], x);
#pragma unroll
            for (int x = CL; x < 32; x <<= 1) {
                o[r].x += __shfl_xor_sync(0xffffffffu, o[r].x, x);
                o[r].y += __shfl_xor_sync(0xffffffffu, o[r].y, x);
                o[r].z += __shfl_xor_sync(0xffffffffu, o[r].z, x);
                o[r].w += __shfl_xor_sync(0xffffffffu, o[r].w, x);
            }
        }
    }
};

// Values behind the end of the keys may be anything, NaN too, which a probability of zero does not stop: zeros take the place of rows
// [from, to) of a tile's values.  A warp clears what it will read; warps that share keys write the same zeros.
template <typename C> __device__ __forceinline__ void clear_values(uint8_t* tile, int from, int to) {
    constexpr int CH = C::ROW / 16;
    for (int i = from * CH + (threadIdx.x & 31); i < to * CH; i += 32)
        *reinterpret_cast<uint4*>(tile + chunk_at<C>(i / CH, i % CH)) = make_uint4(0, 0, 0, 0);
    __syncwarp();
}

// ------------------------------------------------------------------------------------------------------
// The warp that loads
// ------------------------------------------------------------------------------------------------------
// Lanes 0-15 load keys, 16-31 values, a lane one box (of up to 16) of each tile; the pages of the next tile are looked up while
// this one waits for its stage.
template <typename T, typename C> struct Loader {
    uint8_t *sK, *sV;
    uint64_t *full, *empty;
    uint32_t* there;
    volatile int* abort_flag;
    int it = 0;                                            // tiles so far
    bool ok = true;

    __device__ __forceinline__ void lookup(const MmaParams& p, int seq, int k0, int end, int& page, int& slot) {
        const int key = k0 + (threadIdx.x & 15) * p.box;
        page = -1;
        slot = 0;
        if (key < end && key < k0 + C::KEYS) {
            const int col = p.page.div(key);
            slot = key - col * p.page.d;
            page = p.a.pages[seq * p.a.pages_ld + col];
            if (page < 0 || page >= p.a.num_pages) page = p.a.num_pages;       // behind the cache: TMA fills the box with zeros
        }
    }
    __device__ __forceinline__ void tiles(const MmaParams& p, const CUtensorMap* tmK, const CUtensorMap* tmV, int seq, int head, int begin,
                                          int end) {
        const int lane = threadIdx.x & 31;
        const CUtensorMap* map = lane < 16 ? tmK : tmV;
        const uint32_t base = smem_u32(lane < 16 ? sK : sV) + (lane & 15) * p.box * C::SLAB;
        int page, slot, next_page, next_slot;
        lookup(p, seq, begin, end, page, slot);
        for (int k0 = begin; k0 < end && ok; k0 += C::KEYS, ++it) {
            const int s = it % C::STAGES;
            lookup(p, seq, k0 + C::KEYS, end, next_page, next_slot);
            if (it >= C::STAGES) ok = mbar_wait(&empty[s], (it / C::STAGES - 1) & 1, abort_flag);
            ok = __all_sync(0xffffffffu, ok);
            if (!ok) break;
            const uint32_t mask = __ballot_sync(0xffffffffu, page != p.a.num_pages);
            if (lane == 0) {
                there[s] = mask;
                mbar_arrive_expect_tx(&full[s], (uint32_t)(cme_cdiv_dev(min(C::KEYS, end - k0), p.box) * p.box * C::ROW * 2));
            }
            __syncwarp();
            if (page >= 0) {
#pragma unroll
                for (int c = 0; c < C::SLABS; ++c)
                    tma_load_4d(base + s * C::TILE + c * C::KEYS * 128, map, &full[s], c * (128 / (int)sizeof(T)), slot, head, page);
            }
            page = next_page;
            slot = next_slot;
        }
    }
    __device__ __forceinline__ void drain() {              // after a wait ran out: copies in flight end before the CTA does
        if (!ok && (threadIdx.x & 31) == 0) for (int i = 0; i < 2000; ++i) __nanosleep(500);
    }
};

// Index of (token, head) of row r of a tile.
__device__ __forceinline__ long long row_at(const MmaParams& p, const PagedTile& t, int head, int r) {
    const int rr = t.first + r, tok = rr / p.group;
    return (long long)(t.token0 + tok) * p.a.heads + head * p.group + rr - tok * p.group;
}
template <typename T> __device__ __forceinline__ const T* row_of_q(const MmaParams& p, const PagedTile& t, int head, int r) {
    if (r >= t.rows) return nullptr;
    const int rr = t.first + r, tok = rr / p.group;
    return static_cast<const T*>(p.a.q) + (t.token0 + tok) * p.a.q_token + (head * p.group + rr - tok * p.group) * p.a.q_head;
}
// Keys that row r of a tile sees, if there are so many.
__device__ __forceinline__ int row_sees(const MmaParams& p, const PagedTile& t, int r) {
    return t.length - t.n + (t.first + r) / p.group + 1;
}
// Keys that a row of the tile sees: those of its last row.
__device__ __forceinline__ int tile_sees(const MmaParams& p, const PagedTile& t) {
    return max(0, min(p.a.max_len, row_sees(p, t, t.rows - 1)));
}

// ------------------------------------------------------------------------------------------------------
// Many rows: 16 a warp
// ------------------------------------------------------------------------------------------------------
// What bounds it in fp32: three tf32 products an element at 8 clocks an instruction and scheduler (92 TFLOP/s of the product asked for), and beside
// them 4 instructions to split each element of K and V, which every warp does for itself.  16 heads of 64, 512 tokens over 2048 in 4
// sequences: 351 us, 43 TFLOP/s.  (Two tiles of 16 rows a warp, which split half as often, when it took 378: 344 us there, but 13.0 for 11.4 with
// 64 tokens over 128 and 36 for 28 with head size 32.)
template <typename T, int D>
__global__ void __launch_bounds__(Cfg<T, D, true>::WARPS * 32 + 32, Cfg<T, D, true>::CTAS)
paged_attn_rows_kernel(const __grid_constant__ CUtensorMap tmK, const __grid_constant__ CUtensorMap tmV, const MmaParams p) {
    using C = Cfg<T, D, true>;
    constexpr int NT = D / 8;
    extern __shared__ __align__(1024) uint8_t smem[];
    Loader<T, C> ld;
    ld.sK = smem;
    ld.sV = ld.sK + C::STAGES * C::TILE;
    uint8_t* sQ = ld.sV + C::STAGES * C::TILE;             // fp32: [warp] the rows' fragments
    ld.full = reinterpret_cast<uint64_t*>(sQ + 4 * C::FRAGS);
    ld.empty = ld.full + C::STAGES;
    ld.there = reinterpret_cast<uint32_t*>(ld.empty + C::STAGES);      // [stage] which of its boxes' pages are in the cache
    ld.abort_flag = reinterpret_cast<volatile int*>(ld.there + 7);

    const int warp = __shfl_sync(0xffffffffu, threadIdx.x >> 5, 0), lane = threadIdx.x & 31;
    const CmePaged& a = p.a;
    if (threadIdx.x == 0) {
        *ld.abort_flag = 0;
        for (int s = 0; s < C::STAGES; ++s) { mbar_init(&ld.full[s], 1); mbar_init(&ld.empty[s], C::WARPS); }
        fence_barrier_init();
        prefetch_tmap(&tmK);
        prefetch_tmap(&tmV);
    }
    pdl_release();
    pdl_wait();
    // Where not all CTAs run at once, tiles that see the most keys first (above 32 sequences: late tiles), of all heads: fp32, 16 sequences of
    // up to 400 tokens over 1500, 12 heads of 64 240 / 206 us.
    const int at = p.heads.div(blockIdx.x), head = blockIdx.x - at * a.kv_heads, tile = p.parts.div(at), split = at - tile * p.splits;
    const PagedTile t = p.by_keys ? paged_find_tile_by_keys(a, tile, p.group, 64, C::KEYS) : paged_find_tile(a, p.tiles - 1 - tile, p.group, 64);
    __syncthreads();
    if (t.rows == 0) return;
    // keys [0, limit) are seen by the last row; this CTA takes [begin, end)
    const int limit = tile_sees(p, t);
    const int begin = (int)min((long long)limit, (long long)split * p.split_keys);
    const int end = (int)min((long long)limit, (long long)begin + p.split_keys);
    if (warp == C::WARPS) {
        ld.tiles(p, &tmK, &tmV, t.seq, head, begin, end);
        ld.drain();
    } else {
        const int of = warp & 3, group = warp >> 2;                    // its 16 rows, and which of the keys it takes
        const int row0 = of * 16 + (lane >> 2), tq = lane & 3;         // this thread's rows: row0, row0 + 8
        Rows<T, C, D, 1> q;
        q.load(row_of_q<T>(p, t, head, row0), row_of_q<T>(p, t, head, row0 + 8), 0);
        q.publish(sQ + of * C::FRAGS, 0);                              // (both groups write the same)
        const int see0 = min(end, row_sees(p, t, row0)), see1 = min(end, row_sees(p, t, row0 + 8));
        const int see_first = min(end, row_sees(p, t, of * 16));
        const int last = min(t.rows, of * 16 + 16) - 1;
        const int seen = last < of * 16 ? 0 : min(end, row_sees(p, t, last));      // no row of the warp sees keys from here on
        WarpState<C, D> w;
        w.clear();
        int it = 0;
        for (int k0 = begin; k0 < end; k0 += C::KEYS, ++it) {
            const int s = it % C::STAGES;
            if (!mbar_wait(&ld.full[s], (it / C::STAGES) & 1, ld.abort_flag)) break;
            const uint32_t there = ld.there[s];
            if (k0 < seen && k0 + C::KEYS > end) clear_values<C>(ld.sV + s * C::TILE, end - k0, C::KEYS);
#pragma unroll 1
            for (int key0 = group * C::WARP_KEYS; key0 < C::KEYS && k0 + key0 < seen; key0 += C::GROUPS * C::WARP_KEYS)
                attend(w, q, smem_u32(ld.sK) + s * C::TILE, smem_u32(ld.sV) + s * C::TILE, key0, k0, see0, see1,
                       there != 0xffffffffu || k0 + key0 + C::WARP_KEYS > see_first, there, p.box_log, p.scale_log2);
            __syncwarp();
            if (lane == 0) mbar_arrive(&ld.empty[s]);
        }
        w.finish();
        if constexpr (C::GROUPS > 1) {
            // the second group's part of the rows through the tiles' memory, which nobody reads any more
            static_assert((NT * 4 + 4) * 512 <= 2 * C::STAGES * C::TILE, "memory of the tiles");
            float* x = reinterpret_cast<float*>(smem) + (threadIdx.x & 127);
            named_bar_sync(1, C::WARPS * 32);
            if (group) {
#pragma unroll
                for (int r = 0; r < 2; ++r) { x[r * 256] = w.m[r]; x[r * 256 + 128] = w.l[r]; }
#pragma unroll
                for (int i = 0; i < NT * 4; ++i) x[(4 + i) * 128] = w.o[i >> 2][i & 3];
            }
            named_bar_sync(1, C::WARPS * 32);
            if (!group) {
#pragma unroll
                for (int r = 0; r < 2; ++r) {
                    const float m = x[r * 256], mm = fmaxf(w.m[r], m), f0 = part_factor(w.m[r], mm), f1 = part_factor(m, mm);
                    w.m[r] = mm;
                    w.l[r] = fmaf(f1, x[r * 256 + 128], f0 * w.l[r]);
#pragma unroll
                    for (int d = 0; d < NT; ++d)
#pragma unroll
                        for (int i = 2 * r; i < 2 * r + 2; ++i) w.o[d][i] = fmaf(f1, x[(4 + d * 4 + i) * 128], f0 * w.o[d][i]);
                }
            }
        }
        T* out = static_cast<T*>(a.o);
#pragma unroll
        for (int r = 0; r < 2; ++r) {
            const int row = row0 + 8 * r;
            if (group || row >= t.rows) continue;
            long long at = row_at(p, t, head, row);
            if (p.splits == 1) {
                const float inv = inverse(w.l[r]);
#pragma unroll
                for (int d = 0; d < NT; ++d) {
                    T* dst = out + at * D + d * 8 + tq * 2;
                    if constexpr (C::F32) *reinterpret_cast<float2*>(dst) = make_float2(w.o[d][2 * r] * inv, w.o[d][2 * r + 1] * inv);
                    else *reinterpret_cast<uint32_t*>(dst) = f2_to_bf2(w.o[d][2 * r] * inv, w.o[d][2 * r + 1] * inv);
                }
                if (tq == 0) a.lse[at] = log_sum(w.m[r], w.l[r]);
            } else {
                at = at * p.splits + split;
                if (begin < end) {
#pragma unroll
                    for (int d = 0; d < NT; ++d)
                        *reinterpret_cast<float2*>(p.part_o + at * D + d * 8 + tq * 2) = make_float2(w.o[d][2 * r], w.o[d][2 * r + 1]);
                }
                if (tq == 0) p.part_ml[at] = make_float2(w.m[r], w.l[r]);
            }
        }
    }
    if (threadIdx.x == 0 && *ld.abort_flag && p.status) atomicExch(p.status, CME_ERR_TIMEOUT);
}

// ------------------------------------------------------------------------------------------------------
// Up to 16 rows: each warp takes a quarter of every key tile
// ------------------------------------------------------------------------------------------------------
// What bounds it: the bytes of the cache, so the loads must never stop.  An item is a tile of rows and a key head.
//   stream   as many CTAs as fit the GPU; all items' key tiles in a row are divided among them evenly, whatever the sequences'
//            lengths.  A CTA's loads run on into its next item while the last one's warps are joined.  An item that lies in one CTA is
//            finished there, the others' parts are left in scratch (at most two a CTA) and joined by a small kernel.
//   cluster  a CTA has one part of one item, and up to eight CTAs join theirs through shared memory: one launch, for few items.
// Single tokens, bf16, calls one after the other: one sequence of 701, 12 heads of 64 5.6 us (a launch, three dependent lookups, a tile, the join;
// 5.0 as a graph); 64 of up to 1024, 16 heads of 64 31.8 us, 4.2 TB/s of 135 MB; 16 of 2000 to 32768, 32 heads of 128 on 8 166 us, 6.1 TB/s.  fp32: 32
// of up to 2048, 4 heads of 128 34.3 us, 3.9 TB/s.
constexpr int REC_INTS = 8;                // of an item that ends in a CTA other than it began in: first CTA or -1, rows, token0, first, head

// Walks over the key tiles of all items, in the order sequence, tile of rows, key head, key tile.  What an item costs besides its tiles
// (its rows, the join of the warps) counts as ITEM_COST more tiles before them, so that CTAs with many short items get fewer tiles.
constexpr int ITEM_COST = 2;
struct Walk {
    int seq, tiles, keys;                  // of the current sequence: tiles of rows, key tiles (one at least) and ITEM_COST
    int tile, head, key;                   // where it stands
    int left = 0;                          // key tiles that are still to be taken (the host has checked that all fit 31 bits)
    PagedTile t;

    template <typename C> __device__ __forceinline__ void load_seq(const MmaParams& p, int b) {
        const CmePaged& a = p.a;
        int lo = a.offsets[b], hi = a.offsets[b + 1];
        lo = max(0, min(lo, a.rows));
        hi = max(lo, min(hi, a.rows));
        t.seq = seq = b;
        t.token0 = lo;
        t.n = hi - lo;
        t.length = paged_length(a, a.lengths[b], t.n);
        t.first = t.rows = 0;
        tiles = (int)(((long long)t.n * p.group + 15) / 16);
        keys = max(1, cme_cdiv_dev(min(t.length, a.max_len), C::KEYS)) + ITEM_COST;
    }
    // Takes share `part` of `parts` of the whole; returns how many key tiles a share has.  Whole warps.
    template <typename C> __device__ __forceinline__ int start(const MmaParams& p, int part, int parts) {
        const int lane = threadIdx.x & 31, each = (p.a.seqs + 31) / 32;
        long long own = 0;
        for (int i = 0; i < each; ++i) {                   // a lane's sequences
            const int b = lane * each + i;
            if (b < p.a.seqs) { load_seq<C>(p, b); own += (long long)tiles * p.a.kv_heads * keys; }
        }
        // Sequences that share rows, which no offsets in order make, can have more than 31 bits of tiles: none is taken then.
        if (__any_sync(0xffffffffu, own > INT_MAX / 32)) {
            const unsigned high = __reduce_add_sync(0xffffffffu, (unsigned)min(own >> 16, 1ll << 16)), low = __reduce_add_sync(0xffffffffu, (unsigned)own & 0xffffu);
            if (((unsigned long long)high << 16) + low > INT_MAX) return 1;
        }
        const int sum = (int)own;
        int upto = sum;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const int v = __shfl_up_sync(0xffffffffu, upto, o);
            if (lane >= o) upto += v;
        }
        // (share * part passes 31 bits only where nothing is left)
        const int all = __shfl_sync(0xffffffffu, upto, 31), share = (int)(((unsigned)all + parts - 1) / parts);
        const int first = (int)min((long long)all, (long long)share * part);
        left = min(share, all - first);
        if (left <= 0) return share;
        const int who = __ffs(__ballot_sync(0xffffffffu, first < upto)) - 1;
        int skip = first - __shfl_sync(0xffffffffu, upto - sum, who);
        int b = who * each;
        for (;; ++b) {
            load_seq<C>(p, b);
            const int own = tiles * p.a.kv_heads * keys;
            if (skip < own) break;
            skip -= own;
        }
        const int item = skip / keys;
        key = skip - item * keys;
        tile = item / p.a.kv_heads;
        head = item - tile * p.a.kv_heads;
        return share;
    }
    // The next part of an item that is this CTA's, if there is one.
    struct Part {
        PagedTile t;
        int head, begin, end;              // keys
        bool first, last;                  // whether the item's first (last) key tile is in it
    };
    template <typename C> __device__ __forceinline__ bool next(const MmaParams& p, Part& part) {
        while (left > 0) {
            const int n = min(left, keys - key), k0 = max(0, key - ITEM_COST), k1 = key + n - ITEM_COST;
            if (k1 > 0) {
                t.first = tile * 16;
                t.rows = (int)min(16ll, (long long)t.n * p.group - t.first);
                const int limit = tile_sees(p, t);
                part.t = t;
                part.head = head;
                part.begin = (int)min((long long)limit, (long long)k0 * C::KEYS);
                part.end = (int)min((long long)limit, (long long)k1 * C::KEYS);
                part.first = k0 == 0;
                part.last = key + n == keys;
            }
            step<C>(p, n);
            if (k1 > 0) return true;
        }
        return false;
    }
    template <typename C> __device__ __forceinline__ void step(const MmaParams& p, int n) {
        left -= n;
        key += n;
        if (key < keys || left == 0) return;
        key = 0;
        if (++head < p.a.kv_heads) return;
        head = 0;
        if (++tile < tiles) return;
        tile = 0;
        do load_seq<C>(p, seq + 1); while (tiles == 0);    // (something is left, so there is such a sequence)
    }
};

template <typename T, int D, bool CLUSTER>
__global__ void __launch_bounds__(Cfg<T, D, false>::WARPS * 32 + 32, Cfg<T, D, false>::CTAS)
paged_attn_single_kernel(const __grid_constant__ CUtensorMap tmK, const __grid_constant__ CUtensorMap tmV, const MmaParams p) {
    using C = Cfg<T, D, false>;
    constexpr int NT = D / 8;
    extern __shared__ __align__(1024) uint8_t smem[];
    Loader<T, C> ld;
    ld.sK = smem;
    ld.sV = ld.sK + C::STAGES * C::TILE;
    constexpr int JR = C::JOIN_ROWS, COMPUTE = C::WARPS * 32;
    float* sums = reinterpret_cast<float*>(ld.sV + C::STAGES * C::TILE);       // [warps][JR rows][D]
    uint8_t* sQ = reinterpret_cast<uint8_t*>(sums + 32 * D);                // fp32: the rows' fragments
    ld.full = reinterpret_cast<uint64_t*>(sQ + C::FRAGS);
    ld.empty = ld.full + C::STAGES;
    ld.there = reinterpret_cast<uint32_t*>(ld.empty + C::STAGES);
    ld.abort_flag = reinterpret_cast<volatile int*>(ld.there + 7);
    float2* sML = reinterpret_cast<float2*>(ld.there + 8);                     // [warps][JR rows] m and l

    const int warp = __shfl_sync(0xffffffffu, threadIdx.x >> 5, 0), lane = threadIdx.x & 31;
    const CmePaged& a = p.a;
    if (threadIdx.x == 0) {
        *ld.abort_flag = 0;
        for (int s = 0; s < C::STAGES; ++s) { mbar_init(&ld.full[s], 1); mbar_init(&ld.empty[s], C::WARPS); }
        fence_barrier_init();
        prefetch_tmap(&tmK);
        prefetch_tmap(&tmV);
    }
    pdl_release();
    pdl_wait();
    Walk wk{};
    typename Walk::Part part;
    int share = 0;
    bool some = true;
    if constexpr (CLUSTER) {
        part.t = paged_find_tile(a, blockIdx.x / p.splits, p.group, 16);
        part.head = blockIdx.y;
        const int limit = tile_sees(p, part.t);
        const int span = cme_cdiv_dev(cme_cdiv_dev(limit, C::KEYS), p.splits) * C::KEYS;
        part.begin = (int)min((long long)limit, (long long)(blockIdx.x % p.splits) * span);
        part.end = (int)min((long long)limit, (long long)part.begin + span);
        part.first = part.last = true;
    } else {
        share = wk.start<C>(p, blockIdx.x, gridDim.x);
        if (threadIdx.x == 0) {            // does the first item begin in another CTA, and end here?
            int* rec = p.records + blockIdx.x * REC_INTS;
            rec[0] = -1;
            if (wk.left > 0 && wk.key > ITEM_COST && wk.key + wk.left >= wk.keys) {
                rec[0] = (int)(((long long)blockIdx.x * share - wk.key + ITEM_COST) / share);      // the CTA of the item's first key tile
                rec[1] = (int)min(16ll, (long long)wk.t.n * p.group - wk.tile * 16);
                rec[2] = wk.t.token0;
                rec[3] = wk.tile * 16;
                rec[4] = wk.head;
            }
        }
        some = wk.next<C>(p, part);
    }
    __syncthreads();
    if (CLUSTER && part.t.rows == 0) return;               // all CTAs of a cluster

    if (warp == C::WARPS) {
        while (some) {
            ld.tiles(p, &tmK, &tmV, part.t.seq, part.head, part.begin, part.end);
            some = !CLUSTER && wk.next<C>(p, part);
        }
        ld.drain();
    } else {
        const int g = lane >> 2, tq = lane & 3;
        T* out = static_cast<T*>(a.o);
        int it = 0;
        bool ok = true;
        Rows<T, C, D, C::WARPS> coming;
        if (some) coming.load(row_of_q<T>(p, part.t, part.head, g), row_of_q<T>(p, part.t, part.head, g + 8), warp);
        while (some) {
            const PagedTile t = part.t;
            const int head = part.head, begin = part.begin, end = part.end;
            const bool first = part.first, last = part.last;
            Rows<T, C, D, C::WARPS> q = coming;
            const int key0 = (warp & 3) * C::WARP_KEYS, see_first = min(end, row_sees(p, t, 0));
            some = !CLUSTER && wk.next<C>(p, part);
            // f(stage, first key, which boxes' pages are there, whether some key of the warp's is not visible to a row) for its tiles
            auto tiles = [&](auto&& f) {
                for (int k0 = begin; k0 < end && ok; k0 += C::KEYS, ++it) {
                    const int s = it % C::STAGES;
                    const bool own = C::GROUPS == 1 || it % C::GROUPS == warp >> 2;
                    // (all warps wait for every tile and hand it back: who skips a phase of a barrier cannot tell the next from the last)
                    ok = mbar_wait(&ld.full[s], (it / C::STAGES) & 1, ld.abort_flag);
                    if (!ok) break;
                    const uint32_t there = ld.there[s];
                    if (own && k0 + key0 + C::WARP_KEYS > end) clear_values<C>(ld.sV + s * C::TILE, max(key0, end - k0), key0 + C::WARP_KEYS);
                    if (own && k0 + key0 < end) f(s, k0, there, there != 0xffffffffu || k0 + key0 + C::WARP_KEYS > see_first);
                    if (k0 + C::KEYS > end) fence_proxy_async();       // the cleared values' place will be loaded again
                    __syncwarp();
                    if (lane == 0) mbar_arrive(&ld.empty[s]);
                    // the next item's rows are on their way under this one's tiles
                    if (k0 == begin && some) coming.load(row_of_q<T>(p, part.t, part.head, g), row_of_q<T>(p, part.t, part.head, g + 8), warp);
                }
                if (begin >= end && some) coming.load(row_of_q<T>(p, part.t, part.head, g), row_of_q<T>(p, part.t, part.head, g + 8), warp);
            };
            WarpState<C, D> w;
            bool simt = false;
            auto on_cuda_cores = [&](auto rows) {
                constexpr int R = decltype(rows)::value;
                simt = true;
                q.publish_rows(reinterpret_cast<float*>(sQ), warp, R);
                int see[R];
#pragma unroll
                for (int r = 0; r < R; ++r) see[r] = min(end, row_sees(p, t, r));
                SimtState<C, D, R> x;
                x.clear();
                tiles([&](int s, int k0, uint32_t there, bool masked) {
                    x.attend(reinterpret_cast<const float*>(sQ), smem_u32(ld.sK) + s * C::TILE, smem_u32(ld.sV) + s * C::TILE, key0, k0, see,
                             masked, there, p.box_log, p.scale_log2);
                });
                x.finish();
#pragma unroll
                for (int r = 0; r < R; ++r) {
                    if (lane < D / 4) *reinterpret_cast<float4*>(sums + (warp * JR + r) * D + lane * 4) = x.o[r];
                    if (lane == 0) sML[warp * JR + r] = make_float2(x.m[r], x.l[r]);
                }
            };
            if constexpr (C::F32) {
                if (t.rows == 1) on_cuda_cores(std::integral_constant<int, 1>{});
                else if (t.rows == 2) on_cuda_cores(std::integral_constant<int, 2>{});
                else if (t.rows <= 4) on_cuda_cores(std::integral_constant<int, 4>{});
            }
            if (!simt) {
                q.publish(sQ, warp);
                const int see0 = min(end, row_sees(p, t, g)), see1 = min(end, row_sees(p, t, g + 8));
                w.clear();
                tiles([&](int s, int k0, uint32_t there, bool masked) {
                    attend(w, q, smem_u32(ld.sK) + s * C::TILE, smem_u32(ld.sV) + s * C::TILE, key0, k0, see0, see1, masked, there, p.box_log,
                           p.scale_log2);
                });
                w.finish();
            }
            // join the warps, some rows at a time
            float* own = reinterpret_cast<float*>(smem);   // cluster: [16 rows][D], this CTA's sums (its key tiles are done with)
            float2* own_ml = reinterpret_cast<float2*>(own + 16 * D);
#pragma unroll
            for (int r0 = 0; r0 < 16; r0 += JR) {
                if (r0 >= t.rows) break;
                const int r = r0 / 8, own_row = g - r0 % 8;             // this lane has row r0 + own_row, if it is one of them
                if (!simt && own_row >= 0 && own_row < JR && r0 + own_row < t.rows) {
#pragma unroll
                    for (int d = 0; d < NT; ++d)
                        *reinterpret_cast<float2*>(sums + (warp * JR + own_row) * D + d * 8 + tq * 2) = make_float2(w.o[d][2 * r], w.o[d][2 * r + 1]);
                    if (tq == 0) sML[warp * JR + own_row] = make_float2(w.m[r], w.l[r]);
                }
                named_bar_sync(1, COMPUTE);
                for (int i = threadIdx.x; i < min(JR, t.rows - r0) * (D / 4); i += COMPUTE) {
                    const int row = i / (D / 4), c = i % (D / 4) * 4;
                    float mm = -INFINITY, ll = 0.f;
#pragma unroll
                    for (int k = 0; k < C::WARPS; ++k) mm = fmaxf(mm, sML[k * JR + row].x);
                    float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
                    for (int k = 0; k < C::WARPS; ++k) {
                        const float2 ml = sML[k * JR + row];
                        const float f = part_factor(ml.x, mm);
                        ll = fmaf(f, ml.y, ll);
                        add4(v, f, *reinterpret_cast<const float4*>(sums + (k * JR + row) * D + c));
                    }
                    if (CLUSTER ? p.splits > 1 : !(first && last)) {
                        if constexpr (CLUSTER) {
                            *reinterpret_cast<float4*>(own + (r0 + row) * D + c) = v;
                            if (c == 0) own_ml[r0 + row] = make_float2(mm, ll);
                        } else {                           // slot 0: an item that ends here, 1: one that goes on in the next CTA
                            const long long at = (blockIdx.x * 2ll + !last) * 16 + r0 + row;
                            *reinterpret_cast<float4*>(p.part_o + at * D + c) = v;
                            if (c == 0) p.part_ml[at] = make_float2(mm, ll);
                        }
                    } else {
                        const long long at = row_at(p, t, head, r0 + row);
                        store4(out + at * D + c, v, inverse(ll));
                        if (c == 0) a.lse[at] = log_sum(mm, ll);
                    }
                }
                named_bar_sync(1, COMPUTE);
            }
        }
    }
    if constexpr (CLUSTER) {
        if (p.splits > 1) {
            // the parts of the cluster's CTAs, each CTA joins its share of the elements
            cg::cluster_group cl = cg::this_cluster();
            const PagedTile& t = part.t;
            float* own = reinterpret_cast<float*>(smem);
            float2* own_ml = reinterpret_cast<float2*>(own + 16 * D);
            cl.sync();
            for (int i = (blockIdx.x % p.splits) * (int)blockDim.x + threadIdx.x; i < t.rows * (D / 4); i += p.splits * (int)blockDim.x) {
                const int row = i / (D / 4), c = i % (D / 4) * 4;
                float mm = -INFINITY, ll = 0.f;
                float2 ml[8];
                float4 x[8];
#pragma unroll
                for (int k = 0; k < 8; ++k) {
                    ml[k] = make_float2(-INFINITY, 0.f);
                    if (k < p.splits) {
                        ml[k] = *reinterpret_cast<const float2*>(cl.map_shared_rank(own_ml + row, k));
                        x[k] = *reinterpret_cast<const float4*>(cl.map_shared_rank(own + row * D + c, k));
                    }
                    mm = fmaxf(mm, ml[k].x);
                }
                float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
                for (int k = 0; k < 8; ++k) {
                    if (k >= p.splits) break;
                    const float f = part_factor(ml[k].x, mm);
                    ll = fmaf(f, ml[k].y, ll);
                    add4(v, f, x[k]);
                }
                const long long at = row_at(p, t, part.head, row);
                store4(static_cast<T*>(a.o) + at * D + c, v, inverse(ll));
                if (c == 0) a.lse[at] = log_sum(mm, ll);
            }
            cl.sync();                                     // nobody's shared memory goes while it is read
        }
    }
    if (threadIdx.x == 0 && *ld.abort_flag && p.status) atomicExch(p.status, CME_ERR_TIMEOUT);
}

// Joins the parts of the items that several CTAs of the stream had: block (c, y) those of the item that ends in CTA c, rows 4 y to 4 y + 3, or,
// of items in many parts, rows y, y + 4, ...
template <typename T, int D>
__global__ void __launch_bounds__(128) paged_stream_join_kernel(const MmaParams p) {
    constexpr int COLS = D / 4, GROUPS = 128 / COLS;       // threads of a row, and how many of its parts are added at a time
    __shared__ float scratch[32];
    __shared__ float4 sum[GROUPS][COLS];
    __shared__ float sum_l[GROUPS];
    pdl_release();
    pdl_wait();
    const int* rec = p.records + blockIdx.x * REC_INTS;
    const int c0 = rec[0], c1 = blockIdx.x;
    if (c0 < 0) return;
    PagedTile t{};
    t.rows = rec[1];
    t.token0 = rec[2];
    t.first = rec[3];
    const int head = rec[4], group = threadIdx.x / COLS, c = threadIdx.x % COLS * 4;
    auto slot_of = [&](int k, int row) { return (k * 2ll + (k != c1)) * 16 + row; };
    constexpr int FEW = 8;
    if (c1 - c0 < FEW) {
        // A warp a row, all loads at once (64 sequences of up to 1024, 16 heads of 64: 31.3 us, in the way of many parts 32.2)
        const int row = blockIdx.y * 4 + (threadIdx.x >> 5), lane = threadIdx.x & 31;
        if (row >= t.rows) return;
        float2 ml[FEW];
        float4 x[FEW];
#pragma unroll
        for (int k = 0; k < FEW; ++k) {
            ml[k] = make_float2(-INFINITY, 0.f);
            x[k] = make_float4(0.f, 0.f, 0.f, 0.f);
            if (c0 + k <= c1) {
                ml[k] = p.part_ml[slot_of(c0 + k, row)];
                if (lane < COLS) x[k] = *reinterpret_cast<const float4*>(p.part_o + slot_of(c0 + k, row) * D + lane * 4);
            }
        }
        float mm = -INFINITY, l = 0.f;
        float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
        for (int k = 0; k < FEW; ++k) mm = fmaxf(mm, ml[k].x);
#pragma unroll
        for (int k = 0; k < FEW; ++k) {
            const float f = part_factor(ml[k].x, mm);
            l = fmaf(f, ml[k].y, l);
            add4(v, f, x[k]);
        }
        const long long at = row_at(p, t, head, row);
        if (lane < COLS) store4(static_cast<T*>(p.a.o) + at * D + lane * 4, v, inverse(l));
        if (lane == 0) p.a.lse[at] = log_sum(mm, l);
        return;
    }
    for (int row = blockIdx.y; row < t.rows; row += 4) {
        auto slot = [&](int k) { return slot_of(k, row); };
        float mm = -INFINITY;
        for (int k = c0 + threadIdx.x; k <= c1; k += 128) mm = fmaxf(mm, p.part_ml[slot(k)].x);
        mm = block_max(mm, scratch);
        float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
        float l = 0.f;
#pragma unroll 4
        for (int k = c0 + group; k <= c1; k += GROUPS) {
            const float2 ml = p.part_ml[slot(k)];
            const float f = part_factor(ml.x, mm);
            l = fmaf(f, ml.y, l);
            add4(v, f, *reinterpret_cast<const float4*>(p.part_o + slot(k) * D + c));
        }
        sum[group][c / 4] = v;
        if (c == 0) sum_l[group] = l;
        __syncthreads();
        if (group == 0) {
            l = 0.f;
            v = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
            for (int k = 0; k < GROUPS; ++k) { l += sum_l[k]; add4(v, 1.f, sum[k][c / 4]); }
            const long long at = row_at(p, t, head, row);
            store4(static_cast<T*>(p.a.o) + at * D + c, v, inverse(l));
            if (c == 0) p.a.lse[at] = log_sum(mm, l);
        }
        __syncthreads();
    }
}

// Joins the parts of a row that CTAs left in scratch: one warp per row.  A part that summed nothing has left no sums either.
template <typename T, int D>
__global__ void __launch_bounds__(128) paged_join_kernel(const float* __restrict__ part_o, const float2* __restrict__ part_ml, T* out,
                                                         float* lse, long long rows, int splits) {
    constexpr int VEC = D / 32;
    pdl_release();
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
    return 2 * C::STAGES * C::TILE + (ROWS ? 4 : 1) * C::FRAGS + C::STAGES * 16 + 32 + (ROWS ? 0 : 32 * D * 4 + 32 * 8);
}

template <typename T, int D, bool ROWS, auto Kernel>
int launch(dim3 grid, const CmePaged* a, int cluster, const MmaParams& p, cudaStream_t st) {
    using C = Cfg<T, D, ROWS>;
    constexpr int SMEM = smem_bytes<T, D, ROWS>();
    static_assert(SMEM <= 227 * 1024 && C::CTAS * (SMEM + 1024) <= 228 * 1024, "shared memory of a CTA");
    static bool attr[CME_MAX_DEVICES] = {};               // function attributes are per device
    int dev = 0;
    CME_CUDA(cudaGetDevice(&dev));
    if (!attr[dev % CME_MAX_DEVICES]) {
        CME_CUDA(cudaFuncSetAttribute(Kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, SMEM));
        attr[dev % CME_MAX_DEVICES] = true;
    }
    CUtensorMap mk, mv;
    const auto swizzle = C::SLAB == 64 ? CU_TENSOR_MAP_SWIZZLE_64B : CU_TENSOR_MAP_SWIZZLE_128B;
    int rc;
    if ((rc = paged_make_map(&mk, a, a->k, a->k_page_stride, a->k_head_stride, a->k_slot_stride, C::SLAB / (int)sizeof(T), p.box, swizzle))) return rc;
    if ((rc = paged_make_map(&mv, a, a->v, a->v_page_stride, a->v_head_stride, a->v_slot_stride, C::SLAB / (int)sizeof(T), p.box, swizzle))) return rc;
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = grid;
    cfg.blockDim = dim3(C::WARPS * 32 + 32);
    cfg.dynamicSmemBytes = SMEM;
    cfg.stream = st;
    cudaLaunchAttribute at[2];
    at[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    at[0].val.programmaticStreamSerializationAllowed = 1;
    at[1].id = cudaLaunchAttributeClusterDimension;
    at[1].val.clusterDim.x = cluster;
    at[1].val.clusterDim.y = at[1].val.clusterDim.z = 1;
    cfg.attrs = at;
    cfg.numAttrs = cluster > 1 ? 2 : 1;
    CME_CUDA(cudaLaunchKernelEx(&cfg, Kernel, mk, mv, p));
    CME_LAUNCH_CHECK();
    return CME_OK;
}

template <typename T, int D> int launch_any(const CmePaged* a, const PagedPlan& plan, MmaParams& p, cudaStream_t st) {
    if (plan.kernel == PAGED_ROWS) {
        int sms;
        if (const int rc = cme_num_sms(&sms)) return rc;
        const unsigned ctas = (unsigned)(plan.tiles * plan.splits) * a->kv_heads;
        p.by_keys = paged_by_keys(a, p.group) && ctas > (unsigned)sms * Cfg<T, D, true>::CTAS;
        p.heads = paged_div(a->kv_heads);
        p.parts = paged_div(plan.splits);
        return launch<T, D, true, paged_attn_rows_kernel<T, D>>(dim3(ctas), a, 1, p, st);
    }
    const dim3 grid((unsigned)(plan.tiles * plan.splits), a->kv_heads);
    if (plan.kernel == PAGED_CLUSTER) return launch<T, D, false, paged_attn_single_kernel<T, D, true>>(grid, a, plan.splits, p, st);
    const int rc = launch<T, D, false, paged_attn_single_kernel<T, D, false>>(dim3(plan.splits), a, 1, p, st);
    if (rc) return rc;
    CME_CUDA(cme_launch_dependent(paged_stream_join_kernel<T, D>, dim3(plan.splits, 4), dim3(128), 0, st, p));
    CME_LAUNCH_CHECK();
    return CME_OK;
}

}  // namespace

int paged_mma_key_tile(int dtype, int head_dim) { return head_dim * (dtype == CME_F32 ? 4 : 2) <= 128 ? 128 : 64; }
int paged_mma_ctas(int dtype, int head_dim) { return dtype == CME_F32 && head_dim == 128 ? 1 : 2; }

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
    p.split_keys = plan.split_keys;
    p.tiles = plan.tiles;
    p.scale_log2 = a->scale * LOG2E;
    // scratch: m and l of the parts (16-byte aligned by their size), their sums; stream: a record for each CTA before them
    const long long parts = plan.kernel == PAGED_STREAM ? plan.splits * 32ll : (long long)a->rows * a->heads * plan.splits;
    p.records = reinterpret_cast<int*>(a->ws);
    float* ml = a->ws + (plan.kernel == PAGED_STREAM ? (long long)plan.splits * REC_INTS : 0);
    p.part_ml = reinterpret_cast<float2*>(ml);
    p.part_o = ml + (parts * 2 + 3) / 4 * 4;
    p.status = cme_attn_status_ptr();
    CME_REQUIRE(p.status != nullptr, CME_ERR_CUDA, "paged attention: device state unavailable");
    if (a->dtype == CME_F32)
        return a->head_dim == 32 ? launch_any<float, 32>(a, plan, p, st) : a->head_dim == 64 ? launch_any<float, 64>(a, plan, p, st)
                                                                                            : launch_any<float, 128>(a, plan, p, st);
    return a->head_dim == 32   ? launch_any<__nv_bfloat16, 32>(a, plan, p, st)
           : a->head_dim == 64 ? launch_any<__nv_bfloat16, 64>(a, plan, p, st)
                               : launch_any<__nv_bfloat16, 128>(a, plan, p, st);
}
