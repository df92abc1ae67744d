// Attention of chunks of new tokens over a paged cache on tcgen05 (bf16): scores, probabilities and sums of
// 128 rows live in tensor memory; a row is a token and one of the query heads that share the key head, token by token.
//
//     S_j = Q K_j^T (TMEM) -> registers -> online softmax -> P_j (bf16 pairs over the columns of S_j) -> O += P_j V_j (TMEM)
//
// P_j is bf16 because V is, the type of both operands of a product; the sum l is of the unrounded probabilities.  Errors against 64 bits are 0.0020 to
// 0.0023 of a result's size, 0.0016 to 0.0017 with probabilities in 32 bits (the result's own rounding).
// 64 keys at a time, loaded by TMA, a box per page (or tile); the swizzle repeats every eight keys, so that boxes of 8, 16 or 32 keys
// make up one tile.  A page that is not there is a box behind the cache, which TMA fills with zeros, and a bit in the row's mask.
// What bounds it: the exponentials (16 a clock and SM: 512 clocks for 128 rows x 64 keys) and, with head size 128, as many clocks of the
// tensor pipe; one hides behind the other only if several tiles of rows are on their way at a time.
//   head size 64   128 rows a CTA, three CTAs an SM (128 columns of tensor memory each): a tile's chain of steps, its start and its end run
//                  under the others'.  Where that many CTAs are not there, two an SM at the most, with two buffers of scores (256 columns): a
//                  tile's steps are shorter, all SMs' together fewer (1 / 8 / 16 chunks of GPT-2 small, us: 16.4 / 20.4 / 31.8, three an SM
//                  17.6 / 24.5 / 31.9; 512 tokens over 4096 in 4 sequences 73.5 / 65.4).
//   head size 32   as 64: the boxes reach over the head's end, where TMA puts zeros, and the sums' second half is left.  What bounds the steps
//                  is the same (1566 tokens over 6081, 12 heads: 74 us, with warp-level products 94).
//   head size 128  256 rows a CTA, one CTA an SM, two buffers of scores for each half: S_{j+1} is made while softmax_j runs.  Both halves
//                  read the same keys: with 128 rows a CTA the tiles of K and V would come out of L2 at 53 bytes a clock and SM.
// 16 chunks of GPT-2 small, 1 to 511 tokens over up to 1024: 25.8 us, 190 TFLOP/s; two of 1500 to 2048 over 8192, 32 heads of 128 on 8: 363 us, 0.96
// PFLOP/s, calls one after the other, where the power limit sets the clocks; after a pause 20 replays of a graph take 326 us each, 1.07 PFLOP/s.
// Every mbarrier wait is bounded; on expiry the CTA flags the status word, frees TMEM and returns.
#include "paged.h"
#include "sm100_ptx.cuh"

#include <algorithm>
#include <mutex>

using namespace sm100;

int* cme_attn_status_ptr();

namespace {

constexpr float LOG2E = 1.4426950408889634f;
constexpr int KEYS = PAGED_TC_KEYS;
// log2 units: the reference maximum is only raised when it would grow by more than 2^8 (settled after 128 keys, whose largest probability
// bf16 then holds exactly)
constexpr float RESCALE_THRESHOLD = 8.f;

template <int D, bool FEW> struct Cfg;
template <> struct Cfg<64, false> {
    static constexpr int HALVES = 1, STAGES = 3, BUFFERS = 1, CTAS = 3, COLS = 128;
};
template <> struct Cfg<64, true> {
    static constexpr int HALVES = 1, STAGES = 3, BUFFERS = 2, CTAS = 2, COLS = 256;
};
template <> struct Cfg<128, false> {
    static constexpr int HALVES = 2, STAGES = 4, BUFFERS = 2, CTAS = 1, COLS = 512;
};
template <int D, bool FEW> struct Sizes : Cfg<D, FEW> {
    using C = Cfg<D, FEW>;
    static constexpr int SLABS = D / 64;                              // 64 columns = 128 bytes each
    static constexpr int Q_SLAB = 128 * 128, KV_SLAB = KEYS * 128;
    static constexpr int Q_BYTES = SLABS * Q_SLAB, KV_BYTES = SLABS * KV_SLAB;
    static constexpr int LOADER = 5 * C::HALVES;                      // four warps of softmax and one that issues MMAs for each half, one that loads
    static constexpr int THREADS = (LOADER + 1) * 32;
    static constexpr int SMEM = C::HALVES * Q_BYTES + 2 * C::STAGES * KV_BYTES + 384;
    static constexpr int HALF_COLS = C::COLS / C::HALVES;            // S buffers, then O
    static_assert(C::BUFFERS * KEYS + D <= HALF_COLS && C::CTAS * C::COLS <= 512, "tensor memory");
    static_assert(C::CTAS * (SMEM + 1024) <= 228 * 1024, "shared memory");      // (1 KB of each CTA is the system's)
};

struct TcParams {
    CmePaged a;
    PagedDiv page, heads, parts;           // slots of a page; key heads whose tiles are taken together; splits
    int group, row_tile, half_rows, box, box_log, splits, split_keys, tiles, by_keys;
    float scale_log2;
    float* part_o;
    float2* part_ml;
    int* status;
};

__device__ __forceinline__ void tma_load_4d(uint32_t dst, const CUtensorMap* m, uint64_t* bar, int c0, int c1, int c2, int c3) {
    asm volatile(
        "cp.async.bulk.tensor.4d.shared::cta.global.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4, %5, %6}], [%2];"
        ::"r"(dst), "l"(reinterpret_cast<uint64_t>(m)), "r"(smem_u32(bar)), "r"(c0), "r"(c1), "r"(c2), "r"(c3)
        : "memory");
}
__device__ __forceinline__ float max3(float a, float b, float c) {
    float y;
    asm("max.f32 %0, %1, %2, %3;" : "=f"(y) : "f"(a), "f"(b), "f"(c));
    return y;
}
__device__ __forceinline__ uint32_t swz(int r, int c) { return (uint32_t)(r * 128 + ((c ^ (r & 7)) << 4)); }

template <int D, bool FEW>
__global__ void __launch_bounds__(Sizes<D, FEW>::THREADS, Sizes<D, FEW>::CTAS)
paged_attn_tc_kernel(const __grid_constant__ CUtensorMap tmQ, const __grid_constant__ CUtensorMap tmK,
                     const __grid_constant__ CUtensorMap tmV, const TcParams p) {
    using C = Sizes<D, FEW>;
    extern __shared__ __align__(1024) uint8_t smem[];
    if (smem_u32(smem) & 1023u) {             // swizzled tiles need a 1024-byte aligned base
        if (threadIdx.x == 0 && p.status) atomicExch(p.status, CME_ERR_SHAPE);
        return;
    }
    uint8_t* sQ = smem;
    uint8_t* sK = sQ + C::HALVES * C::Q_BYTES;
    uint8_t* sV = sK + C::STAGES * C::KV_BYTES;
    uint64_t* bars = reinterpret_cast<uint64_t*>(sV + C::STAGES * C::KV_BYTES);
    uint64_t* q_full = bars;
    uint64_t* k_full = bars + 1;              // [stage]
    uint64_t* v_full = k_full + C::STAGES;
    uint64_t* k_empty = v_full + C::STAGES;   // its products are complete
    uint64_t* v_empty = k_empty + C::STAGES;
    uint64_t* s_full = v_empty + C::STAGES;   // [half][buffer] S_j is ready (one buffer: and P V complete up to block j - 1, two: j - 2)
    // [half][buffer] S_j read, P_j written over it, O rescaled (128 arrivals).  A barrier for each buffer: with two of them a warp may be a step
    // ahead of another one, whose arrival its own for S_{j+1} must not stand in for; S_{j+2} comes when P_j V_j is complete.
    uint64_t* p_ready = s_full + C::HALVES * C::BUFFERS;
    uint64_t* pv_done = p_ready + C::HALVES * C::BUFFERS;     // [half] P_j V_j complete
    uint64_t* o_done = pv_done + C::HALVES;   // [half] the last one
    uint64_t* turn = o_done + C::HALVES;      // (two halves only) [softmax warp] it may take its turn at the exponentials
    uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(turn + (C::HALVES > 1 ? 8 : 0));
    volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);
    static_assert((1 + 4 * C::STAGES + C::HALVES * (2 * C::BUFFERS + 2) + 8) * 8 + 8 <= 384, "barriers");

    const CmePaged& a = p.a;
    const int cols = D == 64 ? a.head_dim : D;                         // of the head (32 or 64)
    const int warp = __shfl_sync(0xffffffffu, threadIdx.x >> 5, 0), lane = threadIdx.x & 31;
    if (warp == C::LOADER && elect_one()) {
        *abort_flag = 0;
        mbar_init(q_full, 1);
        for (int s = 0; s < C::STAGES; ++s) {
            mbar_init(&k_full[s], 1);
            mbar_init(&v_full[s], 1);
            mbar_init(&k_empty[s], C::HALVES);
            mbar_init(&v_empty[s], C::HALVES);
        }
        for (int h = 0; h < C::HALVES; ++h) {
            for (int b = 0; b < C::BUFFERS; ++b) {
                mbar_init(&s_full[h * C::BUFFERS + b], 1);
                mbar_init(&p_ready[h * C::BUFFERS + b], 128);
            }
            mbar_init(&pv_done[h], 1);
            mbar_init(&o_done[h], 1);
        }
        for (int w = 0; w < (C::HALVES > 1 ? 8 : 0); ++w) mbar_init(&turn[w], 1);
        fence_barrier_init();
        prefetch_tmap(&tmQ);
        prefetch_tmap(&tmK);
        prefetch_tmap(&tmV);
    }
    __syncwarp();                             // the loading lanes see the barriers
    if (warp == 0) { tmem_alloc(tmem_slot, C::COLS); tmem_relinquish(); }
    pdl_wait();
    // Where not all CTAs run at once, tiles that see the most keys first (above 32 sequences: late tiles); of all heads, or (two halves, which
    // take more keys a clock out of L2) of one to four, so that fewer heads' keys are in use at a time.  us, late tiles first / most keys
    // first: 16 chunks of GPT-2 small 31.9 / 26.3, 16 of 1024 77 / 72; head size 128 (there head by head), two of up to 2048 over 8192 328 /
    // 321, four 396 / 377.
    const int at = p.heads.div(blockIdx.x), head = blockIdx.y * p.heads.d + blockIdx.x - at * p.heads.d;
    const int tile = p.parts.div(at), split = at - tile * p.splits;
    const PagedTile t = p.by_keys ? paged_find_tile_by_keys(a, tile, p.group, p.row_tile, KEYS)
                                     : paged_find_tile(a, p.tiles - 1 - tile, p.group, p.row_tile);
    if (t.rows == 0) {
        if (warp == 0) { __syncwarp(); tmem_dealloc(*tmem_slot, C::COLS); }
        return;
    }
    const int limit = max(0, min(a.max_len, t.length - t.n + (t.first + t.rows - 1) / p.group + 1));
    const int begin = (int)min((long long)limit, (long long)split * p.split_keys);
    const int end = (int)min((long long)limit, (long long)begin + p.split_keys);
    const int nkv = cme_cdiv_dev(end - begin, KEYS);
    const int halves = t.rows > p.half_rows ? C::HALVES : 1;           // with rows

    // Of tile j's boxes lane b's page and slot (the lanes of a warp count to eight, again and again)
    const int b = lane & 7;
    auto lookup = [&](int j, int& page, int& slot) {
        const int key = begin + j * KEYS + b * p.box;
        page = -1;
        slot = 0;
        if (j < nkv && key < end && b < KEYS >> p.box_log) {
            const int col = p.page.div(key);
            slot = key - col * p.page.d;
            page = a.pages[t.seq * a.pages_ld + col];
            if (page < 0 || page >= a.num_pages) page = a.num_pages;
        }
    };
    // The warp that loads: lanes 0-15 keys, 16-31 values, a lane one box and slab of each tile.  It looks up the next tile's pages while it
    // waits for a stage.  (Done by the warp that issues the MMAs, the loads of a tile held these up by 2500 clocks.)
    int page0 = -1, slot0 = 0, loaded = 0;
    auto load_tiles = [&](int upto) {
        const int slab = (lane >> 3) & 1;
        const bool values = lane >= 16;
        const uint32_t dst = smem_u32(values ? sV : sK) + slab * C::KV_SLAB + b * p.box * 128;
        for (; loaded < upto; ++loaded) {
            const int s = loaded % C::STAGES;
            int page1, slot1;
            lookup(loaded + 1, page1, slot1);
            bool free = true;
            if (loaded >= C::STAGES) {
                const uint32_t parity = (loaded / C::STAGES - 1) & 1;
                free = mbar_wait(&k_empty[s], parity, abort_flag) && mbar_wait(&v_empty[s], parity, abort_flag);
            }
            if (!__all_sync(0xffffffffu, free)) return false;
            if ((lane & 15) == 0) {
                const int boxes = cme_cdiv_dev(min(KEYS, end - begin - loaded * KEYS), p.box);
                mbar_arrive_expect_tx(values ? &v_full[s] : &k_full[s], (uint32_t)(boxes * p.box * D * 2));
            }
            __syncwarp();
            if (page0 >= 0 && slab < C::SLABS)
                tma_load_4d(dst + s * C::KV_BYTES, values ? &tmV : &tmK, values ? &v_full[s] : &k_full[s], slab * 64, slot0, head, page0);
            page0 = page1;
            slot0 = slot1;
        }
        return true;
    };
    if (warp == C::LOADER && nkv > 0) {
        if (elect_one()) {
            mbar_arrive_expect_tx(q_full, (uint32_t)(halves * p.half_rows * D * 2));
            for (int h = 0; h < halves; ++h)
                for (int s = 0; s < C::SLABS; ++s)
                    tma_load_4d(smem_u32(sQ) + h * C::Q_BYTES + s * C::Q_SLAB, &tmQ, q_full, s * 64, head * p.group,
                                t.token0 + (t.first + h * p.half_rows) / p.group, 0);
        }
        __syncwarp();
        lookup(0, page0, slot0);
        load_tiles(min(nkv, C::STAGES));
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem_base = *tmem_slot;
    pdl_release();

    constexpr uint32_t idesc_s = make_idesc(1, false, false, 128, KEYS);      // Q K^T: both K-major
    constexpr uint32_t idesc_o = make_idesc(1, false, true, 128, D);          // P V: V is MN-major
    const uint64_t q_desc = make_smem_desc(smem_u32(sQ), 0, 1024), k_desc = make_smem_desc(smem_u32(sK), 0, 1024);
    const uint64_t v_desc = make_smem_desc(smem_u32(sV), C::KV_SLAB, 1024);
    auto issue_s = [&](int half, int j, uint32_t tmem_S) {
        const uint64_t qd = desc_at(q_desc, (half * C::Q_BYTES) >> 4), kd = desc_at(k_desc, ((j % C::STAGES) * C::KV_BYTES) >> 4);
#pragma unroll
        for (int k = 0; k < D / 16; ++k)
            mma_f16_ss(tmem_S, desc_at(qd, ((k >> 2) * C::Q_SLAB + (k & 3) * 32) >> 4),
                       desc_at(kd, ((k >> 2) * C::KV_SLAB + (k & 3) * 32) >> 4), idesc_s, k > 0);
    };
    auto issue_pv = [&](int j, uint32_t tmem_O, uint32_t tmem_P) {
        const uint64_t vd = desc_at(v_desc, ((j % C::STAGES) * C::KV_BYTES) >> 4);
#pragma unroll
        for (int k = 0; k < KEYS / 16; ++k)                  // A = P from tensor memory: 16 keys = 8 columns per step
            mma_f16_ts(tmem_O, tmem_P + k * 8, desc_at(vd, k * 2048 >> 4), idesc_o, j > 0 || k > 0);
    };
    bool ok = true;

    if (warp >= 4 * C::HALVES) {
        if (warp == C::LOADER) {
            ok = load_tiles(nkv);
        } else if (elect_one()) {
            // ---------------- MMAs of one half (one thread) ----------------
            const int half = warp - 4 * C::HALVES;
            const uint32_t tmem_S = tmem_base + half * C::HALF_COLS, tmem_O = tmem_S + C::BUFFERS * KEYS;
            if (half < halves) {
                // PTX orders two MMAs only if they accumulate in the same place, and S_j takes the columns of the P before it there: it is issued
                // once that P V is complete.
                auto scores = [&](int j) {
                    if (!mbar_wait(&k_full[j % C::STAGES], (j / C::STAGES) & 1, abort_flag) ||
                        (j >= C::BUFFERS && !mbar_wait(&pv_done[half], (j - C::BUFFERS) & 1, abort_flag))) return false;
                    tc_fence_after();
                    issue_s(half, j, tmem_S + (C::BUFFERS > 1 ? (j & 1) * KEYS : 0));
                    mma_commit(&s_full[half * C::BUFFERS + (C::BUFFERS > 1 ? j & 1 : 0)]);
                    mma_commit(&k_empty[j % C::STAGES]);
                    return true;
                };
                if (nkv > 0) ok = mbar_wait(q_full, 0, abort_flag) && scores(0);
                for (int j = 0; j < nkv && ok; ++j) {
                    if (C::BUFFERS > 1 && j + 1 < nkv && !scores(j + 1)) { ok = false; break; }
                    ok = mbar_wait(&v_full[j % C::STAGES], (j / C::STAGES) & 1, abort_flag) &&
                         (C::BUFFERS > 1 ? mbar_wait(&p_ready[half * C::BUFFERS + (j & 1)], (j >> 1) & 1, abort_flag)
                                         : mbar_wait(&p_ready[half], j & 1, abort_flag));
                    if (!ok) break;
                    tc_fence_after();
                    issue_pv(j, tmem_O, tmem_S + (C::BUFFERS > 1 ? (j & 1) * KEYS : 0));
                    mma_commit(j + 1 < nkv ? &pv_done[half] : &o_done[half]);
                    mma_commit(&v_empty[j % C::STAGES]);
                    if (C::BUFFERS == 1 && j + 1 < nkv) ok = scores(j + 1);
                }
            } else {
                for (int j = 0; j < nkv && ok; ++j) {        // no rows: only hands the tiles back
                    const int s = j % C::STAGES;
                    ok = mbar_wait(&k_full[s], (j / C::STAGES) & 1, abort_flag) && mbar_wait(&v_full[s], (j / C::STAGES) & 1, abort_flag);
                    mbar_arrive(&k_empty[s]);
                    mbar_arrive(&v_empty[s]);
                }
            }
        }
        if (!ok && lane == 0) for (int i = 0; i < 2000; ++i) __nanosleep(500);      // what is in flight ends before the CTA does
    } else if (warp >> 2 < halves) {
        // ---------------- softmax warps: thread = row ----------------
        const int half = warp >> 2;
        const int row = half * p.half_rows + (warp & 3) * 32 + lane;      // of the CTA's tile
        const bool mine = (warp & 3) * 32 + lane < p.half_rows && row < t.rows;
        const uint32_t lane_addr = uint32_t((warp & 3) * 32) << 16;
        const uint32_t tmem_S0 = tmem_base + half * C::HALF_COLS + lane_addr, tmem_O = tmem_S0 + C::BUFFERS * KEYS;
        const int sees = min(end, t.length - t.n + (t.first + row) / p.group + 1);
        const int warp_sees = min(end, t.length - t.n + (t.first + half * p.half_rows + (warp & 3) * 32) / p.group + 1);   // its first row
        float m_ref = -INFINITY, l = 0.f;                 // reference maximum (log2 units) and running row sum
        int page, slot;
        lookup(0, page, slot);
        for (int j = 0; j < nkv; ++j) {
            const uint32_t tmem_S = tmem_S0 + (C::BUFFERS > 1 ? (j & 1) * KEYS : 0);
            const uint32_t there = __ballot_sync(0xffffffffu, page != a.num_pages);      // bit b: box b of the tile
            lookup(j + 1, page, slot);
            ok = C::BUFFERS > 1 ? mbar_wait(&s_full[half * C::BUFFERS + (j & 1)], (j >> 1) & 1, abort_flag)
                                : mbar_wait(s_full, j & 1, abort_flag);
            if (!ok) break;
            tc_fence_after();
            uint32_t r[64];
            tmem_ld32(tmem_S, r);
            tmem_ld32(tmem_S + 32, r + 32);
            tmem_wait_ld();
            const int k0 = begin + j * KEYS;
            if (k0 + KEYS > warp_sees) {                  // diagonal or ragged: keys [0, lim) of this tile are visible to this row
                const int lim = sees - k0;
#pragma unroll
                for (int i = 0; i < 64; ++i) r[i] = i < lim ? r[i] : 0xff800000u;     // -inf
            }
            if (there != 0xffffffffu) {
#pragma unroll
                for (int i = 0; i < 64; ++i) r[i] = (there >> (i >> p.box_log)) & 1 ? r[i] : 0xff800000u;
            }
            float mx4[4];
#pragma unroll
            for (int c = 0; c < 4; ++c) mx4[c] = __uint_as_float(r[c]);
#pragma unroll
            for (int i = 4; i + 8 <= 64; i += 8) {
#pragma unroll
                for (int c = 0; c < 4; ++c)
                    mx4[c] = max3(mx4[c], __uint_as_float(r[i + 2 * c]), __uint_as_float(r[i + 2 * c + 1]));
            }
#pragma unroll
            for (int c = 0; c < 4; ++c) mx4[c] = fmaxf(mx4[c], __uint_as_float(r[60 + c]));
            float mx = fmaxf(max3(mx4[0], mx4[1], mx4[2]), mx4[3]);
            mx *= p.scale_log2;                            // scale > 0, so the maximum commutes with it
            const bool raise = j == 0 || mx > m_ref + (j == 1 ? 0.f : RESCALE_THRESHOLD);
            float alpha = 1.f;
            if (raise) {
                alpha = (m_ref == -INFINITY) ? 0.f : ex2_approx(m_ref - mx);
                m_ref = mx;
            }
            if (j > 0 && __any_sync(0xffffffffu, raise)) {
                // (with one buffer S_j came after P_{j-1} V_{j-1}; with two after P_{j-2} V_{j-2}, so that the parity is that of j - 1)
                if (!mbar_wait(&pv_done[half], (j - 1) & 1, abort_flag)) { ok = false; break; }
                tc_fence_after();
#pragma unroll 1
                for (int c = 0; c < cols / 16; ++c) {      // 16 columns at a time: the score row stays in registers
                    uint32_t o[16];
                    tmem_ld16(tmem_O + c * 16, o);
                    tmem_wait_ld();
#pragma unroll
                    for (int i = 0; i < 16; ++i) o[i] = __float_as_uint(__uint_as_float(o[i]) * alpha);
                    tmem_st16(tmem_O + c * 16, o);
                }
                l *= alpha;
            }
            const float m_use = (m_ref == -INFINITY) ? 0.f : m_ref;
            // The two halves' warps of a scheduler take turns at the exponentials; left alone they fall into step, both wait for the tensor
            // core, and then for one another.
            if (C::HALVES > 1 && halves > 1 && half + j > 0 && !mbar_wait(&turn[warp], (half ? j : j - 1) & 1, abort_flag)) { ok = false; break; }
            // scale-and-shift and the row sum on packed pairs (one instruction per two keys); four independent chains
            const F32x2 sc2 = f2_splat(p.scale_log2), nm2 = f2_splat(-m_use);
            F32x2 sum2[4];
#pragma unroll
            for (int c = 0; c < 4; ++c) sum2[c] = f2_splat(0.f);
#pragma unroll
            for (int c = 0; c < 2; ++c) {
                float* x = reinterpret_cast<float*>(r + c * 32);
#pragma unroll
                for (int i = 0; i < 32; i += 2) f2_unpack(f2_fma(f2_pack(x[i], x[i + 1]), sc2, nm2), x[i], x[i + 1]);
#pragma unroll
                for (int i = 0; i < 32; ++i) x[i] = ex2_approx(x[i]);
#pragma unroll
                for (int i = 0; i < 32; i += 2) sum2[(i >> 1) & 3] = f2_add(sum2[(i >> 1) & 3], f2_pack(x[i], x[i + 1]));
                uint32_t pw[16];
#pragma unroll
                for (int i = 0; i < 16; ++i) pw[i] = f2_to_bf2(x[2 * i], x[2 * i + 1]);
                tmem_st16(tmem_S + c * 16, pw);
            }
            if (C::HALVES > 1 && halves > 1 && lane == 0) mbar_arrive(&turn[warp ^ 4]);
            if (k0 + KEYS > end) {
                // values behind the end may be anything, NaN too, which a probability of zero does not stop: zeros take their place
                const int s = j % C::STAGES;
                if (!mbar_wait(&v_full[s], (j / C::STAGES) & 1, abort_flag)) { ok = false; break; }
                const int from = end - k0, n = (KEYS - from) * C::SLABS * 8;
                for (int i = (warp & 3) * 32 + lane; i < n; i += 128) {
                    const int rr = from + i / (C::SLABS * 8), c = i % (C::SLABS * 8);
                    *reinterpret_cast<uint4*>(sV + s * C::KV_BYTES + (c >> 3) * C::KV_SLAB + swz(rr, c & 7)) = make_uint4(0, 0, 0, 0);
                }
                fence_proxy_async();
            }
            tmem_wait_st();
            tc_fence_before();
            mbar_arrive(&p_ready[C::BUFFERS > 1 ? half * C::BUFFERS + (j & 1) : half]);
            float s0, s1;
            f2_unpack(f2_add(f2_add(sum2[0], sum2[1]), f2_add(sum2[2], sum2[3])), s0, s1);
            l += s0 + s1;
        }
        // (a barrier of its own: the parity of pv_done does not tell the last phase from the one before the one before)
        if (ok && nkv > 0) ok = mbar_wait(&o_done[half], 0, abort_flag);
        if (ok) {
            tc_fence_after();
            const int rr = t.first + row, tok = rr / p.group;
            const long long at = (long long)(t.token0 + tok) * a.heads + head * p.group + rr - tok * p.group;
            if (p.splits == 1) {
                // the warp's rows through its part of the Q tile (every product is complete), then whole rows to memory
                const float inv = l == 0.f ? 0.f : 1.f / l;
                uint8_t* stage = sQ + half * C::Q_BYTES + (warp & 3) * 4096;
#pragma unroll 1
                for (int c = 0; c < cols / 32; ++c) {
                    uint32_t o32[32];
                    if (nkv > 0) { tmem_ld32(tmem_O + c * 32, o32); tmem_wait_ld(); }
                    float* o = reinterpret_cast<float*>(o32);
#pragma unroll
                    for (int i = 0; i < 32; ++i) o[i] = l == 0.f ? 0.f : o[i] * inv;
#pragma unroll
                    for (int g = 0; g < 4; ++g)
                        *reinterpret_cast<uint4*>(stage + (c >> 1) * C::Q_SLAB + swz(lane, (c & 1) * 4 + g)) = pack8(o + g * 8);
                }
                __syncwarp();
                __nv_bfloat16* out = static_cast<__nv_bfloat16*>(a.o);
#pragma unroll
                for (int i = 0; i < D / 8; ++i) {
                    const int src = i * 32 + lane, r = src / (D / 8), c = src % (D / 8);
                    const long long to = __shfl_sync(0xffffffffu, mine ? at : -1ll, r);
                    if (to >= 0 && c * 8 < cols)
                        *reinterpret_cast<uint4*>(out + to * cols + c * 8) =
                            *reinterpret_cast<const uint4*>(stage + (c >> 3) * C::Q_SLAB + swz(r, c & 7));
                }
                if (mine) a.lse[at] = l == 0.f ? -INFINITY : m_ref == -INFINITY ? l : (m_ref + log2f(l)) / LOG2E;
            } else {
                const long long part = at * p.splits + split;
                if (nkv > 0) {
#pragma unroll 1
                    for (int c = 0; c < cols / 32; ++c) {
                        uint32_t o[32];
                        tmem_ld32(tmem_O + c * 32, o);
                        tmem_wait_ld();
                        if (mine) {
#pragma unroll
                            for (int i = 0; i < 32; i += 4)
                                *reinterpret_cast<uint4*>(p.part_o + part * cols + c * 32 + i) = make_uint4(o[i], o[i + 1], o[i + 2], o[i + 3]);
                        }
                    }
                }
                if (mine) p.part_ml[part] = make_float2(m_ref, l);
            }
        }
    }
    tc_fence_before();
    __syncthreads();
    if (threadIdx.x == 0 && *abort_flag && p.status) atomicExch(p.status, CME_ERR_TIMEOUT);
    if (warp == 0) { tc_fence_after(); tmem_dealloc(tmem_base, C::COLS); }
}

// Shared memory of a CTA that keeps more than `each` of them off an SM.  Where CTAs are few the hardware still puts several on one SM
// (chunks of GPT-2 small, 1 / 2 / 8 sequences, us: 19.3 / 19.0 / 25.6, spread over the SMs 17.6 / 17.1 / 24.5).
constexpr int spread(int each) { return 228 * 1024 / (each + 1); }

template <int D, bool FEW> int launch(const CmePaged* a, const PagedPlan& plan, long long ctas, int sms, TcParams& p, cudaStream_t st) {
    using C = Sizes<D, FEW>;
    auto* kernel = paged_attn_tc_kernel<D, FEW>;
    static bool attr[CME_MAX_DEVICES] = {};               // function attributes are per device
    int dev = 0;
    CME_CUDA(cudaGetDevice(&dev));
    if (!attr[dev % CME_MAX_DEVICES]) {
        CME_CUDA(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, C::CTAS > 1 ? spread(1) : C::SMEM));
        attr[dev % CME_MAX_DEVICES] = true;
    }
    p.half_rows = p.row_tile / C::HALVES;
    CUtensorMap mq, mk, mv;
    int rc;
    if ((rc = paged_make_q_map(&mq, a, p.group, p.half_rows / p.group))) return rc;
    if ((rc = paged_make_map(&mk, a, a->k, a->k_page_stride, a->k_head_stride, a->k_slot_stride, 64, p.box, CU_TENSOR_MAP_SWIZZLE_128B))) return rc;
    if ((rc = paged_make_map(&mv, a, a->v, a->v_page_stride, a->v_head_stride, a->v_slot_stride, 64, p.box, CU_TENSOR_MAP_SWIZZLE_128B))) return rc;
    const long long each = std::max(1ll, (ctas + sms - 1) / sms);
    p.by_keys = paged_by_keys(a, p.group) && ctas > (long long)sms * C::CTAS;
    const int smem = each < C::CTAS ? spread((int)each) : C::SMEM;
    CME_CUDA(cme_launch_dependent(kernel, dim3((unsigned)(plan.tiles * plan.splits) * p.heads.d, a->kv_heads / p.heads.d), dim3(C::THREADS), (size_t)smem, st,
                                  mq, mk, mv, p));
    CME_LAUNCH_CHECK();
    return CME_OK;
}

}  // namespace

int paged_attention_tc(const CmePaged* a, const PagedPlan& plan, cudaStream_t st) {
    TcParams p;
    p.a = *a;
    p.page = paged_div(a->page);
    p.group = a->heads / a->kv_heads;
    p.row_tile = plan.row_tile;
    p.box = 1;
    p.box_log = 0;
    while (p.box < KEYS && a->page % (p.box * 2) == 0) { p.box *= 2; ++p.box_log; }
    p.splits = plan.splits;
    p.split_keys = plan.split_keys;
    p.tiles = plan.tiles;
    int heads = a->kv_heads;
    if (a->head_dim == 128) for (heads = 4; a->kv_heads % heads; --heads) {}
    p.heads = paged_div(heads);
    p.parts = paged_div(plan.splits);
    p.scale_log2 = a->scale * LOG2E;
    const long long parts = (long long)a->rows * a->heads * plan.splits;
    p.part_ml = reinterpret_cast<float2*>(a->ws);
    p.part_o = a->ws + (parts * 2 + 3) / 4 * 4;
    p.status = cme_attn_status_ptr();
    CME_REQUIRE(p.status != nullptr, CME_ERR_CUDA, "paged attention: device state unavailable");
    int sms;
    if (const int rc = cme_num_sms(&sms)) return rc;
    const long long ctas = (long long)plan.tiles * plan.splits * a->kv_heads;
    if (a->head_dim == 128) return launch<128, false>(a, plan, ctas, sms, p, st);
    return ctas <= sms * 2ll ? launch<64, true>(a, plan, ctas, sms, p, st) : launch<64, false>(a, plan, ctas, sms, p, st);
}
