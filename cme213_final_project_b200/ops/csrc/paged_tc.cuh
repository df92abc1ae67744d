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
//
// Q8: the cache holds 8-bit integers with a scale for each block of tokens and head,  k_t = sk_t k8_t,  v_t = sv_t v8_t.  TMA brings them as they are,
// four more warps turn them into fp16 (five instructions for four; bf16 has a bit too few and takes eight) in the tiles that the tensor core
// reads, so that all operands are fp16:
//   q   times a power of two that takes a row's largest element to 2^14 .. 2^15 (exact for elements down to 2^-32 of that one), which the softmax
//       warps do to their rows first; its inverse belongs to the factor of the exponents, as sk does, of eight keys at a time (the
//       maximum is taken of these groups' maxima times theirs);
//   p   times sv 2^7: log2 sv is added to the exponents x, and the reference maximum M is a row's own one of x + log2 sv, so that no more than 2^15 comes
//       out, whatever scales the keys have that a row does not see.  Rounded to fp16, 2^-11, and what is below 2^-14 to 2^-25: 2^-32 of the
//       row's largest p sv.  l is the sum of the groups' sums times 2^-8 / (2^7 sv) (2^-8: with sv = 2^-100 the sum of 2^27 keys has room).  A part
//       of the keys leaves sums that are divided by l, and M + log2 l: 2^M, sv with it, would go out of range in the join.
//       Values whose sv is below 2^-100, or 2^-100 of a larger one of their tile or before, count as zeros: their p stays in l, which takes no
//       wider range of log2 sv.
// Results are as near to 64 bits as 32-bit sums give (0.0017 of their size; with bf16 operands 0.0023).  Head size 64 has two CTAs an SM: ten warps' registers
// leave no room for three.  16 chunks of GPT-2 small 36 us; two of 1500 to 2048 over 8192, 32 heads of 128 on 8, 414 us, 0.84 PFLOP/s: shared memory,
// which the products' operands take for 1000 of a step's 1400 clocks and the tiles' arrival, reading and writing as fp16 for 400 (without those 361 us).
#pragma once
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

template <int D, bool FEW, bool Q8> struct Cfg;
template <> struct Cfg<64, false, false> {
    static constexpr int HALVES = 1, STAGES = 3, BUFFERS = 1, CTAS = 3, COLS = 128, RAW = 0;
};
template <> struct Cfg<64, true, false> {
    static constexpr int HALVES = 1, STAGES = 3, BUFFERS = 2, CTAS = 2, COLS = 256, RAW = 0;
};
template <> struct Cfg<128, false, false> {
    static constexpr int HALVES = 2, STAGES = 4, BUFFERS = 2, CTAS = 1, COLS = 512, RAW = 0;
};
// (RAW: stages of the 8-bit tiles)
template <> struct Cfg<64, true, true> {
    static constexpr int HALVES = 1, STAGES = 3, BUFFERS = 2, CTAS = 2, COLS = 256, RAW = 3;
};
template <> struct Cfg<128, false, true> {
    static constexpr int HALVES = 2, STAGES = 3, BUFFERS = 2, CTAS = 1, COLS = 512, RAW = 3;
};
constexpr int PER_STAGE = 32;              // of a tile: 8 factors of the exponents, 8 log2 sv, 8 that are added to the exponents, 8 factors of l
template <int D, bool FEW, bool Q8_> struct Sizes : Cfg<D, FEW, Q8_> {
    using C = Cfg<D, FEW, Q8_>;
    static constexpr bool Q8 = Q8_;
    static constexpr int SLABS = D / 64;                              // 64 columns = 128 bytes each
    static constexpr int Q_SLAB = 128 * 128, KV_SLAB = KEYS * 128;
    static constexpr int Q_BYTES = SLABS * Q_SLAB, KV_BYTES = SLABS * KV_SLAB;
    static constexpr int LOADER = 5 * C::HALVES;                      // four warps of softmax and one that issues MMAs for each half, one that loads
    static constexpr int CONVERTERS = Q8 ? 4 : 0;                     // warps, behind the one that loads
    static constexpr int THREADS = (LOADER + 1 + CONVERTERS) * 32;
    static constexpr int RAW_TILE = KEYS * D;                         // bytes of 8-bit keys, or values
    static constexpr int RAW_BYTES = Q8 ? 2 * RAW_TILE + 64 : 0;      // of a stage: both and their 16 scales
    static constexpr int FACTORS = Q8 ? C::STAGES * PER_STAGE * 4 : 0;           // bytes: what the scales come to
    static constexpr int SMEM = C::HALVES * Q_BYTES + 2 * C::STAGES * KV_BYTES + C::RAW * RAW_BYTES + FACTORS + 384;
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
    CmePagedScales scales;                 // Q8
    PagedDiv block;                        // Q8: tokens of a scale
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

template <int D, bool FEW, bool Q8>
__global__ void __launch_bounds__(Sizes<D, FEW, Q8>::THREADS, Sizes<D, FEW, Q8>::CTAS)
paged_attn_tc_kernel(const __grid_constant__ CUtensorMap tmQ, const __grid_constant__ CUtensorMap tmK,
                     const __grid_constant__ CUtensorMap tmV, const TcParams p) {
    using C = Sizes<D, FEW, Q8>;
    extern __shared__ __align__(1024) uint8_t smem[];
    if (smem_u32(smem) & 1023u) {             // swizzled tiles need a 1024-byte aligned base
        if (threadIdx.x == 0 && p.status) atomicExch(p.status, CME_ERR_SHAPE);
        return;
    }
    uint8_t* sQ = smem;
    uint8_t* sK = sQ + C::HALVES * C::Q_BYTES;
    uint8_t* sV = sK + C::STAGES * C::KV_BYTES;
    uint8_t* sRaw = sV + C::STAGES * C::KV_BYTES;              // Q8: [stage] keys and values, then [stage] 8 scales of keys, 8 of values
    float* sRawScales = reinterpret_cast<float*>(sRaw + C::RAW * 2 * C::RAW_TILE);
    float* sFactors = reinterpret_cast<float*>(sRaw + C::RAW * C::RAW_BYTES);    // Q8: [stage of values][PER_STAGE]
    uint64_t* bars = reinterpret_cast<uint64_t*>(sRaw + C::RAW * C::RAW_BYTES + C::FACTORS);
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
    uint64_t* raw_full = turn + (C::HALVES > 1 ? 8 : 0);      // Q8: [stage] 8-bit tiles and scales are there
    uint64_t* raw_empty = raw_full + C::RAW;
    uint64_t* q_ready = raw_empty + C::RAW;                   // Q8: [half] Q as fp16 (128 arrivals)
    uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(q_ready + (Q8 ? C::HALVES : 0));
    volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);
    static_assert((1 + 4 * C::STAGES + C::HALVES * (2 * C::BUFFERS + 2) + 8 + 2 * C::RAW + C::HALVES) * 8 + 8 <= 384, "barriers");

    const CmePaged& a = p.a;
    const int cols = D == 64 ? a.head_dim : D;                         // of the head (32 or 64)
    const int warp = __shfl_sync(0xffffffffu, threadIdx.x >> 5, 0), lane = threadIdx.x & 31;
    if (warp == C::LOADER && elect_one()) {
        *abort_flag = 0;
        mbar_init(q_full, 1);
        for (int s = 0; s < C::STAGES; ++s) {
            mbar_init(&k_full[s], Q8 ? C::CONVERTERS : 1);
            mbar_init(&v_full[s], Q8 ? C::CONVERTERS : 1);
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
        for (int s = 0; s < C::RAW; ++s) { mbar_init(&raw_full[s], 33); mbar_init(&raw_empty[s], C::CONVERTERS); }
        for (int h = 0; h < (Q8 ? C::HALVES : 0); ++h) mbar_init(&q_ready[h], 128);
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
        if constexpr (Q8) {
            const bool values = lane >= 16;
            for (; loaded < upto; ++loaded) {
                const int s = loaded % C::RAW;
                int page1, slot1;
                lookup(loaded + 1, page1, slot1);
                const bool free = loaded < C::RAW || mbar_wait(&raw_empty[s], (loaded / C::RAW - 1) & 1, abort_flag);
                if (!__all_sync(0xffffffffu, free)) return false;
                if (lane == 0) {
                    const int boxes = cme_cdiv_dev(min(KEYS, end - begin - loaded * KEYS), p.box);
                    mbar_arrive_expect_tx(&raw_full[s], (uint32_t)(boxes * p.box * D * 2));
                }
                __syncwarp();
                if (page0 >= 0 && (lane & 15) < 8)
                    tma_load_4d(smem_u32(sRaw) + (s * 2 + values) * C::RAW_TILE + b * p.box * D, values ? &tmV : &tmK, &raw_full[s], 0, slot0, head, page0);
                // the scales of the tile's groups of eight keys, a lane one; zeros where no key is
                const int at = b * 8, key = begin + loaded * KEYS + at;
                const int page = __shfl_sync(0xffffffffu, page0, at >> p.box_log), slot = __shfl_sync(0xffffffffu, slot0, at >> p.box_log) + (at & (p.box - 1));
                const bool in = key < end && page >= 0 && page < a.num_pages;
                const float* src = values ? p.scales.v : p.scales.k;
                if (in) src += (values ? page * p.scales.v_page + head * p.scales.v_head : page * p.scales.k_page + head * p.scales.k_head) + p.block.div(slot);
                if ((lane & 15) < 8)
                    asm volatile("cp.async.ca.shared.global [%0], [%1], 4, %2;" ::"r"(smem_u32(sRawScales + s * 16 + values * 8 + b)), "l"(src), "r"(in ? 4 : 0)
                                 : "memory");
                asm volatile("cp.async.mbarrier.arrive.noinc.shared::cta.b64 [%0];" ::"r"(smem_u32(&raw_full[s])) : "memory");
                page0 = page1;
                slot0 = slot1;
            }
            return true;
        }
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
        load_tiles(min(nkv, Q8 ? C::RAW : C::STAGES));
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem_base = *tmem_slot;
    pdl_release();

    constexpr uint32_t idesc_s = make_idesc(!Q8, false, false, 128, KEYS);    // Q K^T: both K-major
    constexpr uint32_t idesc_o = make_idesc(!Q8, false, true, 128, D);        // P V: V is MN-major
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
        } else if (Q8 && warp > C::LOADER) {
            // ---------------- 8 bits to fp16 ----------------
            constexpr int CH = D / 16, T = C::CONVERTERS * 32;             // 16-byte pieces of a key
            const int tid = threadIdx.x - (C::LOADER + 1) * 32;
            auto convert = [&](const uint8_t* from, uint8_t* to, auto&& kept) {      // kept(row): all ones, or 0 for zeros in its place
#pragma unroll
                for (int i = 0; i < KEYS * CH / T; ++i) {
                    const int at = i * T + tid, r = at / CH, c = at % CH;
                    const uint4 v = *reinterpret_cast<const uint4*>(from + at * 16);
                    const uint32_t k = kept(r);
                    const uint32_t a = (v.x & k) ^ 0x80808080u, b = (v.y & k) ^ 0x80808080u, d = (v.z & k) ^ 0x80808080u, e = (v.w & k) ^ 0x80808080u;
                    const uint4 x = make_uint4(bytes_to_h2(a, 0x4140), bytes_to_h2(a, 0x4342), bytes_to_h2(b, 0x4140), bytes_to_h2(b, 0x4342));
                    const uint4 y = make_uint4(bytes_to_h2(d, 0x4140), bytes_to_h2(d, 0x4342), bytes_to_h2(e, 0x4140), bytes_to_h2(e, 0x4342));
                    // (eight lanes' stores of a row with 128 bytes go to both slabs: the second four begin with their odd piece, in other banks)
                    const bool odd = D == 128 && c >= CH / 2;
                    uint8_t* slab = to + (c >> 2) * C::KV_SLAB;
                    const int c2 = (c & 3) * 2;
                    *reinterpret_cast<uint4*>(slab + swz(r, c2 + odd)) = odd ? y : x;
                    *reinterpret_cast<uint4*>(slab + swz(r, c2 + !odd)) = odd ? x : y;
                }
                fence_proxy_async();
                __syncwarp();
            };
            float largest = 1.f;                                           // scale of values so far, 1 at least
            for (int j = 0; j < nkv; ++j) {
                const int s = j % C::STAGES, r = j % C::RAW;
                const uint32_t parity = (j / C::STAGES - 1) & 1;
                ok = mbar_wait(&raw_full[r], (j / C::RAW) & 1, abort_flag) && (j < C::STAGES || mbar_wait(&k_empty[s], parity, abort_flag));
                if (!ok) break;
                convert(sRaw + r * 2 * C::RAW_TILE, sK + s * C::KV_BYTES, [](int) { return 0xffffffffu; });
                if (lane == 0) mbar_arrive(&k_full[s]);
                ok = j < C::STAGES || mbar_wait(&v_empty[s], parity, abort_flag);
                if (!ok) break;
                const float* sv = sRawScales + r * 16 + 8;
#pragma unroll
                for (int g = 0; g < 8; ++g) largest = sv[g] < INFINITY ? fmaxf(largest, sv[g]) : largest;
                const float least = largest * PAGED_SMALLEST_SCALE;
                if (tid < 8) {
                    // Where the scale of values is not finite or that of keys a NaN, what is added makes infinite probabilities, of which infinite sums
                    // become NaN in the end: a NaN would stay where the mask takes the group from a row.
                    const float f = sv[tid - 8] * p.scale_log2, v = sv[tid], c = log2f(v >= least && v < INFINITY ? v : least);
                    float* to = sFactors + s * PER_STAGE + tid;
                    to[0] = f == f ? f : 0.f;
                    to[8] = c;
                    to[16] = f != f || !(v < INFINITY) ? 0x1p127f : c + 7.f;
                    to[24] = exp2f(-15.f - c);
                }
                convert(sRaw + (r * 2 + 1) * C::RAW_TILE, sV + s * C::KV_BYTES, [&](int row) { return sv[row >> 3] >= least ? 0xffffffffu : 0u; });
                if (lane == 0) { mbar_arrive(&v_full[s]); mbar_arrive(&raw_empty[r]); }
            }
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
                if (nkv > 0) ok = mbar_wait(Q8 ? &q_ready[half] : q_full, 0, abort_flag) && scores(0);
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
        float row_scale = 1.f;                            // Q8: what S of the row is multiplied by
        if constexpr (Q8) {
            if (nkv > 0 && (ok = mbar_wait(q_full, 0, abort_flag))) {
                uint4 x[D / 8];
                uint8_t* base = sQ + half * C::Q_BYTES;
                unsigned most = 0;                        // largest magnitude, as the bits of an fp32 number
#pragma unroll
                for (int c = 0; c < D / 8; ++c) {
                    x[c] = *reinterpret_cast<const uint4*>(base + (c >> 3) * C::Q_SLAB + swz((warp & 3) * 32 + lane, c & 7));
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        const unsigned w = (&x[c].x)[e];
                        most = max(most, max(w & 0x7fff0000u, (w << 16) & 0x7fff0000u));
                    }
                }
                const unsigned up = min(268u - (most >> 23), 253u);        // (as far as its inverse is not denormal)
                const float f = __uint_as_float(up << 23);
                row_scale = __uint_as_float((254u - up) << 23);
#pragma unroll
                for (int c = 0; c < D / 8; ++c) {
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        const float2 y = bf2_to_f2((&x[c].x)[e]);
                        (&x[c].x)[e] = f2_to_h2(y.x * f, y.y * f);
                    }
                    *reinterpret_cast<uint4*>(base + (c >> 3) * C::Q_SLAB + swz((warp & 3) * 32 + lane, c & 7)) = x[c];
                }
                fence_proxy_async();
                mbar_arrive(&q_ready[half]);
            }
        }
        int page, slot;
        lookup(0, page, slot);
        for (int j = 0; j < nkv && ok; ++j) {
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
            const float* factors = sFactors + (j % C::STAGES) * PER_STAGE;
            // (the stage is not filled again before P_j is written)
            if (Q8 && !mbar_wait(&v_full[j % C::STAGES], (j / C::STAGES) & 1, abort_flag)) { ok = false; break; }
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
            float mx, by[8];                               // (by: Q8, the groups' factors of the exponents)
            if constexpr (Q8) {
                float best[8];
#pragma unroll
                for (int g = 0; g < 8; ++g) {
                    const float* x = reinterpret_cast<const float*>(r + g * 8);
                    by[g] = fmaxf(factors[g] * row_scale, 0x1p-126f);      // (above zero: a masked -inf is multiplied by it)
                    best[g] = fmaf(max3(max3(x[0], x[1], x[2]), max3(x[3], x[4], x[5]), fmaxf(x[6], x[7])), by[g], factors[8 + g]);
                }
                mx = max3(max3(best[0], best[1], best[2]), max3(best[3], best[4], best[5]), fmaxf(best[6], best[7]));
            } else {
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
                mx = fmaxf(max3(mx4[0], mx4[1], mx4[2]), mx4[3]);
                mx *= p.scale_log2;                            // scale > 0, so the maximum commutes with it
            }
            const bool raise = j == 0 || mx > m_ref + (j == 1 ? 0.f : RESCALE_THRESHOLD);
            float alpha = 1.f, root = 1.f;                     // (root: Q8, of alpha, which can be 0 where l times it is not)
            if (raise) {
                if (Q8) {
                    root = (m_ref == -INFINITY) ? 0.f : ex2_approx(0.5f * (m_ref - mx));
                    alpha = root * root;
                } else {
                    alpha = (m_ref == -INFINITY) ? 0.f : ex2_approx(m_ref - mx);
                }
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
                l = Q8 ? l * root * root : l * alpha;
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
                for (int i = 0; i < 32; i += 2)
                    f2_unpack(f2_fma(f2_pack(x[i], x[i + 1]), Q8 ? f2_splat(by[c * 4 + (i >> 3)]) : sc2,
                                     Q8 ? f2_splat(factors[16 + c * 4 + (i >> 3)] - m_use) : nm2), x[i], x[i + 1]);
#pragma unroll
                for (int i = 0; i < 32; ++i) x[i] = ex2_approx(x[i]);
                if constexpr (Q8) {
#pragma unroll
                    for (int g = 0; g < 4; ++g) {
                        F32x2 t = f2_add(f2_pack(x[g * 8], x[g * 8 + 1]), f2_pack(x[g * 8 + 2], x[g * 8 + 3]));
                        t = f2_add(t, f2_add(f2_pack(x[g * 8 + 4], x[g * 8 + 5]), f2_pack(x[g * 8 + 6], x[g * 8 + 7])));
                        sum2[g] = f2_fma(t, f2_splat(factors[24 + c * 4 + g]), sum2[g]);
                    }
                } else {
#pragma unroll
                    for (int i = 0; i < 32; i += 2) sum2[(i >> 1) & 3] = f2_add(sum2[(i >> 1) & 3], f2_pack(x[i], x[i + 1]));
                }
                uint32_t pw[16];
#pragma unroll
                for (int i = 0; i < 16; ++i) pw[i] = Q8 ? f2_to_h2(x[2 * i], x[2 * i + 1]) : f2_to_bf2(x[2 * i], x[2 * i + 1]);
                tmem_st16(tmem_S + c * 16, pw);
            }
            if (C::HALVES > 1 && halves > 1 && lane == 0) mbar_arrive(&turn[warp ^ 4]);
            if (!Q8 && k0 + KEYS > end) {
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
        if (Q8) l += l - l;                               // (infinite: NaN)
        if (ok) {
            tc_fence_after();
            const int rr = t.first + row, tok = rr / p.group;
            const long long at = (long long)(t.token0 + tok) * a.heads + head * p.group + rr - tok * p.group;
            constexpr float UNIT = Q8 ? 0x1p-15f : 1.f, RAISED = Q8 ? 8.f : 0.f;       // of the sums over l; log2 of l's own
            if (p.splits == 1) {
                // the warp's rows through its part of the Q tile (every product is complete), then whole rows to memory
                const float inv = l == 0.f ? 0.f : UNIT / l;
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
                if (mine) a.lse[at] = l == 0.f ? -INFINITY : m_ref == -INFINITY ? l : (m_ref + (log2f(l) + RAISED)) / LOG2E;
            } else {
                const long long part = at * p.splits + split;
                const float inv = Q8 ? (l == 0.f ? 0.f : UNIT / l) : 1.f;
                if (nkv > 0) {
#pragma unroll 1
                    for (int c = 0; c < cols / 32; ++c) {
                        uint32_t o[32];
                        tmem_ld32(tmem_O + c * 32, o);
                        tmem_wait_ld();
                        if (mine) {
#pragma unroll
                            for (int i = 0; i < 32; i += 4)
                                *reinterpret_cast<float4*>(p.part_o + part * cols + c * 32 + i) =
                                    make_float4(__uint_as_float(o[i]) * inv, __uint_as_float(o[i + 1]) * inv, __uint_as_float(o[i + 2]) * inv,
                                                __uint_as_float(o[i + 3]) * inv);
                        }
                    }
                }
                if (mine) p.part_ml[part] = !Q8 ? make_float2(m_ref, l) : l == 0.f ? make_float2(-INFINITY, 0.f) : make_float2(m_ref + (log2f(l) + RAISED), 1.f);
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

template <int D, bool FEW, bool Q8> int launch(const CmePaged* a, const PagedPlan& plan, long long ctas, int sms, TcParams& p, cudaStream_t st) {
    using C = Sizes<D, FEW, Q8>;
    auto* kernel = paged_attn_tc_kernel<D, FEW, Q8>;
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
    const auto swizzle = Q8 ? CU_TENSOR_MAP_SWIZZLE_NONE : CU_TENSOR_MAP_SWIZZLE_128B;
    const int cols = Q8 ? D : 64;
    if ((rc = paged_make_map(&mk, a, a->k, a->k_page_stride, a->k_head_stride, a->k_slot_stride, cols, p.box, swizzle, Q8))) return rc;
    if ((rc = paged_make_map(&mv, a, a->v, a->v_page_stride, a->v_head_stride, a->v_slot_stride, cols, p.box, swizzle, Q8))) return rc;
    const long long each = std::max(1ll, (ctas + sms - 1) / sms);
    p.by_keys = paged_by_keys(a, p.group) && ctas > (long long)sms * C::CTAS;
    const int smem = each < C::CTAS ? spread((int)each) : C::SMEM;
    CME_CUDA(cme_launch_dependent(kernel, dim3((unsigned)(plan.tiles * plan.splits) * p.heads.d, a->kv_heads / p.heads.d), dim3(C::THREADS), (size_t)smem, st,
                                  mq, mk, mv, p));
    CME_LAUNCH_CHECK();
    return CME_OK;
}

template <bool Q8> int run(const CmePaged* a, const CmePagedScales* scales, const PagedPlan& plan, cudaStream_t st) {
    TcParams p;
    p.a = *a;
    p.scales = Q8 ? *scales : CmePagedScales{};
    p.block = paged_div(Q8 ? scales->block : 1);
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
    if (a->head_dim == 128) return launch<128, false, Q8>(a, plan, ctas, sms, p, st);
    if constexpr (Q8) return launch<64, true, true>(a, plan, ctas, sms, p, st);
    else return ctas <= sms * 2ll ? launch<64, true, false>(a, plan, ctas, sms, p, st) : launch<64, false, false>(a, plan, ctas, sms, p, st);
}

}  // namespace
