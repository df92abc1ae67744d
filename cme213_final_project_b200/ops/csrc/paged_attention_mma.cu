// Attention over a paged cache of bf16 or fp32 on warp-level matrix instructions, and the join of parts that CTAs left in scratch.
#include "paged_mma.cuh"

int paged_mma_key_tile(int dtype, int head_dim, bool q8) { return q8 || head_dim * (dtype == CME_F32 ? 4 : 2) <= 128 ? 128 : 64; }
int paged_mma_ctas(int dtype, int head_dim, bool q8) { return !q8 && dtype == CME_F32 && head_dim == 128 ? 1 : 2; }

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

int paged_attention_mma(const CmePaged* a, const PagedPlan& plan, cudaStream_t st) { return run<false>(a, nullptr, plan, st); }
