// Attention over a paged cache of 8-bit integers on warp-level matrix instructions.
#include "paged_mma.cuh"

int paged_attention8_mma(const CmePaged* a, const CmePagedScales* scales, const PagedPlan& plan, cudaStream_t st) {
    return run<true>(a, scales, plan, st);
}
