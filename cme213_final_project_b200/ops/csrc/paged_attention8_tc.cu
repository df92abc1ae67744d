// Attention of chunks over a paged cache of 8-bit integers on tcgen05 (bf16 queries).
#include "paged_tc.cuh"

int paged_attention8_tc(const CmePaged* a, const CmePagedScales* scales, const PagedPlan& plan, cudaStream_t st) { return run<true>(a, scales, plan, st); }
