// Attention of chunks over a paged cache of bf16 on tcgen05.
#include "paged_tc.cuh"

int paged_attention_tc(const CmePaged* a, const PagedPlan& plan, cudaStream_t st) { return run<false>(a, nullptr, plan, st); }
