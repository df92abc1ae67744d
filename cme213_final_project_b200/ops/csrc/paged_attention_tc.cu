// Attention of chunks over a paged cache on tcgen05: not there yet, the rows kernel takes them.
#include "paged.h"

int paged_attention_tc(const CmePaged*, const PagedPlan&, cudaStream_t) {
    CME_REQUIRE(false, CME_ERR_UNSUPPORTED, "paged attention: the tcgen05 kernel is not built");
}
