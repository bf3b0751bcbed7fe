// The paged attention's kernels of fp16 caches (a file per type, so that they build side by side).
#include "hm_paged_attention_kernel.hpp"

hipError_t hm::launch_paged_attention_f16(const PagedAttentionArgs &a, const AttentionPlan &plan, hipStream_t stream) { return launch_t<F16>(a, plan, stream); }
