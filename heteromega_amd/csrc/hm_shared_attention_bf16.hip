// The kernels of bf16 caches for attention over shared pages (a file per type, so that they build side by side).
#include "hm_shared_attention_kernel.hpp"

hipError_t hm::launch_shared_attention_bf16(const SharedAttentionArgs &a, hipStream_t stream) { return launch_shared_t<BF16>(a, stream); }
