// Attention of one query token per row over a paged cache in which rows share pages: out = softmax(scale q K^T) V per query head.
//
// A row's keys are cut into segments (hm_share_plan.hip): those that it shares with its neighbours, by levels, and its own. Each is worked on once for all its
// rows, whose query heads are the columns of the matrix products, and gives each column a maximum m, a sum l and an output o relative to it; a second launch joins
// the parts of a column: out = sum of o 2^(m - M) / sum of l 2^(m - M).
//
// Up to 16 columns a segment is bound by the reads of its keys and values, as a row of its own is; it is worked on as in hm_paged_attention.hip, four waves to a tile
// of 128 keys. With more, the four waves share tiles of 64 keys and have up to 32 columns each, as for the rows of prompts; from about 128 columns the matrix
// cores bound it. The tiles of each kind lie in a line that is cut into equal runs, one of each for every workgroup, and half of the workgroups begin with
// the one and half with the other, so that reads and products overlap.
#include "hm_shared_attention.hpp"

namespace hm {
size_t shared_attention_workspace(int64_t rows, int64_t q_heads, int64_t head_dim) {
    const int64_t columns = shared_columns(rows, q_heads, share_groups());
    return static_cast<size_t>((columns + 1) / 2 * 2 * 8 + columns * head_dim * 4);
}

hipError_t launch_shared_attention(SharedAttentionArgs a, hipStream_t stream) {
    a.groups = share_groups();
    a.xcds = device_topology().xcds;
    return a.dtype == HM_FP16 ? launch_shared_attention_f16(a, stream) : launch_shared_attention_bf16(a, stream);
}

} // namespace hm
