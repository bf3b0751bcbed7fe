// Attention of one query token per row over a paged cache in which rows share pages: out = softmax(scale q K^T) V per query head.
//
// A row's keys are cut into segments (hm_share_plan.hip): those that it shares with its neighbours, by levels, and its own. Each is worked on once for all its
// rows, whose query heads are the columns of the matrix products, and gives each column a maximum m, a sum l and an output o relative to it; a second launch joins
// the parts of a column: out = sum of o 2^(m - M) / sum of l 2^(m - M).
//
// Up to 32 columns a segment is bound by the reads of its keys and values, as a row of its own is. A wave has a unit (a segment and key head) to itself, in tiles of
// 32 keys that pass through its registers and its part of LDS, and the next tile is on the way meanwhile. With more, up to 128 columns, the four waves of a workgroup
// have 32 each and share tiles of 32 keys; from about 128 columns the matrix cores bound it, and it is worked on as a pipeline of transfers, products and weights.
// (Units of 17 to 32 columns as wide ones, of which one wave in four had work: 88 us instead of 81 at 256 rows in groups of 8 with 4 query heads to a key head.) The tiles of each kind lie in a line that is cut into equal runs. The first workgroups, one per CU at most, have a run of the wide line each, the waves of the
// others one of the narrow line, so that a CU has work that reads and work that multiplies.
//
// 128 rows, 32 / 8 heads of 128, bf16: 16 384 keys shared by all 81 us (424 TFLOP/s; the products of both halves of the weights are 636), 65 536 keys 248 (554 and 831;
// a large product reaches 1199); up to 1024 keys of its own for each row 58 us (5.1 TB/s); both 95 to 107.
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
