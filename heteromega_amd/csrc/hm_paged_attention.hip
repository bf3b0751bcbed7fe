// Attention of one query token per row over a paged key-value cache: out = softmax(scale q K^T) V per query head.
//
// Bound by memory: every key and value is read once (4 D bytes per key and key head) for 4 D flops per query head on it, and
// the query heads of a key head (G) are the columns of one or two MFMA tiles, so that they share the reads.
//
// A wave takes 32 keys at a time, as two sub-tiles of 16 keys (a page holds whole sub-tiles):
//   S^T [key, q] = K Q^T   v_mfma_f32_16x16x32: A = K, lane L holds key L & 15 and 8 consecutive elements; B = Q^T, kept in
//                          registers.
//   O^T [d, q] += V^T P^T  A = V^T, read from LDS transposed (ds_read_b64_tr_b16); B = P^T.
// Rows of K and V are loaded whole by neighbouring lanes and pass through LDS, K as well as V: loads in A's own order touch 64
// bytes of 16 rows each, and took 381 us instead of 362 (64 rows of 8192 keys, 8 key heads of 128).
// In S^T a lane holds, for one column q = L & 15, keys 4 (L >> 4) + i of each sub-tile. The k index of the second product may
// be dealt in any order that A and B share, so those eight weights are its B operand as they are: no weight crosses
// lanes. O^T keeps one q per lane too, so rescaling by a new maximum is one factor per lane.
// The scores' running maximum m and the sum l of p = 2^(c s - m) (c = scale log2 e) are fp32. p enters the second product as
// hi + lo, two 16-bit floats of which lo holds what hi lacks (to 2^-16 of p in bf16, 2^-20 in fp16): 16-bit weights alone would add
// an error the size of the output's own rounding, and the matrix cores are idle most of the time here.
//
// Rows differ in length, and their lengths are known on the device only. So the work is dealt in tiles of keys: all tiles of all
// units (a row and a key head, with up to 32 of its query heads) in one line, cut into equal runs. A run may end inside a unit; then
// each run's part (fp32 O, m, l) goes to the workspace and a second launch joins the parts. Every workgroup finds its place by
// summing the rows' tile counts itself, or those of 256 chunks of rows where a launch before has summed them up.
// Where rows must share requests (prompts, drafted tokens: a call of more rows than the block table has), the heads of up to 16 / G rows that
// follow each other in one request are a unit, and read the cache once. They are masked one by one. Which rows share is known on the device only, so calls of
// no more rows than the table take units of one row, whatever they hold: 64 rows, 4 of each of 16 requests of 4096 keys, 58 us in a table of up to 63
// requests and 103 to 107 in taller ones, a prompt of 2048 rows 104 us in a table of up to 2047 and 1375 in one of 2048.
// Blocks of many rows of one request go to a kernel of their own (hm_paged_attention_prompt.hpp), in a launch before; what is one is found
// out on the device from the blocks' first and last rows, against a limit that every wave of both kernels sums up, or that the counting launch leaves.
// A run is shared by the four waves of a workgroup, 32 keys of a 128-key tile each, which join over LDS, or is one wave's own. The first
// keeps the parts few; the second wastes nothing on rows shorter than a tile and lets waves go on to their next unit by
// themselves. It is taken where there are units for three of four waves that fit the card (32 query and 8 key heads of 128: 1024 rows of up to 60
// keys 75 -> 46 us, 256 rows of up to 500 keys 61 -> 56 us; 1824 units of up to 218 keys of 64 24 -> 21 us; 1024 units of 2040 keys would
// take 67 us instead of 65).
// Plain reads of 2 GB reach 6.3 TB/s: 64 rows of 8192 keys take 325 us (6.4 TB/s), one row of 130987 keys 91 us (5.9 TB/s with the join); one row
// of 1037 keys takes 10 us, of which the join's launch is 3.
#include "hm_paged_attention.hpp"

#include <algorithm>

namespace hm {
namespace {

// Workgroups per CU. Two where the registers allow it: with three, squeezed into 168 VGPRs, 64 rows of 8192 keys took 358 us instead of
// 330, and with one, one row of 130987 keys took 91 instead of 95, but 32 ragged rows 65 instead of 56.
int64_t workgroups(int64_t head_dim) { return (head_dim > 128 ? 1 : 2) * device_topology().cus; }

// Columns of a unit: 16 rows' heads, or up to 32 heads of a row. Units of several rows with 32 columns do not fit the registers: 2048 rows
// of a prompt took 687 us with them and 415 with 16.
constexpr int kMaxCols = 32, kGroupedCols = 16;

// Rows from which their tiles are summed up in a launch before, where each is looked at once. Up to here every workgroup sums them up itself, which takes
// 8 us per 1000 rows (32 query and 8 key heads of 128: 1100 rows of 100 keys 100 us and with the launch 102, 16 prompts of 512 rows 217 and
// 153, 300 of 100 rows 769 and 514).
constexpr int64_t kCountedRows = 1024;

// A launch has less than 2^32 threads.
constexpr int64_t kMostPromptUnits = int64_t(1) << 23;

// Rows that a unit may have, where rows share requests.
int unit_rows(int64_t group_heads) { return static_cast<int>(std::max<int64_t>(1, kGroupedCols / group_heads)); }

} // namespace

size_t paged_attention_workspace(int64_t q_heads, int64_t kv_heads, int64_t head_dim) {
    // The most columns, with the runs that they may have.
    const int64_t group_heads = q_heads / kv_heads, cols = std::min<int64_t>(kMaxCols, group_heads * unit_rows(group_heads));
    return static_cast<size_t>(attention_workspace_bytes(workgroups(head_dim) * (cols <= 16 ? kAttentionWaves : 1), cols, head_dim));
}

hipError_t launch_paged_attention(const PagedAttentionArgs &a, hipStream_t stream) {
    if (a.rows == 0) {
        return hipSuccess;
    }
    AttentionPlan p;
    p.group_heads = a.q_heads / a.kv_heads;
    p.rows = a.requests != nullptr && a.rows > a.requests_count ? unit_rows(p.group_heads) : 1;
    p.cols = p.rows > 1 ? p.rows * p.group_heads : std::min(kMaxCols, p.group_heads);
    p.shares = (p.group_heads + p.cols - 1) / p.cols;
    p.units = a.kv_heads * p.shares;
    const int64_t all_units = (a.rows + p.rows - 1) / p.rows * p.units, groups = workgroups(a.head_dim);
    const int64_t capacity = a.width << a.page_shift;
    const auto most_tiles = [&](int64_t keys) { return a.rows * p.units * ((capacity + keys - 1) / keys + 1); };
    // All tiles are counted in 32 bits.
    p.team = p.cols <= 16 && all_units >= 3 * groups && most_tiles(32) <= INT32_MAX ? 1 : kAttentionWaves;
    const int64_t most = most_tiles(32 * p.team);
    p.runs = static_cast<int>(std::min(groups * kAttentionWaves / p.team, most));
    p.counted = a.rows > kCountedRows;
    p.joins = capacity > 32 * p.team;
    p.few_units = 16 * all_units < p.runs;
    // Units may have many parts each where there are fewer of them than runs: then a wave per column.
    p.join_cols = std::min(p.cols, 2 * all_units < p.runs ? kMaxCols : 4);
    // Blocks of rows of the prompts' kernel, if there may be enough of them (which are some is found out there).
    const int prompt_rows = 16 * kAttentionWaves * prompt_tiles(a.head_dim) / p.group_heads / p.rows * p.rows;
    const int64_t prompt_units = prompt_rows < 2 ? 0 : a.rows / prompt_rows * a.kv_heads;
    const bool prompts = a.requests != nullptr && a.rows > a.requests_count && p.group_heads <= kGroupedCols && kPromptShare * prompt_units > groups &&
                         prompt_units <= kMostPromptUnits;
    p.prompt_rows = prompts ? prompt_rows : 0;
    p.prompt_slots = static_cast<int>(std::max<int64_t>(1, groups / a.kv_heads));
    return a.dtype == HM_FP16 ? launch_paged_attention_f16(a, p, stream) : launch_paged_attention_bf16(a, p, stream);
}

} // namespace hm
