// One-token attention over a paged cache: the launch plan and the workspace, shared by the planner (hm_paged_attention.hip) and the
// kernels (hm_paged_attention_kernel.hpp).
#pragma once

#include "hm_internal.hpp"

namespace hm {

constexpr int kAttentionWaves = 4; // of a workgroup

// The prompts' kernel does not split keys: a block of its goes there if it takes less than so many times what all of them take on average per
// place on the card. With an eighth of the places in use both kernels are about as fast (a prompt of 512 rows 38 us, of 256 rows 29, by the
// other kernel 49 and 26; the last 256 of 32768 rows 1296 and 1130, the last 512 1302 and 2378; 32 query and 8 key heads of 128).
constexpr int kPromptShare = 8;

// Tiles of 16 columns that a wave of the prompts' kernel has: two do not fit the registers next to 256 rows of outputs.
constexpr int prompt_tiles(int64_t head_dim) { return head_dim <= 128 ? 2 : 1; }

// A unit's columns are query heads of one key head: of one row, heads of it; or of several rows of one request, all heads of each.
struct Column {
    int row, q_head; // row: behind the unit's first
};

struct AttentionPlan {
    int runs;        // equal shares of the tiles
    int team;        // waves that share a run: 4 or 1
    int cols;        // columns of a unit, up to 32
    int rows;        // rows that a unit may have; 1: it has `cols` heads of one
    int units;       // of a row, or of a unit's rows: key heads times shares of their query heads
    int shares;      // units of one key head
    int group_heads; // query heads of one key head
    bool joins;      // units may have more than one tile, and so parts
    bool counted;    // the rows' tiles are summed up in a launch before, and the limit of prompt blocks
    bool few_units;  // join with a workgroup per unit and column
    int join_cols;   // else: workgroups that share the columns of a unit's join
    int prompt_rows; // rows of a block that the prompts' kernel may take; 0: it is not launched
    int prompt_slots; // its blocks that are on the card at once

    __host__ __device__ int kv_head(int unit) const { return shares == 1 ? unit : unit / shares; }
    // Columns of a unit that has `count` rows. GROUPED: rows > 1.
    template <bool GROUPED> __host__ __device__ int columns(int unit, int count) const {
        if (GROUPED) {
            return count * group_heads;
        }
        const int left = group_heads - (unit - kv_head(unit) * shares) * cols;
        return left < cols ? left : cols;
    }
    template <bool GROUPED> __host__ __device__ Column column(int unit, int j) const {
        const int kv = kv_head(unit);
        if (GROUPED) {
            const int row = j / group_heads;
            return {row, kv * group_heads + j - row * group_heads};
        }
        return {0, kv * group_heads + (unit - kv * shares) * cols + j};
    }
};

// Tiles dealt in equal runs: the first `longer` runs have per_run + 1 tiles, the others per_run.
struct Runs {
    int per_run, longer;

    static __host__ __device__ Runs deal(int tiles, int runs) {
        const int n = static_cast<int>(static_cast<uint32_t>(tiles) / static_cast<uint32_t>(runs));
        return {n, tiles - n * runs};
    }
    __host__ __device__ int begin(int w) const { return w * per_run + (w < longer ? w : longer); }
    // The run of a tile.
    __host__ __device__ int of(int tile) const {
        const uint32_t t = static_cast<uint32_t>(tile), n = static_cast<uint32_t>(per_run), in_longer = static_cast<uint32_t>(longer) * (n + 1);
        return static_cast<int>(t < in_longer ? t / (n + 1) : static_cast<uint32_t>(longer) + (t - in_longer) / n);
    }
};

struct AttentionDescriptor { // of the unit that a run begins and does not finish
    int32_t row, unit, pieces, count; // pieces: runs behind this one that hold its other parts; 0: there is none. count: rows
};

constexpr int kChunks = 64 * kAttentionWaves; // of rows: a thread of a workgroup has the sum of each
constexpr int kCountBytes = kChunks * 4 + 16;

// The workspace of `runs` runs with units of `cols` columns.
struct AttentionWorkspace {
    AttentionDescriptor *desc; // [runs]
    int32_t *counts;           // [kChunks]: tiles of each chunk's rows, and behind them the most keys of a prompt block
    float2 *stats;             // [2 runs][cols]: m, l of each part; part 2 w: of the unit that run w goes on with, 2 w + 1: of the one it begins
    float *o;                  // [2 runs][cols][D]
};

__host__ __device__ __forceinline__ int64_t attention_workspace_bytes(int64_t runs, int64_t cols, int64_t head_dim) {
    return runs * static_cast<int64_t>(sizeof(AttentionDescriptor)) + kCountBytes + (2 * runs * cols * 8 + 15) / 16 * 16 + 2 * runs * cols * head_dim * 4;
}

__host__ __device__ __forceinline__ AttentionWorkspace carve(void *p, int64_t runs, int64_t cols) {
    uint8_t *b = static_cast<uint8_t *>(p);
    uint8_t *counts = b + runs * static_cast<int64_t>(sizeof(AttentionDescriptor)), *stats = counts + kCountBytes;
    return {reinterpret_cast<AttentionDescriptor *>(b), reinterpret_cast<int32_t *>(counts), reinterpret_cast<float2 *>(stats),
            reinterpret_cast<float *>(stats + (2 * runs * cols * 8 + 15) / 16 * 16)};
}

// The launches of one type (hm_paged_attention_f16.hip, hm_paged_attention_bf16.hip).
hipError_t launch_paged_attention_f16(const PagedAttentionArgs &a, const AttentionPlan &plan, hipStream_t stream);
hipError_t launch_paged_attention_bf16(const PagedAttentionArgs &a, const AttentionPlan &plan, hipStream_t stream);

} // namespace hm
