// Attention over shared pages: the plan of what rows share, and the workspace, as the planner (hm_share_plan.hip), the launch
// (hm_shared_attention.hip) and the kernels (hm_shared_attention_kernel.hpp) see them.
#pragma once

#include "hm_paged_attention.hpp"

namespace hm {

constexpr int kShareLevels = 3;                 // shared segments that a row may be in, one within the other
constexpr int kPathEntries = kShareLevels + 2;  // of a row: its own keys, those that its window leaves before the shared ones, and the shared segments
constexpr int kNarrowCols = 16, kNarrowTile = 128; // units of up to 16 columns: tiles of 32 keys per wave
constexpr int kWideCols = 128, kWideTile = 64;     // units of more: 32 columns per wave, which share tiles of 64 keys

// Rows [row0, row0 + rows) that see keys [lo, hi) in the same pages, as a place in one of two lines of tiles: those of narrow units, whose
// rows x query heads of a key head are at most kNarrowCols columns, and of wide ones. A segment has a unit for each key head and, in turn, each `chunk`
// rows. Its units' results lie behind each other from row slot0 on.
struct ShareSegment {
    int32_t row0, rows, lo, hi;
    int32_t tile0, tiles; // of a unit; tile0: of the first
    int32_t slot0, chunk;

    __host__ __device__ int start() const { return lo & ~15; } // of its first tile
    __host__ __device__ int chunks() const { return (rows + chunk - 1) / chunk; }
};

// What the segments of a line come to.
struct ShareLine {
    int32_t segments, tiles;
};

// What a plan was made for: a call that does not fit it finds no segments.
struct ShareHeader {
    ShareLine lines[2]; // narrow, wide
    int32_t rows, group_heads, kv_heads, spare;
};

// Memory of a plan. A line's segments are those with tiles, in the order of the line.
struct ShareWorkspace {
    ShareHeader *header;
    int32_t *paths;         // [rows][kPathEntries]: 2 * segment + line of the row's segments, -1: none
    ShareSegment *narrow;   // [3 rows]
    ShareSegment *wide;     // [3 rows]
};

__host__ __device__ __forceinline__ int64_t share_plan_bytes(int64_t rows) {
    return sizeof(ShareHeader) + (rows * kPathEntries * 4 + 31) / 32 * 32 + 6 * rows * static_cast<int64_t>(sizeof(ShareSegment));
}

__host__ __device__ __forceinline__ ShareWorkspace carve_share(void *p, int64_t rows) {
    uint8_t *b = static_cast<uint8_t *>(p);
    ShareSegment *segments = reinterpret_cast<ShareSegment *>(b + sizeof(ShareHeader) + (rows * kPathEntries * 4 + 31) / 32 * 32);
    return {reinterpret_cast<ShareHeader *>(b), reinterpret_cast<int32_t *>(b + sizeof(ShareHeader)), segments, segments + 3 * rows};
}

// The parts of units: a run of a line leaves at most one unit that it does not finish, whose part goes to the run's own columns; the parts that end a unit
// lie by row slot, query head.
struct SharedParts {
    float2 *stats; // m, l of each column
    float *o;      // [columns][D]
};

__host__ __device__ __forceinline__ int64_t shared_columns(int64_t rows, int64_t q_heads, int64_t runs) {
    return rows * kPathEntries * q_heads + runs * (kNarrowCols + kWideCols);
}

__host__ __device__ __forceinline__ SharedParts carve_parts(void *p, int64_t columns) {
    float2 *stats = static_cast<float2 *>(p);
    return {stats, reinterpret_cast<float *>(stats + (columns + 1) / 2 * 2)};
}

// First column of run w's unfinished unit in a line, behind the row slots'.
__host__ __device__ __forceinline__ int64_t run_column(int64_t rows, int64_t q_heads, int64_t runs, int line, int64_t w) {
    return rows * kPathEntries * q_heads + (line == 0 ? w * kNarrowCols : runs * kNarrowCols + w * kWideCols);
}

struct SharedAttentionArgs : PagedAttentionArgs {
    void *plan;
    int runs;
    int group_heads;
};

hipError_t launch_shared_attention_f16(const SharedAttentionArgs &a, hipStream_t stream);
hipError_t launch_shared_attention_bf16(const SharedAttentionArgs &a, hipStream_t stream);

} // namespace hm
