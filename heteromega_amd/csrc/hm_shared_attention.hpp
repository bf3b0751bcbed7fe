// Attention over shared pages: the plan of what rows share, and the workspace, as the planner (hm_share_plan.hip), the launch
// (hm_shared_attention.hip) and the kernels (hm_shared_attention_kernel.hpp) see them.
#pragma once

#include "hm_paged_attention.hpp"

namespace hm {

constexpr int kShareLevels = 3;                // shared segments that a row may be in, one within the other
constexpr int kPathEntries = kShareLevels + 2; // of a row: its own keys, those that its window leaves before the shared ones, and the shared segments
constexpr int kNarrowCols = 32, kNarrowTile = 32; // units of up to 32 columns: a wave's, in tiles of 32 keys
constexpr int kWideCols = 128, kWideTile = 32; // units of more: a workgroup's, 32 columns per wave, in tiles of 32 keys

// Workgroups, two per CU (with heads of 256 they follow each other). The first ones have a run of the wide line (below) each, the others' waves one of the
// narrow line.
inline int share_groups() { return 2 * device_topology().cus; }
__host__ __device__ __forceinline__ int cols_of(int line) { return line == 0 ? kNarrowCols : kWideCols; }

// The workgroups that the wide line gets: one per CU at most, since two are hardly faster and leave twice the parts, and no more than have four tiles each. A
// wide run has one tile for each 512 narrow ones of the call, so that with many narrow tiles the wide line ends before the narrow one and leaves it most of the
// card: the card reads 500 to 600 tiles of heads of 128 while a workgroup works on one wide tile. 256 rows whose 6.4k keys were shared by all and, mostly, by 8 took
// 67 us so and 79 with a workgroup per CU; 16 384 keys shared by 128 rows with 1024 of their own as long either way, and no less with fewer. To begin and end a
// unit takes a workgroup as long as about eight tiles, which counts where units are short: 84 rows of 32 key heads under a window of 30 keys, with 32 units of a tile or
// two, took 45 us with four of them for each workgroup and 19 with one; 126 rows on 358 keys and 2193 of their own 133 and 94.
__host__ __device__ __forceinline__ int wide_groups(int wide_tiles, int64_t wide_units, int narrow_tiles, int groups) {
    const uint32_t each = static_cast<uint32_t>(narrow_tiles) / 512, long_each = each > 4 ? each : 4, short_each = each > 9 ? each : 9;
    const uint32_t tiles = static_cast<uint32_t>(wide_tiles), units = wide_units < 1 << 24 ? static_cast<uint32_t>(wide_units) : 1u << 24; // more are enough for all
    const uint32_t of_long = (tiles + long_each - 1) / long_each, of_short = (tiles + 8 * units + short_each - 1) / short_each;
    const uint32_t most = of_long > of_short ? of_long : of_short < tiles ? of_short : tiles;
    return most < static_cast<uint32_t>(groups / 2) ? static_cast<int>(most) : groups / 2;
}

// And the narrow line's runs, of one wave each: of two tiles at least where units have eight or more on the average, since each run leaves a part to join (3 rows of 8628
// shared keys, 28 / 4 heads of 128: 21.5 us, and 24.9 with runs of a tile; 16 rows of 1156 keys, 40 / 8 heads: 18.6 and 21.8), else of one (255 rows of 48 keys, 32 / 8
// heads: 15.2 us, and 17.6 with two).
__host__ __device__ __forceinline__ int narrow_runs(int narrow_tiles, int64_t narrow_units, int wide, int groups) {
    const int most = kAttentionWaves * (groups - wide), wanted = narrow_tiles >= 8 * narrow_units ? narrow_tiles / 2 : narrow_tiles, some = wanted > groups ? wanted : groups;
    return some < most ? some : most;
}

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

// What a row has of a segment, for the join: its unit of key head 0 begins at `tile` of its line, and further ones per_head tiles behind; row: in the
// segment, in_chunk: in the unit. tiles 0: nothing.
struct SharePath {
    int32_t tiles, line, tile, per_head;
    int32_t slot0, rows, row, in_chunk;
};

// What a plan was made for, and how many tiles its lines have: a call that does not fit it finds none.
struct ShareHeader {
    int32_t tiles[2]; // narrow, wide
    int32_t rows, group_heads, kv_heads;
    int32_t groups, wide, narrow; // workgroups, those of the wide line, and the narrow line's runs

    __host__ __device__ bool fits(int64_t n, int group, int heads, int g) const { return rows == n && group_heads == group && kv_heads == heads && groups == g; }
    __host__ __device__ int runs(int line) const { return line == 0 ? narrow : wide; }
};

// Memory of a plan. A line's segments are those with tiles, in the order of the line.
struct ShareWorkspace {
    ShareHeader *header;
    ShareSegment *segments[2]; // [3 rows]: narrow, wide
    SharePath *paths;          // [kPathEntries][rows]
    int32_t *starts[2];        // [runs]: the segment that each run begins in
};

__host__ __device__ __forceinline__ int64_t share_plan_bytes(int64_t rows, int groups) {
    return sizeof(ShareHeader) + 6 * rows * static_cast<int64_t>(sizeof(ShareSegment)) + rows * kPathEntries * static_cast<int64_t>(sizeof(SharePath)) +
           (kAttentionWaves + 1) * static_cast<int64_t>(groups) * 4;
}

__host__ __device__ __forceinline__ ShareWorkspace carve_share(void *p, int64_t rows, int groups) {
    ShareHeader *header = static_cast<ShareHeader *>(p);
    ShareSegment *segments = reinterpret_cast<ShareSegment *>(header + 1);
    SharePath *paths = reinterpret_cast<SharePath *>(segments + 6 * rows);
    int32_t *starts = reinterpret_cast<int32_t *>(paths + rows * kPathEntries);
    return {header, {segments, segments + 3 * rows}, paths, {starts, starts + kAttentionWaves * groups}};
}

// The parts of units: a run of a line leaves at most one unit that it does not finish, whose part goes to the run's own columns; the parts that end a unit
// lie by row slot, query head.
struct SharedParts {
    float2 *stats; // m, l of each column
    float *o;      // [columns][D]
};

__host__ __device__ __forceinline__ int64_t shared_columns(int64_t rows, int64_t q_heads, int groups) {
    return rows * kPathEntries * q_heads + static_cast<int64_t>(groups) * (kAttentionWaves * kNarrowCols + kWideCols);
}

__host__ __device__ __forceinline__ SharedParts carve_parts(void *p, int64_t columns) {
    float2 *stats = static_cast<float2 *>(p);
    return {stats, reinterpret_cast<float *>(stats + (columns + 1) / 2 * 2)};
}

// First column of run w's unfinished unit in a line, behind the row slots'.
__host__ __device__ __forceinline__ int64_t run_column(int64_t rows, int64_t q_heads, int groups, int line, int64_t w) {
    return rows * kPathEntries * q_heads + (line == 0 ? w * kNarrowCols : static_cast<int64_t>(groups) * kAttentionWaves * kNarrowCols + w * kWideCols);
}

struct SharedAttentionArgs : PagedAttentionArgs {
    void *plan;
    int groups, xcds;
    int group_heads;
};

hipError_t launch_shared_attention_f16(const SharedAttentionArgs &a, hipStream_t stream);
hipError_t launch_shared_attention_bf16(const SharedAttentionArgs &a, hipStream_t stream);

} // namespace hm
