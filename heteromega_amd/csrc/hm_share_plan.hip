// What neighbouring rows of a step share of their pages, and the segments that attention over shared pages works on.
//
// shared[t], the leading tokens that rows t - 1 and t read from the same pages, is found by comparing their table rows, a wave per row. In units of kShareStep
// tokens it is the depth of the boundary between the rows, and the segments are the tree of its intervals: rows between two boundaries of less depth than v
// share v steps, of which their parent's are the lowest. Each boundary finds the nearest ones of less depth by a tree of minima in LDS; the first of those
// with the same depth and interval stands for the segment. Segments in more than kShareLevels others are left out: their keys stay with the rows
// or segments within them.
//
// With a window a segment has the keys from the latest window's beginning on, so that all its rows see all its keys and nothing is masked by row; what the
// earlier windows have before that are a row's own.
//
// Bound by latency: the launch, and about four reads of the table one after the other for each 4096 tokens that two rows share; then a workgroup's scans.
#include "hm_device.hpp"
#include "hm_shared_attention.hpp"

#include <algorithm>

namespace hm {
namespace {

constexpr int kShareStep = 64; // tokens: less is not worth a part of its own
struct RowKeys {
    int32_t request, first, end; // end 0: none
};

__device__ __forceinline__ RowKeys row_keys(const SharePlanArgs &a, int64_t t) {
    const int32_t request = a.requests != nullptr ? a.requests[t] : static_cast<int32_t>(t), pos = a.positions[t];
    const bool good = request >= 0 && request < a.requests_count && pos >= 0 && pos < (a.width << a.page_shift);
    const int32_t end = good ? pos + 1 : 0;
    return {good ? request : 0, a.window > 0 && a.window < end ? end - static_cast<int32_t>(a.window) : 0, end};
}

// A wave per row.
__global__ void __launch_bounds__(256) shared_tokens_kernel(SharePlanArgs a) {
    const int lane = threadIdx.x & 63;
    const int64_t t = static_cast<int64_t>(blockIdx.x) * 4 + (threadIdx.x >> 6);
    if (t >= a.rows) {
        return;
    }
    int32_t shared = 0;
    if (t > 0) {
        const RowKeys mine = row_keys(a, t), other = row_keys(a, t - 1);
        const int32_t most = min(mine.end, other.end);
        const int32_t *p = a.block_table + mine.request * a.ld_table, *q = a.block_table + other.request * a.ld_table;
        const int blocks = static_cast<int>((static_cast<int64_t>(most) + (int64_t(1) << a.page_shift) - 1) >> a.page_shift);
        shared = most;
        constexpr int kAhead = 4;
        for (int b = 0; b < blocks && mine.request != other.request; b += 64 * kAhead) {
            bool differ[kAhead];
#pragma unroll
            for (int i = 0; i < kAhead; ++i) {
                const int at = b + 64 * i + lane;
                differ[i] = at < blocks && p[min(at, blocks - 1)] != q[min(at, blocks - 1)];
            }
            int found = -1;
#pragma unroll
            for (int i = kAhead - 1; i >= 0; --i) {
                const uint64_t who = __ballot(differ[i]);
                found = who != 0 ? b + 64 * i + static_cast<int>(__builtin_ctzll(who)) : found;
            }
            if (found >= 0) {
                shared = static_cast<int32_t>(min(static_cast<int64_t>(most), static_cast<int64_t>(found) << a.page_shift));
                break;
            }
        }
    }
    if (lane == 0) {
        a.shared[t] = shared;
    }
}

struct Count {
    int32_t narrow, narrow_tiles, wide, wide_tiles, slots;
};

__device__ __forceinline__ Count operator+(const Count &a, const Count &b) {
    return {a.narrow + b.narrow, a.narrow_tiles + b.narrow_tiles, a.wide + b.wide, a.wide_tiles + b.wide_tiles, a.slots + b.slots};
}

// Depths of the boundaries 0..R (of rows t - 1 and t; none at the ends), with the minima of pairs, pairs of pairs and so on above them.
struct Depths {
    int32_t *tree;
    int base;

    __device__ __forceinline__ int32_t at(int i) const { return tree[base + i]; }
    // The nearest boundary before i (BACK) or after it with a depth below v, or not above it (EQUAL). There is one: the ends have depth 0.
    template <bool BACK, bool EQUAL> __device__ __forceinline__ int nearest(int i, int32_t v) const {
        const auto fits = [&](int p) { return EQUAL ? tree[p] <= v : tree[p] < v; };
        int p = base + i;
        while (p > 1) {
            if ((p & 1) == (BACK ? 1 : 0) && fits(BACK ? p - 1 : p + 1)) {
                p = BACK ? p - 1 : p + 1;
                break;
            }
            p >>= 1;
        }
        while (p < base) {
            p = 2 * p + (BACK ? 1 : 0);
            if (!fits(p)) {
                p += BACK ? -1 : 1;
            }
        }
        return p - base;
    }
};

__device__ __forceinline__ Count count_of(const SharePlanArgs &a, const ShareSegment &s) {
    if (s.tiles == 0) {
        return Count{0, 0, 0, 0, 0};
    }
    return s.rows * a.group_heads <= kNarrowCols ? Count{1, s.tiles * a.kv_heads, 0, 0, s.rows} : Count{0, 0, 1, s.tiles * a.kv_heads * s.chunks(), s.rows};
}

__device__ __forceinline__ SharePath path_of(const ShareSegment &s, int line, int t) {
    if (s.tiles == 0) {
        return SharePath{0, 0, 0, 0, 0, 0, 0, 0};
    }
    const int row = t - s.row0, chunk = row / s.chunk;
    return SharePath{s.tiles, line, s.tile0 + chunk * s.tiles, s.chunks() * s.tiles, s.slot0, s.rows, row, row - chunk * s.chunk};
}

// One workgroup, of PER rows a thread at most.
template <int THREADS, int PER> __global__ void __launch_bounds__(THREADS) share_plan_kernel(SharePlanArgs a) {
    extern __shared__ int32_t lds[];
    __shared__ Count waves[THREADS / 64];
    constexpr int kDropped = kShareLevels;
    const int R = static_cast<int>(a.rows), lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const Depths depth{lds, a.tree_base};
    int32_t *alike = lds + max(2 * a.tree_base, 3 * R), *parent = alike + R, *level = parent + R, *record = level + R, *lo = record + R;
    const ShareWorkspace ws = carve_share(a.plan, a.rows, a.groups);
    const auto row_of = [&](int j) { return j * THREADS + static_cast<int>(threadIdx.x); };

    for (int i = threadIdx.x; i < a.tree_base; i += THREADS) {
        lds[a.tree_base + i] = i > 0 && i < R ? a.shared[i] / kShareStep : 0;
    }
    RowKeys keys[PER];
#pragma unroll
    for (int j = 0; j < PER; ++j) {
        const int i = row_of(j);
        keys[j] = i < R ? row_keys(a, i) : RowKeys{0, 0, 0};
        if (i < R) {
            record[i] = keys[j].first; // for the windows' beginnings, until it has its own use
        }
    }
    __syncthreads();
    for (int n = a.tree_base >> 1; n > 0; n >>= 1) {
        for (int i = threadIdx.x; i < n; i += THREADS) {
            lds[n + i] = min(lds[2 * (n + i)], lds[2 * (n + i) + 1]);
        }
        __syncthreads();
    }
    // ---- the segments of boundaries ----
    int from[PER], to[PER];
#pragma unroll
    for (int j = 0; j < PER; ++j) {
        const int i = row_of(j);
        const int32_t v = i < R ? depth.at(i) : 0;
        from[j] = to[j] = 0;
        if (v > 0) {
            from[j] = depth.nearest<true, false>(i, v), to[j] = depth.nearest<false, false>(i, v);
            alike[i] = depth.nearest<false, true>(from[j], v); // the boundary that stands for the segment
        }
    }
    __syncthreads();
#pragma unroll
    for (int j = 0; j < PER; ++j) {
        const int i = row_of(j);
        if (i < R && depth.at(i) > 0 && alike[i] == i) {
            const int32_t above = max(depth.at(from[j]), depth.at(to[j]));
            parent[i] = above == 0 ? -1 : alike[depth.at(from[j]) == above ? from[j] : to[j]];
            int32_t begin = above * kShareStep;
            if (a.window > 0) {
                for (int t = from[j]; t < to[j]; ++t) {
                    begin = max(begin, (record[t] + 15) & ~15);
                }
            }
            lo[i] = begin;
        }
    }
    __syncthreads();
#pragma unroll
    for (int j = 0; j < PER; ++j) { // the number of segments that each is within, or that there are too many
        const int i = row_of(j);
        if (i < R && depth.at(i) > 0 && alike[i] == i) {
            int n = 0;
            for (int p = parent[i]; p >= 0 && n < kDropped; p = parent[p]) {
                ++n;
            }
            level[i] = n;
        }
    }
    __syncthreads();

    // ---- segments of each row: its own, what its window leaves before the shared ones, and the boundary's before it ----
    ShareSegment segments[PER][3];
    int inner[PER]; // the innermost segment that the row is in, or -1
    Count own{0, 0, 0, 0, 0};
#pragma unroll
    for (int j = 0; j < PER; ++j) {
        const int t = row_of(j);
        inner[j] = -1;
#pragma unroll
        for (int n = 0; n < 3; ++n) {
            segments[j][n] = ShareSegment{t, 1, 0, 0, 0, 0, 0, 1};
        }
        if (t < R) {
            const int32_t before = depth.at(t), after = t + 1 < R ? depth.at(t + 1) : 0;
            if (max(before, after) > 0) {
                inner[j] = alike[before >= after ? t : t + 1];
                while (level[inner[j]] >= kDropped) {
                    inner[j] = parent[inner[j]];
                }
            }
            int32_t covered = INT32_MAX; // the first key of a shared segment
            for (int i = inner[j]; i >= 0; i = parent[i]) {
                covered = lo[i] < depth.at(i) * kShareStep ? lo[i] : covered;
            }
            segments[j][0].lo = covered == INT32_MAX ? keys[j].first : depth.at(inner[j]) * kShareStep;
            segments[j][0].hi = keys[j].end;
            segments[j][1].lo = keys[j].first;
            segments[j][1].hi = covered == INT32_MAX ? 0 : covered;
            if (before > 0 && alike[t] == t && level[t] < kDropped) {
                segments[j][2].row0 = from[j], segments[j][2].rows = to[j] - from[j];
                segments[j][2].lo = lo[t], segments[j][2].hi = before * kShareStep;
            }
        }
#pragma unroll
        for (int n = 0; n < 3; ++n) {
            ShareSegment &s = segments[j][n];
            const int columns = s.rows * a.group_heads, tile = columns <= kNarrowCols ? kNarrowTile : kWideTile;
            s.tiles = s.lo < s.hi ? (s.hi - s.start() + tile - 1) / tile : 0;
            s.chunk = s.rows;
            if (columns > kNarrowCols) {
                const int most = kWideCols / a.group_heads, chunks = (s.rows + most - 1) / most;
                s.chunk = (s.rows + chunks - 1) / chunks;
            }
            own = own + count_of(a, s);
        }
    }
    Count upto = own;
#pragma unroll
    for (int off = 1; off < 64; off <<= 1) {
        const Count v{__shfl_up(upto.narrow, off), __shfl_up(upto.narrow_tiles, off), __shfl_up(upto.wide, off), __shfl_up(upto.wide_tiles, off),
                      __shfl_up(upto.slots, off)};
        if (lane >= off) {
            upto = upto + v;
        }
    }
    if (lane == 63) {
        waves[wave] = upto;
    }
    Count at{__shfl_up(upto.narrow, 1), __shfl_up(upto.narrow_tiles, 1), __shfl_up(upto.wide, 1), __shfl_up(upto.wide_tiles, 1), __shfl_up(upto.slots, 1)};
    if (lane == 0) {
        at = Count{0, 0, 0, 0, 0};
    }
    __syncthreads(); // the depths are not read any more either: the lines' first tiles take their place
    Count total{0, 0, 0, 0, 0};
#pragma unroll
    for (int w = 0; w < THREADS / 64; ++w) {
        at = w < wave ? at + waves[w] : at;
        total = total + waves[w];
    }
    const ShareHeader header{{total.narrow_tiles, total.wide_tiles}, R, a.group_heads, a.kv_heads, a.groups,
                             wide_groups(total.wide_tiles, total.narrow_tiles, a.groups), 0};
    if (threadIdx.x == 0) {
        *ws.header = header;
    }
    int32_t *tile0[2] = {lds, lds + total.narrow};
#pragma unroll
    for (int j = 0; j < PER; ++j) {
        const int t = row_of(j);
#pragma unroll
        for (int n = 0; n < 3; ++n) {
            ShareSegment &s = segments[j][n];
            const int line = s.rows * a.group_heads > kNarrowCols ? 1 : 0, place = line == 1 ? at.wide : at.narrow;
            if (s.tiles > 0) {
                s.tile0 = line == 1 ? at.wide_tiles : at.narrow_tiles;
                s.slot0 = at.slots;
                ws.segments[line][place] = s;
                tile0[line][place] = s.tile0;
                at = at + count_of(a, s);
            }
            if (n < 2 && t < R) {
                ws.paths[t * kPathEntries + n] = path_of(s, line, t);
            }
            if (n == 2 && t < R) {
                record[t] = s.tiles > 0 ? 2 * place + line : -1;
            }
        }
    }
    __syncthreads();
#pragma unroll
    for (int j = 0; j < PER; ++j) {
        const int t = row_of(j);
        if (t < R) {
            int i = inner[j];
            for (int n = 2; n < kPathEntries; ++n) {
                SharePath p{0, 0, 0, 0, 0, 0, 0, 0};
                if (i >= 0 && record[i] >= 0) {
                    p = path_of(ws.segments[record[i] & 1][record[i] >> 1], record[i] & 1, t);
                }
                ws.paths[t * kPathEntries + n] = p;
                i = i >= 0 ? parent[i] : -1;
            }
        }
    }
    // ---- where the runs begin ----
    const int narrow_runs = header.runs(0);
    for (int i = threadIdx.x; i < narrow_runs + header.runs(1); i += THREADS) {
        const int line = i < narrow_runs ? 0 : 1, w = line == 0 ? i : i - narrow_runs;
        const int count = line == 0 ? total.narrow : total.wide, tiles = line == 0 ? total.narrow_tiles : total.wide_tiles;
        const int x = Runs::deal(tiles, header.runs(line)).begin(w);
        int first = 0, last = count - 1; // the last segment that begins at x or before it
        while (first < last) {
            const int mid = (first + last + 1) >> 1;
            if (tile0[line][mid] <= x) {
                first = mid;
            } else {
                last = mid - 1;
            }
        }
        ws.starts[line][w] = first;
    }
}

template <int THREADS, int PER> hipError_t launch_plan(const SharePlanArgs &a, hipStream_t stream) {
    const size_t lds = 4 * (static_cast<size_t>(std::max<int64_t>(2 * a.tree_base, 3 * a.rows)) + 5 * static_cast<size_t>(a.rows));
    if (lds > 64 * 1024) {
        const hipError_t e = hipFuncSetAttribute(reinterpret_cast<const void *>(&share_plan_kernel<THREADS, PER>), hipFuncAttributeMaxDynamicSharedMemorySize,
                                                 static_cast<int>(lds));
        if (e != hipSuccess) {
            return e;
        }
    }
    hipLaunchKernelGGL((share_plan_kernel<THREADS, PER>), dim3(1), dim3(THREADS), lds, stream, a);
    return hipGetLastError();
}

} // namespace

size_t share_plan_workspace(int64_t rows) { return static_cast<size_t>(share_plan_bytes(rows, share_groups())); }

hipError_t launch_share_plan(SharePlanArgs a, hipStream_t stream) {
    a.groups = share_groups();
    a.tree_base = 2;
    while (a.tree_base < a.rows + 1) {
        a.tree_base *= 2;
    }
    hipLaunchKernelGGL(shared_tokens_kernel, dim3(static_cast<unsigned>((a.rows + 3) / 4)), dim3(256), 0, stream, a);
    const hipError_t e = hipGetLastError();
    if (e != hipSuccess) {
        return e;
    }
    return a.rows <= 256 ? launch_plan<256, 1>(a, stream) : a.rows <= 1024 ? launch_plan<1024, 1>(a, stream) : launch_plan<1024, HM_SHARE_MAX_ROWS / 1024>(a, stream);
}

} // namespace hm
