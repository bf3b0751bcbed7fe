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
constexpr int kPlanThreads = 1024;

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
    // The boundary that stands for the segment of boundary i's depth.
    __device__ __forceinline__ int first_alike(int i) const { return nearest<false, true>(nearest<true, false>(i, at(i)), at(i)); }
};

// One workgroup.
__global__ void __launch_bounds__(kPlanThreads) share_plan_kernel(SharePlanArgs a) {
    extern __shared__ int32_t lds[];
    __shared__ Count waves[kPlanThreads / 64];
    const int R = static_cast<int>(a.rows), lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const Depths depth{lds, a.tree_base};
    int32_t *parent = lds + 2 * a.tree_base, *level = parent + R, *record = level + R, *lo = record + R;
    const ShareWorkspace ws = carve_share(a.plan, a.rows);

    for (int i = threadIdx.x; i < a.tree_base; i += kPlanThreads) {
        lds[a.tree_base + i] = i > 0 && i < R ? a.shared[i] / kShareStep : 0;
    }
    __syncthreads();
    for (int n = a.tree_base >> 1; n > 0; n >>= 1) {
        for (int i = threadIdx.x; i < n; i += kPlanThreads) {
            lds[n + i] = min(lds[2 * (n + i)], lds[2 * (n + i) + 1]);
        }
        __syncthreads();
    }
    // ---- the segments of boundaries: level -1: the boundary stands for none ----
    for (int i = threadIdx.x; i < R; i += kPlanThreads) {
        parent[i] = -1, level[i] = -1;
        const int32_t v = depth.at(i);
        if (v == 0 || depth.first_alike(i) != i) {
            continue;
        }
        const int from = depth.nearest<true, false>(i, v), to = depth.nearest<false, false>(i, v);
        const int32_t above = max(depth.at(from), depth.at(to));
        parent[i] = above == 0 ? -1 : depth.first_alike(depth.at(from) == above ? from : to);
        level[i] = 0;
        int32_t begin = above * kShareStep;
        if (a.window > 0) {
            for (int t = from; t < to; ++t) {
                begin = max(begin, (row_keys(a, t).first + 15) & ~15);
            }
        }
        lo[i] = begin;
    }
    __syncthreads();
    int32_t levels[HM_SHARE_MAX_ROWS / kPlanThreads];
#pragma unroll
    for (int j = 0; j < HM_SHARE_MAX_ROWS / kPlanThreads; ++j) {
        const int i = j * kPlanThreads + static_cast<int>(threadIdx.x);
        levels[j] = -1;
        if (i < R && level[i] == 0) {
            levels[j] = 0;
            for (int p = parent[i]; p >= 0 && levels[j] < kShareLevels; p = parent[p]) {
                ++levels[j];
            }
        }
    }
    __syncthreads();
#pragma unroll
    for (int j = 0; j < HM_SHARE_MAX_ROWS / kPlanThreads; ++j) {
        const int i = j * kPlanThreads + static_cast<int>(threadIdx.x);
        if (i < R) {
            level[i] = levels[j];
        }
    }
    __syncthreads();

    // ---- segments: of rows, what their windows leave before the shared ones, and of boundaries ----
    const auto shared_of = [&](int t) { // the innermost segment that row t is in, or -1
        const int32_t before = depth.at(t), after = t + 1 < R ? depth.at(t + 1) : 0;
        if (max(before, after) == 0) {
            return -1;
        }
        int i = depth.first_alike(before >= after ? t : t + 1);
        while (level[i] >= kShareLevels) {
            i = parent[i];
        }
        return i;
    };
    const auto segment_of = [&](int e) {
        ShareSegment s{0, 0, 0, 0, 0, 0, 0, 1};
        if (e < 2 * R) {
            const int t = e < R ? e : e - R;
            const RowKeys k = row_keys(a, t);
            s.row0 = t, s.rows = 1;
            int i = shared_of(t);
            int32_t covered = INT32_MAX; // the first key of a shared segment
            const int32_t own = i >= 0 ? depth.at(i) * kShareStep : 0;
            for (; i >= 0; i = parent[i]) {
                covered = lo[i] < depth.at(i) * kShareStep ? lo[i] : covered;
            }
            if (e < R) {
                s.lo = covered == INT32_MAX ? k.first : own, s.hi = k.end;
            } else {
                s.lo = k.first, s.hi = covered == INT32_MAX ? 0 : covered;
            }
        } else if (const int i = e - 2 * R; level[i] >= 0 && level[i] < kShareLevels) {
            const int32_t v = depth.at(i);
            s.row0 = depth.nearest<true, false>(i, v);
            s.rows = depth.nearest<false, false>(i, v) - s.row0;
            s.lo = lo[i], s.hi = v * kShareStep;
        }
        const int columns = s.rows * a.group_heads;
        const int tile = columns <= kNarrowCols ? kNarrowTile : kWideTile;
        s.tiles = s.lo < s.hi ? (s.hi - s.start() + tile - 1) / tile : 0;
        if (columns > kNarrowCols) {
            const int most = kWideCols / a.group_heads, chunks = (s.rows + most - 1) / most;
            s.chunk = (s.rows + chunks - 1) / chunks;
        } else {
            s.chunk = s.rows > 0 ? s.rows : 1;
        }
        return s;
    };
    const auto count_of = [&](const ShareSegment &s) {
        if (s.tiles == 0) {
            return Count{0, 0, 0, 0, 0};
        }
        return s.rows * a.group_heads <= kNarrowCols ? Count{1, s.tiles * a.kv_heads, 0, 0, s.rows} : Count{0, 0, 1, s.tiles * a.kv_heads * s.chunks(), s.rows};
    };
    const int all = 3 * R, per = (all + kPlanThreads - 1) / kPlanThreads, e0 = static_cast<int>(threadIdx.x) * per, e1 = min(e0 + per, all);
    Count own{0, 0, 0, 0, 0};
    for (int e = e0; e < e1; ++e) {
        own = own + count_of(segment_of(e));
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
    __syncthreads();
    Count total{0, 0, 0, 0, 0};
    for (int w = 0; w < kPlanThreads / 64; ++w) {
        at = w < wave ? at + waves[w] : at;
        total = total + waves[w];
    }
    if (threadIdx.x == 0) {
        *ws.header = ShareHeader{{{total.narrow, total.narrow_tiles}, {total.wide, total.wide_tiles}}, R, a.group_heads, a.kv_heads, 0};
    }
    for (int e = e0; e < e1; ++e) {
        ShareSegment s = segment_of(e);
        int32_t place = -1;
        if (s.tiles > 0) {
            const bool wide = s.rows * a.group_heads > kNarrowCols;
            s.tile0 = wide ? at.wide_tiles : at.narrow_tiles;
            s.slot0 = at.slots;
            (wide ? ws.wide : ws.narrow)[wide ? at.wide : at.narrow] = s;
            place = wide ? 2 * at.wide + 1 : 2 * at.narrow;
        }
        at = at + count_of(s);
        if (e < 2 * R) {
            ws.paths[(e < R ? e : e - R) * kPathEntries + (e < R ? 0 : 1)] = place;
        } else {
            record[e - 2 * R] = place;
        }
    }
    __syncthreads();
    for (int t = threadIdx.x; t < R; t += kPlanThreads) {
        int i = shared_of(t);
        for (int j = 2; j < kPathEntries; ++j) {
            ws.paths[t * kPathEntries + j] = i >= 0 ? record[i] : -1;
            i = i >= 0 ? parent[i] : -1;
        }
    }
}

} // namespace

size_t share_plan_workspace(int64_t rows) { return static_cast<size_t>(share_plan_bytes(rows)); }

hipError_t launch_share_plan(SharePlanArgs a, hipStream_t stream) {
    a.tree_base = 2;
    while (a.tree_base < a.rows + 1) {
        a.tree_base *= 2;
    }
    const size_t lds = 4 * (2 * static_cast<size_t>(a.tree_base) + 4 * static_cast<size_t>(a.rows));
    if (lds > 64 * 1024) {
        const hipError_t e = hipFuncSetAttribute(reinterpret_cast<const void *>(&share_plan_kernel), hipFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(lds));
        if (e != hipSuccess) {
            return e;
        }
    }
    hipLaunchKernelGGL(shared_tokens_kernel, dim3(static_cast<unsigned>((a.rows + 3) / 4)), dim3(256), 0, stream, a);
    const hipError_t e = hipGetLastError();
    if (e != hipSuccess) {
        return e;
    }
    hipLaunchKernelGGL(share_plan_kernel, dim3(1), dim3(kPlanThreads), lds, stream, a);
    return hipGetLastError();
}

} // namespace hm
