// What neighbouring rows of a step share of their pages, and the segments that attention over shared pages works on.
//
// shared[t], the leading tokens that rows t - 1 and t read from the same pages, is found by comparing their table rows, a wave per row. In units of kShareStep
// tokens it is the depth of the boundary between the rows, and the segments are the tree of its intervals: rows between two boundaries of less depth than v
// share v steps, of which their parent's are the lowest. Each boundary finds the nearest ones of less depth, within its wave and then among the others' minima; the first of those
// with the same depth and interval stands for the segment. Segments in more than kShareLevels others are left out: their keys stay with the rows
// or segments within them.
//
// With a window a segment has the keys from the latest window's beginning on, so that all its rows see all its keys and nothing is masked by row; what the
// earlier windows have before that are a row's own.
//
// Bound by latency: the launch, and about four reads of the table one after the other for each 4096 tokens that two rows share; then one workgroup's steps, each of
// which waits for LDS, and with 1024 rows for the issue of four waves' instructions to a SIMD: 9 us for 64 rows, 18 for 1024. A tree of minima for the nearest
// boundaries took 3 us more of either, a search per run for the segment that it begins in 2 to 5 us, arrays indexed by the line (in scratch memory) 2 us.
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

// What a row's segments take of the lines: segments and tiles of the narrow and the wide one, slots, and chunks of the wide one. Two words, for the sums over rows.
struct Count {
    uint64_t places, tiles; // narrow, wide << 16, slots << 32, chunks << 48 (at most five for a row); narrow, wide << 32

    __device__ __forceinline__ int narrow() const { return static_cast<int>(places & 0xFFFF); }
    __device__ __forceinline__ int wide() const { return static_cast<int>(places >> 16 & 0xFFFF); }
    __device__ __forceinline__ int slots() const { return static_cast<int>(places >> 32 & 0xFFFF); }
    __device__ __forceinline__ int chunks() const { return static_cast<int>(places >> 48); }
    __device__ __forceinline__ int narrow_tiles() const { return static_cast<int>(tiles); }
    __device__ __forceinline__ int wide_tiles() const { return static_cast<int>(tiles >> 32); }
};

__device__ __forceinline__ Count operator+(const Count &a, const Count &b) { return {a.places + b.places, a.tiles + b.tiles}; }

// n / d for n below 2^13: (n + 1/2) / d lies 2^-14 of itself or more from whole numbers, and the roundings are off by 2^-22.
__device__ __forceinline__ int quotient(int n, int d) { return static_cast<int>((static_cast<float>(n) + 0.5f) * __builtin_amdgcn_rcpf(static_cast<float>(d))); }

// Depths of the boundaries 0..R (of rows t - 1 and t; none at the ends), in chunks of 64, with each chunk's minima up to a boundary and from it on. The last chunk
// is filled up with depths of 0.
struct Depths {
    int32_t *depth, *upto, *onward;
    int count, chunks;

    __device__ __forceinline__ int32_t at(int i) const { return depth[i]; }
    // A wave's 64 boundaries, of chunk c.
    __device__ __forceinline__ void set(int c, int32_t v) const {
        const int lane = threadIdx.x & 63, i = 64 * c + lane;
        int32_t up = v, on = v;
#pragma unroll 1
        for (int off = 1; off < 64; off <<= 1) {
            const int32_t x = __shfl_up(up, off), y = __shfl_down(on, off);
            up = lane >= off ? min(up, x) : up;
            on = lane + off < 64 ? min(on, y) : on;
        }
        depth[i] = v, upto[i] = up, onward[i] = on;
    }
    // The nearest boundaries before the lane's, of chunk c, and after it with a depth below its own, v > 0. There are some: the ends have depth 0.
    __device__ __forceinline__ int2 nearest(int c, int32_t v) const {
        const int lane = threadIdx.x & 63;
        // Within the chunk by halves: minima of the 2^n boundaries behind each lane and before it, then the longest ways over boundaries that are no less deep.
        // What lies outside the chunk counts as less deep.
        int32_t back[6], ahead[6];
#pragma unroll
        for (int n = 0; n < 6; ++n) {
            const int32_t b = __shfl_up(n == 0 ? v : back[n - 1], n == 0 ? 1 : 1 << (n - 1)), f = __shfl_down(n == 0 ? v : ahead[n - 1], n == 0 ? 1 : 1 << (n - 1));
            back[n] = lane < 1 << n ? -1 : n == 0 ? b : min(back[n - 1], b);
            ahead[n] = lane + (1 << n) > 63 ? -1 : n == 0 ? f : min(ahead[n - 1], f);
        }
        int p = lane, q = lane;
#pragma unroll
        for (int n = 5; n >= 0; --n) {
            const int32_t b = __shfl(back[n], p), f = __shfl(ahead[n], q);
            p -= b >= v ? 1 << n : 0;
            q += f >= v ? 1 << n : 0;
        }
        const bool before = p > 0, after = q < 63; // it is the next one then
        // in other chunks: first which, then where
        int left = -1, right = -1;
#pragma unroll 1
        for (int d = c - 1; d >= 0 && __any(v > 0 && !before && left < 0); --d) {
            left = left < 0 && onward[64 * d] < v ? d : left;
        }
#pragma unroll 1
        for (int d = c + 1; d < chunks && __any(v > 0 && !after && right < 0); ++d) {
            right = right < 0 && onward[64 * d] < v ? d : right;
        }
        int last = 0, first = 0; // of those behind it, one is less deep; of those up to it, none
        if (__any(v > 0 && (!before || !after))) {
#pragma unroll 1
            for (int step = 32; step > 0; step >>= 1) {
                last += onward[64 * max(left, 0) + last + step] < v ? step : 0;
                first += upto[64 * max(right, 0) + first + step - 1] >= v ? step : 0;
            }
        }
        return make_int2(before ? 64 * c + p - 1 : 64 * max(left, 0) + last, after ? 64 * c + q + 1 : right >= 0 ? 64 * right + min(first, 63) : count);
    }
};

// One workgroup, of PER rows a thread at most.
template <int THREADS, int PER> __global__ void __launch_bounds__(THREADS) share_plan_kernel(SharePlanArgs a) {
    extern __shared__ int32_t lds[];
    __shared__ Count waves[THREADS / 64];
    constexpr int kDropped = kShareLevels, kOfWide = 1 << 16;
    const int R = static_cast<int>(a.rows), lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int chunks = (R + 63) / 64;
    const Depths depth{lds, lds + 64 * chunks + 1, lds + 128 * chunks + 1, R, chunks};
    int32_t *alike = lds + 192 * chunks + 1, *parent = alike + R, *level = parent + R, *record = level + R, *lo = record + R;
    int32_t *by_begin = parent, *by_end = level; // before parents and levels are known; ends from 1 on
    int32_t *marks = lo + R;                      // of each run
    const ShareWorkspace ws = carve_share(a.plan, a.rows, a.groups);
    const auto row_of = [&](int j) { return j * THREADS + static_cast<int>(threadIdx.x); };

#pragma unroll 1
    for (int i = threadIdx.x; i < 2 * R; i += THREADS) {
        by_begin[i] = INT32_MAX;
    }
#pragma unroll 1
    for (int i = threadIdx.x; i < (kAttentionWaves + 1) * a.groups; i += THREADS) {
        marks[i] = 0;
    }
    RowKeys keys[PER];
#pragma unroll
    for (int j = 0; j < PER; ++j) {
        const int i = row_of(j);
        const int32_t tokens = i > 0 && i < R ? a.shared[i] : 0;
        keys[j] = i < R ? row_keys(a, i) : RowKeys{0, 0, 0};
        if (i < R) {
            record[i] = keys[j].first; // for the windows' beginnings, until it has its own use
        }
        if (i - lane < R) {
            depth.set(i / 64, tokens / kShareStep);
        }
    }
    if (threadIdx.x == 0) {
        depth.depth[64 * chunks] = 0;
    }
    __syncthreads();
    // ---- the segments of boundaries ----
    int from[PER], to[PER];
#pragma unroll
    for (int j = 0; j < PER; ++j) {
        const int i = row_of(j);
        const int32_t v = i < R ? depth.at(i) : 0;
        const int2 ends = depth.nearest(uniform(i / 64), v);
        from[j] = ends.x, to[j] = ends.y;
        if (v > 0) {
            // One segment alone begins at a boundary and ends at one that is not deeper, and one alone ends at a boundary and begins at a less deep one.
            atomicMin(depth.at(from[j]) >= depth.at(to[j]) ? &by_begin[from[j]] : &by_end[to[j] - 1], i);
        }
    }
    __syncthreads();
#pragma unroll
    for (int j = 0; j < PER; ++j) {
        const int i = row_of(j);
        if (i < R && depth.at(i) > 0) { // the first boundary as deep stands for the segment
            alike[i] = depth.at(from[j]) >= depth.at(to[j]) ? by_begin[from[j]] : by_end[to[j] - 1];
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
#pragma unroll 1
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
#pragma unroll 1
            for (int p = parent[i]; p >= 0 && n < kDropped; p = parent[p]) {
                ++n;
            }
            level[i] = n;
        }
    }
    __syncthreads();

    // ---- segments of each row: its own, what its window leaves before the shared ones, and the boundary's before it ----
    int inner[PER];     // the innermost segment that the row is in, or -1
    int32_t covered[PER]; // the first key of a shared segment
    Count own{0, 0};
    const auto segment_of = [&](int j, int n) __attribute__((always_inline)) {
        const int t = row_of(j);
        ShareSegment s{t, 1, 0, 0, 0, 0, 0, 1};
        const bool alone = covered[j] == INT32_MAX;
        if (n == 0) {
            s.lo = alone ? keys[j].first : depth.at(inner[j]) * kShareStep;
            s.hi = keys[j].end;
        } else if (n == 1) {
            s.lo = keys[j].first;
            s.hi = alone ? 0 : covered[j];
        } else if (t < R && depth.at(t) > 0 && alike[t] == t && level[t] < kDropped) {
            s.row0 = from[j], s.rows = to[j] - from[j];
            s.lo = lo[t], s.hi = depth.at(t) * kShareStep;
        }
        static_assert(kNarrowTile == kWideTile, "of one length");
        s.tiles = s.lo < s.hi ? (s.hi - s.start() + kNarrowTile - 1) / kNarrowTile : 0;
        s.chunk = s.rows;
        return s;
    };
    // Splits the rows of a wide segment evenly; what the segment takes of the lines.
    const auto take = [&](ShareSegment &s) __attribute__((always_inline)) {
        const bool wide = s.rows * a.group_heads > kNarrowCols;
        int chunks = 1;
        if (wide) {
            const int most = kWideCols / a.group_heads;
            chunks = quotient(s.rows + most - 1, most);
            s.chunk = quotient(s.rows + chunks - 1, chunks);
            chunks = quotient(s.rows + s.chunk - 1, s.chunk);
        }
        const uint64_t some = s.tiles > 0 ? 1 : 0;
        const uint64_t tiles = static_cast<uint32_t>(s.tiles) * static_cast<uint32_t>(a.kv_heads * chunks);
        const uint64_t of_wide = wide ? chunks : 0;
        return Count{some << (wide ? 16 : 0) | (some != 0 ? static_cast<uint64_t>(s.rows) << 32 | of_wide << 48 : 0), tiles << (wide ? 32 : 0)};
    };
#pragma unroll
    for (int j = 0; j < PER; ++j) {
        const int t = row_of(j);
        inner[j] = -1, covered[j] = INT32_MAX;
        if (t < R) {
            const int32_t before = depth.at(t), after = t + 1 < R ? depth.at(t + 1) : 0;
            if (max(before, after) > 0) {
                int i = alike[before >= after ? t : t + 1];
                while (level[i] >= kDropped) {
                    i = parent[i];
                }
                inner[j] = i;
#pragma unroll 1
                for (; i >= 0; i = parent[i]) {
                    covered[j] = lo[i] < depth.at(i) * kShareStep ? lo[i] : covered[j];
                }
            }
        }
#pragma unroll 1
        for (int n = 0; n < 3; n += a.window > 0 || n > 0 ? 1 : 2) {
            ShareSegment s = segment_of(j, n);
            own = own + take(s);
        }
    }
    Count upto = own;
#pragma unroll 1
    for (int off = 1; off < 64; off <<= 1) {
        const Count v{__shfl_up(upto.places, off), __shfl_up(upto.tiles, off)};
        upto = lane >= off ? upto + v : upto;
    }
    if (lane == 63) {
        waves[wave] = upto;
    }
    __syncthreads();
    Count at{upto.places - own.places, upto.tiles - own.tiles}, total{0, 0};
#pragma unroll 1
    for (int w = 0; w < THREADS / 64; ++w) {
        at = w < wave ? at + waves[w] : at;
        total = total + waves[w];
    }
    const int of_wide = wide_groups(total.wide_tiles(), static_cast<int64_t>(total.chunks()) * a.kv_heads, total.narrow_tiles(), a.groups);
    const ShareHeader header{{total.narrow_tiles(), total.wide_tiles()}, R, a.group_heads, a.kv_heads, a.groups, of_wide,
                             hm::narrow_runs(total.narrow_tiles(), static_cast<int64_t>(total.narrow()) * a.kv_heads, of_wide, a.groups)};
    if (threadIdx.x == 0) {
        *ws.header = header;
    }
    const int narrow_runs = header.narrow, runs = narrow_runs + header.wide;
    const Runs narrow = Runs::deal(header.tiles[0], narrow_runs), wide = Runs::deal(header.tiles[1], max(header.wide, 1));
    ShareSegment *lines = ws.segments[0];
    const int wide_at = static_cast<int>(ws.segments[1] - lines); // no arrays indexed by the line: they would be in memory
#pragma unroll
    for (int j = 0; j < PER; ++j) {
        const int t = row_of(j);
#pragma unroll 1
        for (int n = 0; n < 3; n += a.window > 0 || n > 0 ? 1 : 2) {
            ShareSegment s = segment_of(j, n);
            const Count c = take(s);
            const bool some = s.tiles > 0, is_wide = s.rows * a.group_heads > kNarrowCols;
            const int place = is_wide ? at.wide() : at.narrow();
            s.tile0 = is_wide ? at.wide_tiles() : at.narrow_tiles();
            s.slot0 = at.slots();
            at = at + c;
            if (some) {
                lines[place + (is_wide ? wide_at : 0)] = s;
                // the first run that begins in the segment or behind it; several may have the same, of which the last counts
                const Runs &of = is_wide ? wide : narrow;
                const int w = s.tile0 > 0 ? of.of(s.tile0 - 1) + 1 : 0;
                if (w < (is_wide ? header.wide : narrow_runs)) {
                    atomicMax(&marks[is_wide ? narrow_runs + w : w], is_wide ? kOfWide + place : place);
                }
            }
            if (n == 0 && t < R && a.window == 0) { // then no keys are left before the shared ones
                ws.paths[R + t] = SharePath{0, 0, 0, 0, 0, 0, 0, 0};
            }
            if (n < 2 && t < R) { // a unit of one row for each key head
                ws.paths[n * R + t] = some ? SharePath{s.tiles, is_wide ? 1 : 0, s.tile0, s.tiles, s.slot0, 1, 0, 0} : SharePath{0, 0, 0, 0, 0, 0, 0, 0};
            }
            if (n == 2 && t < R) {
                record[t] = some ? 2 * place + (is_wide ? 1 : 0) : -1;
            }
        }
    }
    __syncthreads();
#pragma unroll
    for (int j = 0; j < PER; ++j) {
        const int t = row_of(j);
        if (t < R) {
            int which[kShareLevels];
            ShareSegment s[kShareLevels];
            int i = inner[j];
#pragma unroll
            for (int n = 0; n < kShareLevels; ++n) {
                which[n] = i >= 0 ? record[i] : -1;
                i = i >= 0 ? parent[i] : -1;
            }
#pragma unroll
            for (int n = 0; n < kShareLevels; ++n) { // all read at once
                s[n] = lines[(max(which[n], 0) >> 1) + ((max(which[n], 0) & 1) != 0 ? wide_at : 0)];
            }
#pragma unroll
            for (int n = 0; n < kShareLevels; ++n) {
                const int row = t - s[n].row0, chunk = quotient(row, s[n].chunk), chunks = quotient(s[n].rows + s[n].chunk - 1, s[n].chunk);
                ws.paths[(2 + n) * R + t] = which[n] >= 0 ? SharePath{s[n].tiles, which[n] & 1, s[n].tile0 + chunk * s[n].tiles, chunks * s[n].tiles, s[n].slot0, s[n].rows, row,
                                                                      row - chunk * s[n].chunk}
                                                          : SharePath{0, 0, 0, 0, 0, 0, 0, 0};
            }
        }
    }
    // ---- where the runs begin: the last segment marked up to each ----
    const int each = (runs + THREADS - 1) / THREADS, first = min(static_cast<int>(threadIdx.x) * each, runs), last = min(first + each, runs);
    int here = 0;
#pragma unroll 4
    for (int i = first; i < last; ++i) {
        here = max(here, marks[i]);
    }
#pragma unroll 1
    for (int off = 1; off < 64; off <<= 1) {
        const int v = __shfl_up(here, off);
        here = lane >= off ? max(here, v) : here;
    }
    if (lane == 63) {
        waves[wave].places = here;
    }
    const int before = __shfl_up(here, 1);
    here = lane > 0 ? before : 0;
    __syncthreads();
#pragma unroll 1
    for (int w = 0; w < wave; ++w) {
        here = max(here, static_cast<int>(waves[w].places));
    }
    int32_t *starts = ws.starts[0];
    const int wide_starts = static_cast<int>(ws.starts[1] - starts);
#pragma unroll 1
    for (int i = first; i < last; ++i) {
        here = max(here, marks[i]);
        starts[i < narrow_runs ? i : wide_starts + i - narrow_runs] = here & (kOfWide - 1);
    }
}

template <int THREADS, int PER> hipError_t launch_plan(const SharePlanArgs &a, hipStream_t stream) {
    const size_t lds = 4 * static_cast<size_t>(1 + 3 * ((a.rows + 63) / 64 * 64) + 5 * a.rows + (kAttentionWaves + 1) * a.groups);
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
    hipLaunchKernelGGL(shared_tokens_kernel, dim3(static_cast<unsigned>((a.rows + 3) / 4)), dim3(256), 0, stream, a);
    const hipError_t e = hipGetLastError();
    if (e != hipSuccess) {
        return e;
    }
    // 256 rows take 12.7 us with 256 threads and 14.3 with 1024.
    return a.rows <= 256 ? launch_plan<256, 1>(a, stream) : a.rows <= 1024 ? launch_plan<1024, 1>(a, stream) : launch_plan<1024, HM_SHARE_MAX_ROWS / 1024>(a, stream);
}

} // namespace hm
