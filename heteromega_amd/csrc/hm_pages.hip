// The page plan of a step: which pages, cache slots and positions its new tokens get, from the requests' lengths.
//
// With n_r tokens held and a_r new ones, pages of P tokens: held_r = ceil(n_r / P), need_r = ceil((n_r + a_r) / P) - held_r,
// first row of r = sum of a before r, first page of r in the ring = head + sum of need before r. Every workgroup makes both
// sums for all requests by itself (one block scan over at most 4096 requests, kept in LDS); a row then finds its request by
// bisecting the first rows. That costs a scan per workgroup and saves the launch that would hand the sums over.
//
// Bound by latency: two dependent reads (lengths, then a table or ring entry), the scan and the stores. Up to kOneBlockRows
// rows a single workgroup does all of it. Above, the rows are dealt over workgroups and a second, single-workgroup launch
// writes what the first one still reads: lengths, queue and the freed pages.
#include "hm_device.hpp"
#include "hm_internal.hpp"

#include <algorithm>

namespace hm {
namespace {

constexpr int kThreads = 1024;
constexpr int kMaxRequests = HM_PAGE_PLAN_MAX_REQUESTS;
constexpr int kPerThread = kMaxRequests / kThreads;
constexpr int64_t kOneBlockRows = 4096;
constexpr int64_t kRowsPerBlock = 1024;

__device__ __forceinline__ int64_t pages_of(int64_t tokens, int shift) { return (tokens + (int64_t(1) << shift) - 1) >> shift; }

struct Scan {
    int64_t rows, need, back;
};

// Sums of (rows, need, back) over the threads before this one; *total gets the sums over all.
__device__ __forceinline__ Scan block_exclusive(Scan v, Scan (*wave_sums)[kThreads / 64], Scan *total) {
    Scan s = v;
#pragma unroll
    for (int off = 1; off < 64; off <<= 1) {
        const int64_t r = __shfl_up(s.rows, off), n = __shfl_up(s.need, off), b = __shfl_up(s.back, off);
        if ((threadIdx.x & 63) >= static_cast<unsigned>(off)) {
            s.rows += r, s.need += n, s.back += b;
        }
    }
    const int wave = threadIdx.x >> 6;
    if ((threadIdx.x & 63) == 63) {
        (*wave_sums)[wave] = s;
    }
    __syncthreads();
    Scan before{0, 0, 0}, all{0, 0, 0};
    for (int w = 0; w < kThreads / 64; ++w) {
        const Scan t = (*wave_sums)[w];
        if (w < wave) {
            before.rows += t.rows, before.need += t.need, before.back += t.back;
        }
        all.rows += t.rows, all.need += t.need, all.back += t.back;
    }
    __syncthreads();
    *total = all;
    return {before.rows + s.rows - v.rows, before.need + s.need - v.need, before.back + s.back - v.back};
}

// ROWS: writes the rows, the starts and the table; FINISH: writes lengths, queue and the freed pages.
template <bool ROWS, bool FINISH> __global__ void __launch_bounds__(kThreads) page_plan_kernel(PagePlanArgs a) {
    // First row of each request; its length, or -1 if it gets nothing; its first page's place in the ring behind the head.
    __shared__ int32_t first_row[kMaxRequests];
    __shared__ int32_t length[kMaxRequests];
    __shared__ int32_t first_page[kMaxRequests];
    __shared__ Scan wave_sums[kThreads / 64];
    __shared__ unsigned long long taken, refused;
    const int R = static_cast<int>(a.requests_count);
    const int per = (R + kThreads - 1) / kThreads;
    const int r0 = min(static_cast<int>(threadIdx.x) * per, R), r1 = min(r0 + per, R);
    const int64_t capacity = a.width << a.page_shift;
    const uint64_t head = static_cast<uint64_t>(a.queue_in[0]), tail = static_cast<uint64_t>(a.queue_in[1]);
    const int64_t left = max(int64_t(0), min(static_cast<int64_t>(tail - head), a.ring_size));
    if (threadIdx.x == 0) {
        taken = 0, refused = 0;
    }
    int32_t n[kPerThread], add[kPerThread];
    Scan own{0, 0, 0};
#pragma unroll
    for (int i = 0; i < kPerThread; ++i) {
        n[i] = r0 + i < r1 ? a.lengths[r0 + i] : 0;
        add[i] = r0 + i < r1 ? a.added[r0 + i] : 0;
        own.rows += max(add[i], 0);
    }
    Scan total;
    // The rows' sums first: whether a request's rows fit decides whether its pages count.
    Scan rows_before = block_exclusive({own.rows, 0, 0}, &wave_sums, &total);
    const int64_t total_rows = total.rows;
    int64_t need[kPerThread];
    bool valid[kPerThread];
    int64_t row = rows_before.rows;
#pragma unroll
    for (int i = 0; i < kPerThread; ++i) {
        const int64_t known = min(max(int64_t(n[i]), int64_t(0)), capacity);
        const int64_t held = pages_of(known, a.page_shift);
        const int64_t more = max(add[i], 0);
        valid[i] = more > 0 && known == n[i] && n[i] + more <= capacity && row + more <= a.rows;
        need[i] = valid[i] ? pages_of(n[i] + more, a.page_shift) - held : 0;
        own.need += need[i];
        own.back += add[i] < 0 ? held : 0;
        row += more;
    }
    const Scan before = block_exclusive({0, own.need, own.back}, &wave_sums, &total);
    row = rows_before.rows;
    int64_t page = before.need, back = before.back;
    unsigned long long my_taken = 0, my_refused = 0;
#pragma unroll
    for (int i = 0; i < kPerThread; ++i) {
        if (r0 + i >= r1) {
            continue;
        }
        const int r = r0 + i;
        const int64_t more = max(add[i], 0);
        const bool served = valid[i] && (need[i] == 0 || page + need[i] <= left);
        if constexpr (ROWS) {
            first_row[r] = static_cast<int32_t>(min(row, a.rows));
            length[r] = served ? n[i] : -1;
            first_page[r] = static_cast<int32_t>(min(page, a.ring_size));
            if (blockIdx.x == 0) {
                a.starts[r] = first_row[r];
            }
        }
        if constexpr (FINISH) {
            if (served && need[i] > 0) {
                my_taken = static_cast<unsigned long long>(page + need[i]);
            }
            my_refused += more > 0 && !served;
            a.lengths_out[r] = add[i] < 0 ? 0 : served ? static_cast<int32_t>(n[i] + more) : n[i];
        }
        row += more;
        page += need[i];
    }
    if constexpr (FINISH) {
        if (my_taken > 0) {
            atomicMax(&taken, my_taken);
        }
        if (my_refused > 0) {
            atomicAdd(&refused, my_refused);
        }
    }
    __syncthreads();
    if constexpr (ROWS) {
        if (blockIdx.x == 0 && threadIdx.x == 0) {
            a.starts[R] = static_cast<int32_t>(min(total_rows, a.rows));
        }
        const int64_t used = min(total_rows, a.rows);
        const int64_t mask = (int64_t(1) << a.page_shift) - 1;
        for (int64_t t = static_cast<int64_t>(blockIdx.x) * kThreads + threadIdx.x; t < a.rows; t += static_cast<int64_t>(gridDim.x) * kThreads) {
            int64_t slot = -1;
            int32_t position = -1, request = -1;
            if (t < used) {
                // The last request whose first row is not behind t: those of the same first row before it have no rows.
                int lo = 0, hi = R - 1;
                while (lo < hi) {
                    const int mid = (lo + hi + 1) >> 1;
                    if (first_row[mid] <= t) {
                        lo = mid;
                    } else {
                        hi = mid - 1;
                    }
                }
                const int32_t have = length[lo];
                if (have >= 0) {
                    const int64_t pos = have + t - first_row[lo];
                    const int64_t block = pos >> a.page_shift, held = pages_of(have, a.page_shift);
                    int32_t *entry = a.block_table + lo * a.ld_table + block;
                    int32_t id;
                    if (block < held) {
                        id = *entry;
                    } else {
                        id = a.free_pages[(head + static_cast<uint64_t>(first_page[lo] + block - held)) % static_cast<uint64_t>(a.ring_size)];
                        if ((pos & mask) == 0) { // a new page's first token is always among the step's rows
                            *entry = id;
                        }
                    }
                    slot = (static_cast<int64_t>(id) << a.page_shift) + (pos & mask);
                    position = static_cast<int32_t>(pos);
                    request = lo;
                }
            }
            a.slots[t] = slot;
            a.positions[t] = position;
            a.requests[t] = request;
        }
    }
    if constexpr (FINISH) {
        // Freed pages: each wave takes the ended requests among its threads' in turn.
#pragma unroll
        for (int i = 0; i < kPerThread; ++i) {
            const int64_t held = r0 + i < r1 && add[i] < 0 ? pages_of(min(max(int64_t(n[i]), int64_t(0)), capacity), a.page_shift) : 0;
            for (uint64_t ended = __ballot(held > 0); ended != 0; ended &= ended - 1) {
                const int lane = __builtin_ctzll(ended);
                const int64_t count = __shfl(held, lane), to = __shfl(back, lane);
                const int r = __shfl(r0 + i, lane);
                for (int64_t b = threadIdx.x & 63; b < count; b += 64) {
                    a.free_pages[(tail + static_cast<uint64_t>(to + b)) % static_cast<uint64_t>(a.ring_size)] = a.block_table[r * a.ld_table + b];
                }
            }
            back += held;
        }
        if (threadIdx.x == 0) {
            a.queue_out[0] = static_cast<int64_t>(head + taken);
            a.queue_out[1] = static_cast<int64_t>(tail + static_cast<uint64_t>(total.back));
            a.queue_out[2] = static_cast<int64_t>(refused);
            a.queue_out[3] = total_rows;
        }
    }
}

} // namespace

hipError_t launch_page_plan(const PagePlanArgs &a, hipStream_t stream) {
    if (a.rows <= kOneBlockRows) {
        hipLaunchKernelGGL((page_plan_kernel<true, true>), dim3(1), dim3(kThreads), 0, stream, a);
        return hipGetLastError();
    }
    const int64_t blocks = std::min<int64_t>((a.rows + kRowsPerBlock - 1) / kRowsPerBlock, 2 * device_topology().cus);
    hipLaunchKernelGGL((page_plan_kernel<true, false>), dim3(static_cast<unsigned>(blocks)), dim3(kThreads), 0, stream, a);
    const hipError_t e = hipGetLastError();
    if (e != hipSuccess) {
        return e;
    }
    hipLaunchKernelGGL((page_plan_kernel<false, true>), dim3(1), dim3(kThreads), 0, stream, a);
    return hipGetLastError();
}

} // namespace hm
