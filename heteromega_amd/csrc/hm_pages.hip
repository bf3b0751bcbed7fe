// The page plan of a step: which pages, cache slots and positions its new tokens get, from the requests' lengths.
//
// With n_r tokens held and a_r new ones, pages of P tokens: held_r = ceil(n_r / P), need_r = ceil((n_r + a_r) / P) - held_r,
// first row of r = sum of a before r, first page of r in the ring = head + sum of need before r. Every workgroup makes these
// sums for all requests by itself (one block scan, the results kept in LDS); a row then finds its request by bisecting the first
// rows. That costs a scan per workgroup and saves the launch that would hand the sums over.
//
// Bound by latency: the launch, two dependent reads (lengths, then a table or ring entry), the scan between them and the stores.
// Up to kOneBlockRows rows a single workgroup does all of it. Above, rows and freed pages are dealt over workgroups and one more writes
// lengths and queue after the step. Where these take the place of those before (in-place calls), which the others may still
// have to read, that workgroup is a launch of its own.
#include "hm_device.hpp"
#include "hm_internal.hpp"

#include <algorithm>

namespace hm {
namespace {

constexpr int kMaxRequests = HM_PAGE_PLAN_MAX_REQUESTS;
constexpr int kSmall = 1024; // requests that 256 threads take; more take 512 (2048 requests 7.8 us, with 256 threads 9.9, with 1024 8.5)
constexpr int64_t kOneBlockRows = 1024;

__device__ __forceinline__ int64_t pages_of(int64_t tokens, int shift) { return (tokens + (int64_t(1) << shift) - 1) >> shift; }

struct Sums {
    int64_t rows;
    int32_t need, back; // pages: the sum of at most 4096 needs may pass 31 bits only if it passes the ring's size, which ends it (add_pages)
};

// Page counts are only compared with what the ring holds (less than 2^31): larger sums stay there.
__device__ __forceinline__ int32_t add_pages(int32_t a, int32_t b) { return static_cast<int32_t>(min(static_cast<uint32_t>(a) + static_cast<uint32_t>(b), 0x7fffffffu)); }

__device__ __forceinline__ Sums operator+(const Sums &a, const Sums &b) { return {a.rows + b.rows, add_pages(a.need, b.need), add_pages(a.back, b.back)}; }

// The sums over the threads before this one; *total: over all threads.
template <int THREADS> __device__ __forceinline__ Sums sums_before(const Sums &own, Sums (&waves)[THREADS / 64], Sums *total) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    Sums s = own;
#pragma unroll
    for (int off = 1; off < 64; off <<= 1) {
        const Sums v{__shfl_up(s.rows, off), __shfl_up(s.need, off), __shfl_up(s.back, off)};
        if (lane >= off) {
            s = s + v;
        }
    }
    if (lane == 63) {
        waves[wave] = s;
    }
    const Sums up{__shfl_up(s.rows, 1), __shfl_up(s.need, 1), __shfl_up(s.back, 1)};
    __syncthreads();
    Sums before{0, 0, 0}, all{0, 0, 0};
#pragma unroll
    for (int w = 0; w < THREADS / 64; ++w) {
        if (w == wave) {
            before = all;
        }
        all = all + waves[w];
    }
    __syncthreads();
    *total = all;
    return lane > 0 ? before + up : before;
}

__device__ __forceinline__ uint32_t ring_place(uint64_t counter, uint32_t size) {
    return (counter >> 32) == 0 ? static_cast<uint32_t>(counter) % size : static_cast<uint32_t>(counter % size);
}

// place + k in the ring, k < size.
__device__ __forceinline__ uint32_t ring_after(uint32_t place, uint32_t k, uint32_t size) {
    const uint64_t at = static_cast<uint64_t>(place) + k;
    return static_cast<uint32_t>(at >= size ? at - size : at);
}

// The last request whose first row (or page) is not behind t: those before it with the same first row have no rows.
__device__ __forceinline__ int last_from(const int32_t *first, int count, int32_t t) {
    int lo = 0, hi = count - 1;
    while (lo < hi) {
        const int mid = (lo + hi + 1) >> 1;
        if (first[mid] <= t) {
            lo = mid;
        } else {
            hi = mid - 1;
        }
    }
    return lo;
}

// PER: requests of a thread at most. Workgroups before `row_blocks` write rows, starts, the table and the freed pages; the one behind them, or with `all` the only
// one too, lengths and queue after the step.
template <int THREADS, int PER> __global__ void __launch_bounds__(THREADS) page_plan_kernel(PagePlanArgs a, int row_blocks, bool all) {
    constexpr int kRequests = THREADS * PER;
    __shared__ int32_t first_row[kRequests];  // of each request
    __shared__ int32_t length[kRequests];     // its length, or -1 if it gets nothing
    __shared__ int32_t first_page[kRequests]; // place of its first page in the ring, behind the head
    __shared__ Sums waves[THREADS / 64];
    __shared__ int32_t taken, given_back, refused;
    const bool does_rows = blockIdx.x < static_cast<unsigned>(row_blocks), finishes = all || !does_rows;
    const int R = static_cast<int>(a.requests_count), shift = a.page_shift;
    const uint32_t ring_size = static_cast<uint32_t>(a.ring_size);
    const int64_t capacity = a.width << shift;
    const uint64_t head = static_cast<uint64_t>(a.queue_in[0]), tail = static_cast<uint64_t>(a.queue_in[1]);
    const int per = (R + THREADS - 1) / THREADS, r0 = static_cast<int>(threadIdx.x) * per;
    int32_t n[PER], add[PER];
#pragma unroll
    for (int i = 0; i < PER; ++i) {
        const bool mine = i < per && r0 + i < R;
        n[i] = mine ? a.lengths[r0 + i] : 0;
        add[i] = mine ? a.added[r0 + i] : 0;
    }
    if (threadIdx.x == 0) {
        taken = 0, given_back = 0, refused = 0;
    }
    const uint32_t head_place = ring_place(head, ring_size);
    const int32_t left = static_cast<int32_t>(max(int64_t(0), min(static_cast<int64_t>(tail - head), a.ring_size)));

    // The pages that a request needs count only if its rows fit: first as if all do, again if their sum shows that some do not.
    int32_t need[PER], back[PER];
    Sums before, total;
    bool again = false;
    int64_t row_before = 0;
    do {
        Sums own{0, 0, 0};
        int64_t row = row_before;
#pragma unroll
        for (int i = 0; i < PER; ++i) {
            const int64_t known = min(max(int64_t(n[i]), int64_t(0)), capacity);
            const int64_t held = pages_of(known, shift);
            const int32_t more = max(add[i], 0);
            const bool fits = more > 0 && known == n[i] && n[i] + static_cast<int64_t>(more) <= capacity && row + more <= a.rows;
            need[i] = fits ? static_cast<int32_t>(pages_of(n[i] + static_cast<int64_t>(more), shift) - held) : -1; // -1: refused
            back[i] = add[i] < 0 ? static_cast<int32_t>(held) : 0;
            row += more;
            own = own + Sums{more, max(need[i], 0), back[i]};
        }
        before = sums_before<THREADS>(own, waves, &total);
        row_before = before.rows;
        again = !again && total.rows > a.rows;
    } while (again);
    // A ring smaller than the pages in circulation may not take all that come back: then some requests do not end (the rows and pages of others are as
    // if they did). Pages handed out by this step make room, so entries that are read may be written too: one workgroup does both in turn.
    const int32_t room_before = static_cast<int32_t>(ring_size) - left;
    const bool crowded = total.back > room_before;
    const int writers = crowded ? 1 : row_blocks;
    const bool writes_rows = does_rows && blockIdx.x < static_cast<unsigned>(writers);
    int64_t row = before.rows;
    int32_t page = before.need;
    int32_t my_taken = 0, my_refused = 0;
#pragma unroll
    for (int i = 0; i < PER; ++i) {
        if (i >= per || r0 + i >= R) {
            break;
        }
        const int r = r0 + i;
        const int32_t more = max(add[i], 0);
        const int32_t page_end = add_pages(page, max(need[i], 0));
        const bool served = need[i] == 0 || (need[i] > 0 && page_end <= left);
        if (does_rows) {
            const int32_t first = static_cast<int32_t>(min(row, a.rows));
            first_row[r] = first;
            length[r] = served ? n[i] : -1;
            first_page[r] = page;
            if (blockIdx.x == 0) {
                a.starts[r] = first;
            }
        }
        my_taken = served && need[i] > 0 ? page_end : my_taken;
        if (finishes) {
            my_refused += more > 0 && !served;
            if (add[i] >= 0 || !crowded) {
                a.lengths_out[r] = add[i] < 0 ? 0 : served ? n[i] + more : n[i];
            }
        }
        row += more;
        page = page_end;
    }
    if (my_taken > 0 && (finishes || crowded)) {
        atomicMax(&taken, my_taken);
    }
    if (my_refused > 0) {
        atomicAdd(&refused, my_refused);
    }
    __syncthreads();
    if (crowded) {
        const int32_t room = room_before + taken;
        int32_t to = before.back, my_back = 0, my_kept = 0;
#pragma unroll
        for (int i = 0; i < PER; ++i) {
            if (i < per && r0 + i < R && add[i] < 0) {
                to = add_pages(to, back[i]);
                const bool ends = back[i] == 0 || to <= room;
                my_back = ends && back[i] > 0 ? to : my_back;
                my_kept += !ends;
                if (finishes) {
                    a.lengths_out[r0 + i] = ends ? 0 : n[i];
                }
            }
        }
        if (my_back > 0) {
            atomicMax(&given_back, my_back);
        }
        if (my_kept > 0) {
            atomicAdd(&refused, my_kept);
        }
        __syncthreads();
    }
    const int32_t freed = crowded ? given_back : total.back;
    if (writes_rows) {
        if (blockIdx.x == 0 && threadIdx.x == 0) {
            a.starts[R] = static_cast<int32_t>(min(total.rows, a.rows));
        }
        const int64_t used = min(total.rows, a.rows);
        const int32_t mask = static_cast<int32_t>((int64_t(1) << shift) - 1);
        const int64_t step = static_cast<int64_t>(writers) * THREADS;
        for (int64_t t = static_cast<int64_t>(blockIdx.x) * THREADS + threadIdx.x; t < a.rows; t += step) {
            int64_t slot = -1;
            int32_t position = -1, request = -1;
            if (t < used) {
                const int lo = last_from(first_row, R, static_cast<int32_t>(t));
                const int32_t have = length[lo];
                if (have >= 0) {
                    const int32_t pos = have + static_cast<int32_t>(t - first_row[lo]);
                    const int32_t block = pos >> shift, held = static_cast<int32_t>(pages_of(have, shift));
                    int32_t *entry = a.block_table + lo * a.ld_table + block;
                    int32_t id;
                    if (block < held) {
                        id = *entry;
                    } else {
                        id = a.free_pages[ring_after(head_place, first_page[lo] + block - held, ring_size)];
                        if ((pos & mask) == 0) { // a new page's first token is always among the step's rows
                            *entry = id;
                        }
                    }
                    slot = (static_cast<int64_t>(id) << shift) + (pos & mask);
                    position = pos;
                    request = lo;
                }
            }
            a.slots[t] = slot;
            a.positions[t] = position;
            a.requests[t] = request;
        }
    }
    if (writes_rows && freed > 0) { // pages of ended requests, dealt and found like rows
        __syncthreads();
        int32_t *first_back = first_page;
        int32_t to = before.back;
#pragma unroll
        for (int i = 0; i < PER; ++i) {
            if (i < per && r0 + i < R) {
                first_back[r0 + i] = to;
            }
            to = add_pages(to, back[i]);
        }
        __syncthreads();
        const uint32_t tail_place = ring_place(tail, ring_size);
        for (int64_t j = static_cast<int64_t>(blockIdx.x) * THREADS + threadIdx.x; j < freed; j += static_cast<int64_t>(writers) * THREADS) {
            const int r = last_from(first_back, R, static_cast<int32_t>(j));
            a.free_pages[ring_after(tail_place, static_cast<uint32_t>(j), ring_size)] = a.block_table[r * a.ld_table + (j - first_back[r])];
        }
    }
    if (finishes && threadIdx.x == 0) {
        a.queue_out[0] = static_cast<int64_t>(head + taken);
        a.queue_out[1] = static_cast<int64_t>(tail + freed);
        a.queue_out[2] = refused;
        a.queue_out[3] = total.rows;
    }
}

template <int THREADS, int PER> hipError_t launch(const PagePlanArgs &a, hipStream_t stream) {
    if (a.rows <= kOneBlockRows) {
        hipLaunchKernelGGL((page_plan_kernel<THREADS, PER>), dim3(1), dim3(THREADS), 0, stream, a, 1, true);
        return hipGetLastError();
    }
    const int blocks = static_cast<int>(std::min<int64_t>((a.rows + THREADS - 1) / THREADS, device_topology().cus));
    const bool in_place = a.lengths_out == a.lengths || a.queue_out == a.queue_in;
    hipLaunchKernelGGL((page_plan_kernel<THREADS, PER>), dim3(blocks + (in_place ? 0 : 1)), dim3(THREADS), 0, stream, a, blocks, false);
    const hipError_t e = hipGetLastError();
    if (e != hipSuccess || !in_place) {
        return e;
    }
    hipLaunchKernelGGL((page_plan_kernel<THREADS, PER>), dim3(1), dim3(THREADS), 0, stream, a, 0, false);
    return hipGetLastError();
}

} // namespace

hipError_t launch_page_plan(const PagePlanArgs &a, hipStream_t stream) {
    return a.requests_count <= kSmall ? launch<256, kSmall / 256>(a, stream) : launch<512, kMaxRequests / 512>(a, stream);
}

} // namespace hm
