// Requests that share pages: page_fork (requests become copies or prefixes of others), page_compact (the pages in use move to the front
// of a cache) and copy_pages (the data of both).
//
// Who holds a page is read off the block table itself: a page's keys carry their positions, so all requests that hold it have it as the same
// block, in one column. So each column is worked on by itself, with a hash table of its pages in LDS, and no counts of holders are kept from call to
// call. The columns meet in two sums only: the pages that copies need, in the order of requests, and the pages that come free, in the
// order of blocks. The first launch counts, the second, which repeats the column's work, takes and gives the pages: with the sums known it is one
// pass, and the old columns are read before the new are written, so the table may be changed in place.
//
// Bound by latency: 16 groups of 4 beams of 500 to 2300 tokens have 6000 entries, 24 KB.
#include "hm_device.hpp"
#include "hm_internal.hpp"

#include <algorithm>

namespace hm {
namespace {

constexpr int kMaxRequests = HM_PAGE_PLAN_MAX_REQUESTS;
constexpr int kMaxChunks = 1024; // of columns

// The fork's workspace. Lengths and counters are kept there for the second launch, since lengths_out and queue_out may take their places.
struct ForkWorkspace {
    int64_t *queue;   // [2]: head, tail
    int32_t *chunks;  // [kMaxChunks]: pages that come free in each chunk of columns
    int32_t *lengths; // [R]
    int32_t *fresh;   // [R]: whether the request's last page is to be a fresh one
};

__host__ __device__ __forceinline__ ForkWorkspace carve_fork(void *p, int64_t requests) {
    uint8_t *b = static_cast<uint8_t *>(p);
    int32_t *chunks = reinterpret_cast<int32_t *>(b + 16), *lengths = chunks + kMaxChunks;
    return {reinterpret_cast<int64_t *>(b), chunks, lengths, lengths + requests};
}

// Exclusive sum of v over the workgroup's threads; *total: over all of them.
template <int THREADS> __device__ __forceinline__ int sum_before(int v, int32_t (&waves)[THREADS / 64], int *total) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    int s = v;
#pragma unroll
    for (int off = 1; off < 64; off <<= 1) {
        const int u = __shfl_up(s, off);
        s += lane >= off ? u : 0;
    }
    if (lane == 63) {
        waves[wave] = s;
    }
    __syncthreads();
    int before = 0, all = 0;
#pragma unroll
    for (int w = 0; w < THREADS / 64; ++w) {
        before += w < wave ? waves[w] : 0;
        all += waves[w];
    }
    __syncthreads();
    *total = all;
    return before + s - v;
}

__device__ __forceinline__ int32_t pages_of(int32_t tokens, int shift) {
    return static_cast<int32_t>((static_cast<uint32_t>(tokens) + ((1u << shift) - 1)) >> shift);
}

// The place of a page among a column's, taken if it has none. The column has at most half as many pages as the table has places.
__device__ __forceinline__ int place_of(int32_t *keys, int bits, int32_t page) {
    uint32_t h = static_cast<uint32_t>(page) * 2654435761u >> (32 - bits);
    for (;;) {
        const int32_t k = keys[h];
        if (k == page) {
            return static_cast<int>(h);
        }
        if (k < 0) {
            const int32_t was = atomicCAS(&keys[h], -1, page);
            if (was < 0 || was == page) {
                return static_cast<int>(h);
            }
        }
        h = (h + 1) & ((1u << bits) - 1);
    }
}

// THREADS threads of at most PER requests each, a chunk of columns per workgroup. APPLY: the second launch.
template <int THREADS, int PER, bool APPLY> __global__ void __launch_bounds__(THREADS) fork_kernel(PageForkArgs a) {
    extern __shared__ int32_t lds[];
    __shared__ int32_t waves[THREADS / 64];
    __shared__ int32_t most;
    constexpr int kNobody = INT32_MAX;
    const int R = static_cast<int>(a.requests_count), shift = a.page_shift, bits = a.hash_bits;
    const int32_t page_tokens = 1 << shift;
    const ForkWorkspace ws = carve_fork(a.workspace, a.requests_count);
    int32_t *length = lds, *after = length + R, *source = after + R; // tokens before and after, and the source or -1
    int32_t *keys = source + R, *holder = keys + (1 << bits), *owner = holder + (1 << bits);
    const int32_t *lengths = APPLY ? ws.lengths : a.lengths;
    const int per = (R + THREADS - 1) / THREADS, r0 = static_cast<int>(threadIdx.x) * per;
    const int32_t capacity = static_cast<int32_t>(a.width << shift);

    // ---- the requests ----
    if (threadIdx.x == 0) {
        most = 0;
    }
    bool bad = false;
    for (int r = threadIdx.x; r < R; r += THREADS) {
        const int32_t n = lengths[r], s = a.sources[r];
        bad |= n < 0 || n > capacity || s >= R || (a.keep != nullptr && a.keep[r] < 0);
        length[r] = n;
        source[r] = s < 0 ? -1 : s;
    }
    bad = __syncthreads_or(bad);
    int held_most = 0;
    for (int r = threadIdx.x; r < R; r += THREADS) {
        const int32_t s = source[r], n = bad || s < 0 ? 0 : length[s];
        after[r] = a.keep != nullptr ? min(n, a.keep[r]) : n;
        held_most = max(held_most, bad ? 0 : pages_of(length[r], shift));
    }
#pragma unroll
    for (int off = 32; off > 0; off >>= 1) {
        held_most = max(held_most, __shfl_xor(held_most, off));
    }
    if ((threadIdx.x & 63) == 0) {
        atomicMax(&most, held_most);
    }
    __syncthreads();
    const int columns = most;
    const int chunk = (columns + gridDim.x - 1) / gridDim.x;
    const int first_column = min(static_cast<int>(blockIdx.x) * chunk, columns), last_column = min(first_column + chunk, columns);

    // ---- what the first launch found ----
    const uint64_t head = static_cast<uint64_t>(APPLY ? ws.queue[0] : a.queue_in[0]), tail = static_cast<uint64_t>(APPLY ? ws.queue[1] : a.queue_in[1]);
    const uint64_t Q = static_cast<uint64_t>(a.ring_size);
    int freed_before = 0;
    int fresh_at[PER]; // place of each request's fresh page behind the head, or -1
    bool refused = bad;
    if constexpr (APPLY) {
        int mine = 0, all = 0;
        for (int i = threadIdx.x; i < static_cast<int>(gridDim.x); i += THREADS) {
            const int n = ws.chunks[i];
            mine += i < static_cast<int>(blockIdx.x) ? n : 0;
            all += n;
        }
        int freed = 0, wanted = 0;
        (void)sum_before<THREADS>(mine, waves, &freed_before);
        (void)sum_before<THREADS>(all, waves, &freed);
        int own = 0;
#pragma unroll
        for (int i = 0; i < PER; ++i) {
            const int r = r0 + i;
            fresh_at[i] = i < per && r < R && !bad ? ws.fresh[r] : 0;
            own += fresh_at[i];
        }
        int place = sum_before<THREADS>(own, waves, &wanted);
#pragma unroll
        for (int i = 0; i < PER; ++i) {
            const int next = place + fresh_at[i];
            fresh_at[i] = fresh_at[i] != 0 ? place : -1;
            place = next;
        }
        const int64_t left = max(int64_t(0), min(static_cast<int64_t>(tail - head), static_cast<int64_t>(Q)));
        refused = bad || wanted > left || left + freed > static_cast<int64_t>(Q);
        if (blockIdx.x == 0) {
            for (int r = threadIdx.x; r < R; r += THREADS) {
                a.lengths_out[r] = refused ? length[r] : after[r];
            }
            for (int i = threadIdx.x; i < 3 * R; i += THREADS) {
                if (refused || i >= 3 * wanted) {
                    a.copies[i] = -1;
                }
            }
            if (threadIdx.x == 0) {
                a.queue_out[0] = static_cast<int64_t>(refused ? head : head + wanted);
                a.queue_out[1] = static_cast<int64_t>(refused ? tail : tail + freed);
                a.queue_out[2] = refused;
                a.queue_out[3] = wanted;
            }
        }
        if (refused) { // all stays as it is
            if (a.table_out != a.block_table) {
                for (int64_t i = static_cast<int64_t>(blockIdx.x) * THREADS + threadIdx.x; i < R * a.width; i += static_cast<int64_t>(gridDim.x) * THREADS) {
                    const int64_t r = i / a.width, b = i - r * a.width;
                    if (b << shift < length[r]) {
                        a.table_out[r * a.ld_out + b] = a.block_table[r * a.ld_table + b];
                    }
                }
            }
            return;
        }
    } else {
        if (blockIdx.x == 0) {
            for (int r = threadIdx.x; r < R; r += THREADS) {
                ws.lengths[r] = length[r];
                if ((after[r] & (page_tokens - 1)) == 0) {
                    ws.fresh[r] = 0; // the others' are set where their last page is looked at
                }
            }
            if (threadIdx.x == 0) {
                ws.queue[0] = static_cast<int64_t>(head);
                ws.queue[1] = static_cast<int64_t>(tail);
            }
        }
    }

    // ---- the columns ----
    int freed_here = 0;
    for (int b = first_column; b < last_column; ++b) {
        for (int i = threadIdx.x; i < 1 << bits; i += THREADS) {
            keys[i] = -1, holder[i] = kNobody, owner[i] = kNobody;
        }
        __syncthreads();
        int32_t page[PER];        // what the request holds after
        int held_at[PER], rank[PER], owned_at[PER];
#pragma unroll
        for (int i = 0; i < PER; ++i) {
            const int r = r0 + i;
            page[i] = -1, held_at[i] = owned_at[i] = -1, rank[i] = 0;
            if (i < per && r < R) {
                const int64_t s = source[r];
                if (b < pages_of(after[r], shift)) {
                    page[i] = a.block_table[s * a.ld_table + b];
                    if (page[i] >= 0) {
                        // Who keeps the page: those that hold it in full, else one that had it, else the first.
                        const bool part = static_cast<int64_t>(after[r]) < static_cast<int64_t>(b + 1) << shift;
                        rank[i] = !part ? 0 : s == r ? 1 + r : 1 + R + r;
                        held_at[i] = place_of(keys, bits, page[i]);
                        atomicMin(&holder[held_at[i]], rank[i]);
                    }
                }
                if (b < pages_of(length[r], shift)) {
                    const int32_t had = a.block_table[r * a.ld_table + b];
                    if (had >= 0) {
                        owned_at[i] = place_of(keys, bits, had);
                        atomicMin(&owner[owned_at[i]], r);
                    }
                }
            }
        }
        __syncthreads();
        bool gone[PER]; // the page is nobody's any more, and the request was the first to have it
        int mine = 0;
#pragma unroll
        for (int i = 0; i < PER; ++i) {
            gone[i] = owned_at[i] >= 0 && holder[owned_at[i]] == kNobody && owner[owned_at[i]] == r0 + i;
            mine += gone[i];
        }
        int total = 0;
        int place = sum_before<THREADS>(mine, waves, &total); // its barriers keep the next column's clearing behind these reads
        if constexpr (APPLY) {
#pragma unroll
            for (int i = 0; i < PER; ++i) {
                const int r = r0 + i;
                if (gone[i]) {
                    a.free_pages[(tail + freed_before + freed_here + place) % Q] = keys[owned_at[i]];
                    ++place;
                }
                if (i < per && r < R && b < pages_of(after[r], shift)) {
                    int32_t id = page[i];
                    if (rank[i] != 0 && fresh_at[i] >= 0) {
                        id = a.free_pages[(head + fresh_at[i]) % Q];
                        int32_t *copy = a.copies + 3 * static_cast<int64_t>(fresh_at[i]);
                        copy[0] = page[i], copy[1] = id, copy[2] = after[r] & (page_tokens - 1);
                    }
                    a.table_out[r * a.ld_out + b] = id;
                }
            }
            __syncthreads(); // keys were read
        } else {
#pragma unroll
            for (int i = 0; i < PER; ++i) {
                const int r = r0 + i;
                if (i < per && r < R && (after[r] & (page_tokens - 1)) != 0 && b == after[r] >> shift) {
                    ws.fresh[r] = held_at[i] >= 0 && holder[held_at[i]] != rank[i];
                }
            }
            __syncthreads();
        }
        freed_here += total;
    }
    if (!APPLY && threadIdx.x == 0) {
        ws.chunks[blockIdx.x] = freed_here;
    }
}

template <int THREADS, int PER> hipError_t launch_fork(PageForkArgs a, int chunks, hipStream_t stream) {
    a.hash_bits = 2;
    while ((int64_t(1) << a.hash_bits) < 2 * a.requests_count) {
        ++a.hash_bits;
    }
    const size_t lds = 4 * (3 * static_cast<size_t>(a.requests_count) + (size_t(3) << a.hash_bits));
    const dim3 grid(static_cast<unsigned>(std::min<int64_t>(a.width, chunks)));
    if (lds > 64 * 1024) { // only then does a launch need the limit raised
        for (const void *f : {reinterpret_cast<const void *>(&fork_kernel<THREADS, PER, false>), reinterpret_cast<const void *>(&fork_kernel<THREADS, PER, true>)}) {
            const hipError_t e = hipFuncSetAttribute(f, hipFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(lds));
            if (e != hipSuccess) {
                return e;
            }
        }
    }
    hipLaunchKernelGGL((fork_kernel<THREADS, PER, false>), grid, dim3(THREADS), lds, stream, a);
    const hipError_t e = hipGetLastError();
    if (e != hipSuccess) {
        return e;
    }
    hipLaunchKernelGGL((fork_kernel<THREADS, PER, true>), grid, dim3(THREADS), lds, stream, a);
    return hipGetLastError();
}

// ---- compaction ----

struct CompactWorkspace {
    int32_t *sums;   // [4]: pages in use, below the limit
    uint32_t *used;  // [words]: a bit per page
    int32_t *before; // [words]: pages in use before the word's
};

__host__ __device__ __forceinline__ CompactWorkspace carve_compact(void *p, int64_t pages) {
    const int64_t words = (pages + 31) / 32;
    int32_t *b = static_cast<int32_t *>(p);
    return {b, reinterpret_cast<uint32_t *>(b + 4), b + 4 + words};
}

__global__ void __launch_bounds__(256) compact_clear_kernel(PageCompactArgs a) {
    const CompactWorkspace ws = carve_compact(a.workspace, a.pages);
    const int64_t words = (a.pages + 31) / 32;
    for (int64_t i = static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x; i < words; i += static_cast<int64_t>(gridDim.x) * 256) {
        ws.used[i] = 0;
    }
}

__device__ __forceinline__ int64_t held_by(const PageCompactArgs &a, int64_t r) {
    const int64_t n = min(max(static_cast<int64_t>(a.lengths[r]), int64_t(0)), a.width << a.page_shift);
    return (n + (int64_t(1) << a.page_shift) - 1) >> a.page_shift;
}

__global__ void __launch_bounds__(256) compact_mark_kernel(PageCompactArgs a) {
    const CompactWorkspace ws = carve_compact(a.workspace, a.pages);
    for (int64_t r = blockIdx.x; r < a.requests_count; r += gridDim.x) {
        const int64_t held = held_by(a, r);
        for (int64_t b = threadIdx.x + 256 * static_cast<int64_t>(blockIdx.y); b < held; b += 256 * static_cast<int64_t>(gridDim.y)) {
            const int32_t page = a.block_table[r * a.ld_table + b];
            if (page >= 0 && page < a.pages) {
                atomicOr(&ws.used[page >> 5], 1u << (page & 31));
            }
        }
    }
}

constexpr int kCountedWords = 8 * 1024;    // a bit per page, in LDS
constexpr int kCountedEntries = 48 * 1024; // of the table, at least 64 a request

// The sums of the words' bits, in one workgroup. MARK: after the bits are set, in LDS, which takes the place of the two launches before.
template <bool MARK> __global__ void __launch_bounds__(1024) compact_sum_kernel(PageCompactArgs a) {
    extern __shared__ int32_t lds[];
    __shared__ int32_t waves[16];
    const CompactWorkspace ws = carve_compact(a.workspace, a.pages);
    const int words = static_cast<int>((a.pages + 31) / 32), limit = static_cast<int>(a.limit);
    uint32_t *marks = reinterpret_cast<uint32_t *>(lds), *used = MARK ? marks : ws.used;
    if constexpr (MARK) {
        constexpr int kRows = 8; // of a wave at once
        for (int i = threadIdx.x; i < words; i += 1024) {
            marks[i] = 0;
        }
        __syncthreads();
        const int lane = threadIdx.x & 63;
        for (int64_t r0 = kRows * (threadIdx.x >> 6); r0 < a.requests_count; r0 += 16 * kRows) {
            int held[kRows], most = 0;
#pragma unroll
            for (int i = 0; i < kRows; ++i) {
                held[i] = r0 + i < a.requests_count ? static_cast<int>(held_by(a, r0 + i)) : 0;
                most = max(most, held[i]);
            }
            for (int b = lane; b < most; b += 64) {
                int32_t page[kRows];
#pragma unroll
                for (int i = 0; i < kRows; ++i) {
                    page[i] = b < held[i] ? a.block_table[(r0 + i) * a.ld_table + b] : -1;
                }
#pragma unroll
                for (int i = 0; i < kRows; ++i) {
                    if (page[i] >= 0 && page[i] < a.pages) {
                        atomicOr(&marks[page[i] >> 5], 1u << (page[i] & 31));
                    }
                }
            }
        }
        __syncthreads();
    }
    int carried = 0;
    for (int from = 0; from < words; from += 4 * 1024) { // four words a thread
        const int w0 = from + 4 * static_cast<int>(threadIdx.x);
        uint32_t word[4];
        int own = 0;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            word[i] = w0 + i < words ? used[w0 + i] : 0;
            own += __popc(word[i]);
        }
        int total = 0;
        int before = carried + sum_before<1024>(own, waves, &total);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            if (w0 + i < words) {
                ws.before[w0 + i] = before;
                if (MARK) {
                    ws.used[w0 + i] = word[i];
                }
                if (w0 + i == limit >> 5) {
                    ws.sums[1] = before + __popc(word[i] & ((1u << (limit & 31)) - 1));
                }
            }
            before += __popc(word[i]);
        }
        carried += total;
    }
    if (threadIdx.x == 0) {
        ws.sums[0] = carried;
        if (limit >> 5 >= words) {
            ws.sums[1] = carried;
        }
    }
}

// The i-th page below the limit that is not in use.
__device__ __forceinline__ int32_t free_page(const CompactWorkspace &ws, int limit, int i) {
    int lo = 0, hi = (limit + 31) / 32 - 1; // the last word that has at most i free pages before it
    while (lo < hi) {
        const int mid = (lo + hi + 1) >> 1;
        if (32 * mid - ws.before[mid] <= i) {
            lo = mid;
        } else {
            hi = mid - 1;
        }
    }
    uint32_t word = ~ws.used[lo];
    for (int skip = i - (32 * lo - ws.before[lo]); skip > 0; --skip) {
        word &= word - 1;
    }
    return 32 * lo + (__ffs(static_cast<int>(word)) - 1);
}

// Workgroups [0, id_blocks): the ring and the copies, a thread per page; those behind: the table, a request at a time.
__global__ void __launch_bounds__(256) compact_apply_kernel(PageCompactArgs a, int id_blocks) {
    const CompactWorkspace ws = carve_compact(a.workspace, a.pages);
    const int used = ws.sums[0], below = ws.sums[1], limit = static_cast<int>(a.limit), moves = used - below;
    const bool refused = used > limit || limit - used > a.ring_size;
    if (static_cast<int>(blockIdx.x) < id_blocks) {
        const uint64_t head = static_cast<uint64_t>(a.queue_in[0]), Q = static_cast<uint64_t>(a.ring_size);
        const int64_t step = static_cast<int64_t>(id_blocks) * 256, from = static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x;
        for (int64_t id = from; id < a.pages && !refused; id += step) {
            const uint32_t word = ws.used[id >> 5];
            const int used_before = ws.before[id >> 5] + __popc(word & ((1u << (id & 31)) - 1));
            const bool is_used = (word >> (id & 31) & 1) != 0;
            if (id >= limit) {
                if (is_used) {
                    a.copies[3 * static_cast<int64_t>(used_before - below)] = static_cast<int32_t>(id);
                }
            } else if (!is_used) {
                const int i = static_cast<int>(id) - used_before;
                if (i < moves) {
                    a.copies[3 * static_cast<int64_t>(i) + 1] = static_cast<int32_t>(id);
                    a.copies[3 * static_cast<int64_t>(i) + 2] = 1 << a.page_shift;
                } else {
                    a.free_pages[(head + (i - moves)) % Q] = static_cast<int32_t>(id);
                }
            }
        }
        for (int64_t i = from + (refused ? 0 : 3 * static_cast<int64_t>(moves)); i < 3 * a.most_copies; i += step) {
            a.copies[i] = -1;
        }
        if (from == 0) { // read by this thread alone once it is written: the others read the head before or never
            const int64_t tail = a.queue_in[1];
            a.queue_out[0] = static_cast<int64_t>(head);
            a.queue_out[1] = refused ? tail : static_cast<int64_t>(head) + limit - used;
            a.queue_out[2] = refused;
            a.queue_out[3] = refused ? 0 : moves;
        }
        return;
    }
    for (int64_t r = blockIdx.x - id_blocks; r < a.requests_count; r += gridDim.x - id_blocks) {
        const int64_t held = held_by(a, r);
        for (int64_t b = threadIdx.x; b < held; b += 256) {
            int32_t page = a.block_table[r * a.ld_table + b];
            if (!refused && page >= limit && page < a.pages) {
                page = free_page(ws, limit, ws.before[page >> 5] + __popc(ws.used[page >> 5] & ((1u << (page & 31)) - 1)) - below);
            }
            a.table_out[r * a.ld_out + b] = page;
        }
    }
}

// ---- copies ----

constexpr int kCopyTokens = 16; // of a wave's piece: 4 KB at 128 elements
constexpr int kCopyAhead = 4;   // 16-byte loads of a lane

typedef uint32_t u32x4_t __attribute__((ext_vector_type(4)));

// Bound by memory: 373 us for the large cache of the compaction (4.9 TB/s read and written), 38 for 32 requests' pages of 16; 41 with one load of a lane at a time.
// A wave per piece: 16 tokens of one page and head; blockIdx.y: layer, and keys or values. The lanes read the entries of a wave's next 64 pieces at once, so
// that lists that are mostly empty are soon passed over.
__global__ void __launch_bounds__(256) copy_pages_kernel(CopyPagesArgs a) {
    const int lane = threadIdx.x & 63;
    const int layer = blockIdx.y >> 1;
    const uint16_t *from = (blockIdx.y & 1) ? a.from_v[layer] : a.from_k[layer];
    uint16_t *to = (blockIdx.y & 1) ? a.to_v[layer] : a.to_k[layer];
    const int per_page = a.kv_heads << (a.page_shift - 4), row_pieces = a.head_dim / 8, per_step = max(64 / row_pieces, 1);
    const int in_step = lane / row_pieces, first_piece = lane - in_step * row_pieces, first_token = in_step < per_step ? in_step : kCopyTokens;
    const int64_t pieces = a.count * per_page, step = static_cast<int64_t>(gridDim.x) * 4;
    for (int64_t p0 = static_cast<int64_t>(blockIdx.x) * 4 + (threadIdx.x >> 6); p0 < pieces; p0 += 64 * step) {
        const int64_t p = p0 + lane * step;
        int32_t source = -1, target = -1, head = 0, t0 = 0, count = 0;
        if (p < pieces) {
            const int64_t entry = p / per_page;
            const int in_page = static_cast<int>(p - entry * per_page);
            source = a.copies[3 * entry], target = a.copies[3 * entry + 1];
            head = in_page % a.kv_heads, t0 = in_page / a.kv_heads * kCopyTokens;
            count = min(kCopyTokens, min(a.copies[3 * entry + 2], 1 << a.page_shift) - t0);
        }
        const bool some = count > 0 && source >= 0 && target >= 0 && source < a.from_pages && target < a.to_pages;
        for (uint64_t left = __ballot(some); left != 0; left &= left - 1) {
            const int i = static_cast<int>(__builtin_ctzll(left));
            const int64_t in_from = __builtin_amdgcn_readlane(source, i) * a.from_page, in_to = __builtin_amdgcn_readlane(target, i) * a.to_page;
            const int at_head = __builtin_amdgcn_readlane(head, i), at_token = __builtin_amdgcn_readlane(t0, i);
            const uint16_t *f = from + in_from + at_head * a.from_head + at_token * a.from_token;
            uint16_t *t = to + in_to + at_head * a.to_head + at_token * a.to_token;
            const int tokens = __builtin_amdgcn_readlane(count, i);
            for (int at = 8 * first_piece; at < a.head_dim; at += 512) { // once, but for heads of more than 512
                for (int token = first_token; token < tokens; token += kCopyAhead * per_step) {
                    u32x4_t v[kCopyAhead]; // all loads before the first store, which may be to their place, for what the compiler knows
#pragma unroll
                    for (int n = 0; n < kCopyAhead; ++n) {
                        v[n] = *reinterpret_cast<const u32x4_t *>(f + min(token + n * per_step, tokens - 1) * a.from_token + at);
                    }
#pragma unroll
                    for (int n = 0; n < kCopyAhead; ++n) {
                        if (token + n * per_step < tokens) {
                            *reinterpret_cast<u32x4_t *>(t + (token + n * per_step) * a.to_token + at) = v[n];
                        }
                    }
                }
            }
        }
    }
}

} // namespace

size_t page_fork_workspace(int64_t requests) { return 16 + 4 * static_cast<size_t>(kMaxChunks + 2 * requests); }

hipError_t launch_page_fork(const PageForkArgs &a, hipStream_t stream) {
    // A thread per request where a workgroup has them: 256 requests 11.3 us with 256 threads and 12.7 with 1024, 512 of the mixed case's 15 with 1024 and
    // 18 with four to a thread; up to 64, one wave 10.9 and four 11.1.
    if (a.requests_count <= 64) {
        return launch_fork<64, 1>(a, kMaxChunks, stream);
    }
    if (a.requests_count <= 256) {
        return launch_fork<256, 1>(a, 512, stream);
    }
    return a.requests_count <= 1024 ? launch_fork<1024, 1>(a, 512, stream) : launch_fork<1024, kMaxRequests / 1024>(a, 256, stream);
}

size_t page_compact_workspace(int64_t pages) { return 4 * static_cast<size_t>(4 + 2 * ((pages + 31) / 32)); }

hipError_t launch_page_compact(const PageCompactArgs &a, hipStream_t stream) {
    const int64_t cus = device_topology().cus, words = (a.pages + 31) / 32;
    const unsigned clear = static_cast<unsigned>(std::min<int64_t>(cus, (words + 255) / 256));
    const unsigned requests = static_cast<unsigned>(std::min<int64_t>(a.requests_count, 4 * cus));
    const unsigned wide = static_cast<unsigned>(std::max<int64_t>(1, std::min<int64_t>((a.width + 255) / 256, 4 * cus / requests)));
    const unsigned ids = static_cast<unsigned>(std::min<int64_t>(4 * cus, (a.pages + 255) / 256));
    // One workgroup marks a small table sooner than two more launches take: 4096 entries 10.1 us instead of 14.6, 24 576 13.7 instead of 18.2; 65 536 entries
    // of 512 requests 20.1 either way, of 1024 requests 23.7 instead of 20.5, and 131 072 32 instead of 23.
    if (words <= kCountedWords && a.requests_count * std::max<int64_t>(a.width, 64) <= kCountedEntries) {
        hipLaunchKernelGGL(compact_sum_kernel<true>, dim3(1), dim3(1024), 4 * static_cast<size_t>(words), stream, a);
    } else {
        hipLaunchKernelGGL(compact_clear_kernel, dim3(clear), dim3(256), 0, stream, a);
        hipLaunchKernelGGL(compact_mark_kernel, dim3(requests, wide), dim3(256), 0, stream, a);
        hipLaunchKernelGGL(compact_sum_kernel<false>, dim3(1), dim3(1024), 0, stream, a);
    }
    hipLaunchKernelGGL(compact_apply_kernel, dim3(ids + requests), dim3(256), 0, stream, a, static_cast<int>(ids));
    return hipGetLastError();
}

hipError_t launch_copy_pages(const CopyPagesArgs &a, hipStream_t stream) {
    const int64_t pieces = a.count * (static_cast<int64_t>(a.kv_heads) << (a.page_shift - 4));
    const int64_t most = std::max<int64_t>(1, 8 * static_cast<int64_t>(device_topology().cus) / (2 * a.layers));
    hipLaunchKernelGGL(copy_pages_kernel, dim3(static_cast<unsigned>(std::min((pieces + 3) / 4, most)), static_cast<unsigned>(2 * a.layers)), dim3(256), 0, stream, a);
    return hipGetLastError();
}

} // namespace hm
