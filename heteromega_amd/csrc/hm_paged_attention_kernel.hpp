// One-token attention over a paged cache: the kernels (hm_paged_attention.hip has the mathematics and the launch rules).
#pragma once

#include "hm_device.hpp"
#include "hm_paged_attention.hpp"

namespace hm {
namespace {

constexpr int kThreads = 64 * kAttentionWaves;
constexpr int kWaveKeys = 32;
constexpr int kLaneRows = 4;
constexpr int kStream = 2; // cache policy of the keys and values, read once: non-temporal

typedef uint32_t u32x4_t __attribute__((ext_vector_type(4)));

// One row's request and keys [first, end).
struct Keys {
    int32_t request, first, end;
    bool bad; // request or position outside the table
};

__device__ __forceinline__ Keys keys_of(const PagedAttentionArgs &a, int64_t t) {
    Keys k;
    k.request = a.requests != nullptr ? a.requests[t] : static_cast<int32_t>(t);
    const int32_t pos = a.positions[t];
    k.bad = k.request >= a.requests_count || pos < -1 || pos >= (a.width << a.page_shift);
    k.end = k.bad ? 0 : pos + 1;
    k.first = a.window > 0 && a.window < k.end ? k.end - static_cast<int32_t>(a.window) : 0;
    return k;
}

// A prompt block's rows lie within an aligned block of `rows` rows whose first and last are of one request, and its last row sees at most
// `limit` keys (kPromptShare): a chunk of a long request next to a few others is better split over its keys. rows 0: there are none.
struct Prompts {
    int rows, limit;
};

// The keys that the last row of block b sees if its first and last row are of one request, else -1.
__device__ __forceinline__ int prompt_keys(const PagedAttentionArgs &a, int rows, int64_t b) {
    const int64_t t0 = b * rows, t1 = t0 + rows - 1;
    if (t1 >= a.rows) {
        return -1;
    }
    const int32_t r0 = a.requests[t0], r1 = a.requests[t1], pos = a.positions[t1];
    return r0 >= 0 && r0 == r1 && pos >= 0 && pos < (a.width << a.page_shift) ? pos + 1 : -1;
}

__device__ __forceinline__ bool of_prompt(const PagedAttentionArgs &a, const Prompts &p, int64_t b) {
    const int keys = prompt_keys(a, p.rows, b);
    return keys >= 0 && keys <= p.limit;
}

// Summed up by each wave for itself.
__device__ __forceinline__ Prompts prompts_of(const PagedAttentionArgs &a, int rows, int slots) {
    if (rows == 0) {
        return {0, 0};
    }
    const int blocks = static_cast<int>(a.rows / rows);
    int64_t sum = 0;
#pragma unroll 4
    for (int b = threadIdx.x & 63; b < blocks; b += 64) {
        sum += max(prompt_keys(a, rows, b), 0);
    }
#pragma unroll
    for (int off = 32; off > 0; off >>= 1) {
        sum += __shfl_xor(sum, off);
    }
    return {rows, uniform(static_cast<int>(min((kPromptShare * sum - 1) / slots, static_cast<int64_t>(INT32_MAX))))};
}

// The rows of a unit, `count` from this one on: keys [first, end) are seen by some of them, [all_first, all_end) by all; the tiles begin
// at start.
struct Row {
    int32_t request, first, end, all_first, all_end, start, tiles, count;
    bool bad;
};

// Row t with those that share units with it. Rows that belong to another row's units or to a prompt block have no tiles, like rows of no
// request. With `rows` > 1, a unit's rows lie within an aligned block of so many, follow each other, are of one request and none is bad.
template <bool GROUPED> __device__ __forceinline__ Row row_of(const PagedAttentionArgs &a, int64_t t, int tile_keys, int rows, const Prompts &prompts) {
    const Keys k = keys_of(a, t);
    Row r{k.request, k.first, k.end, k.first, k.end, 0, 0, 1, k.bad};
    if (k.request < 0) {
        return r;
    }
    if constexpr (GROUPED) {
        if (prompts.rows != 0 && of_prompt(a, prompts, t / prompts.rows)) {
            return r;
        }
        if (t % rows != 0 && !k.bad) {
            const Keys before = keys_of(a, t - 1);
            if (before.request == k.request && !before.bad) {
                return r;
            }
        }
        const int64_t stop = min(a.rows, t - t % rows + rows);
        for (int64_t u = t + 1; u < stop && !k.bad; ++u) {
            const Keys next = keys_of(a, u);
            if (next.request != k.request || next.bad) {
                break;
            }
            r.first = min(r.first, next.first), r.end = max(r.end, next.end);
            r.all_first = max(r.all_first, next.first), r.all_end = min(r.all_end, next.end);
            ++r.count;
        }
    }
    r.start = r.first & ~15;
    r.tiles = max(1, (r.end - r.start + tile_keys - 1) / tile_keys); // a row without keys still has an output to write
    return r;
}

__device__ __forceinline__ int64_t uniform64(int64_t v) {
    const uint32_t lo = __builtin_amdgcn_readfirstlane(static_cast<uint32_t>(v));
    const uint32_t hi = __builtin_amdgcn_readfirstlane(static_cast<uint32_t>(static_cast<uint64_t>(v) >> 32));
    return static_cast<int64_t>((static_cast<uint64_t>(hi) << 32) | lo);
}

// A row that all lanes hold, in scalar registers: page addresses must be known to be uniform, or each load becomes a loop over
// the lanes' addresses (which took 374 us instead of 358 at 64 rows of 8192 keys).
__device__ __forceinline__ Row uniform_row(const Row &r) {
    return Row{uniform(r.request), uniform(r.first), uniform(r.end),   uniform(r.all_first), uniform(r.all_end),
               uniform(r.start),   uniform(r.tiles), uniform(r.count), uniform(r.bad) != 0};
}

// The row that a lane holds, in scalar registers.
__device__ __forceinline__ Row row_of_lane(const Row &r, int lane) {
    const auto of = [&](int v) { return __builtin_amdgcn_readlane(v, lane); };
    return Row{of(r.request), of(r.first), of(r.end), of(r.all_first), of(r.all_end), of(r.start), of(r.tiles), of(r.count), of(r.bad) != 0};
}

__device__ __forceinline__ float exp2_fast(float x) { return __builtin_amdgcn_exp2f(x); }

template <class T> __device__ __forceinline__ void store4(uint16_t *p, float4_t v) {
    uint2 o;
    o.x = static_cast<uint32_t>(T::from_float(v[0])) | (static_cast<uint32_t>(T::from_float(v[1])) << 16);
    o.y = static_cast<uint32_t>(T::from_float(v[2])) | (static_cast<uint32_t>(T::from_float(v[3])) << 16);
    *reinterpret_cast<uint2 *>(p) = o;
}

typedef float float2_t __attribute__((ext_vector_type(2)));

// Pairs of T's weights, and the power of two that the largest weight has: fp16 loses weights below 2^-25, of which a long row can have
// enough to matter next to a weight of 1; from 2^15 down to its subnormals it has 2^40 of range. kBelow keeps hi below p by more than its
// rounding, so that lo is positive as well: an infinite value then gives an infinite output, as p alone would, where a lo of zero or below
// would make it NaN.
template <class T> struct Split;
template <> struct Split<F16> {
    typedef _Float16 elem_t;
    typedef elem_t pair_t __attribute__((ext_vector_type(2)));
    static constexpr float kTop = 15.0f;
    static constexpr float kBelow = 1.0f - 0x1p-11f;
    static constexpr uint32_t kExponent = 0x7C00u; // all bits set: an infinity or NaN
    // Rounded towards zero by an instruction of its own. A plain conversion of a product is made twice by the compiler, once together with
    // the product and once after it, with roundings that differ now and then: then lo does not belong to hi.
    static __device__ __forceinline__ pair_t upper(float2_t p) { return __builtin_bit_cast(pair_t, __builtin_amdgcn_cvt_pkrtz(p[0] * kBelow, p[1] * kBelow)); }
};
template <> struct Split<BF16> {
    typedef __bf16 elem_t;
    typedef elem_t pair_t __attribute__((ext_vector_type(2)));
    static constexpr float kTop = 0.0f;
    static constexpr float kBelow = 1.0f - 0x1p-8f;
    static constexpr uint32_t kExponent = 0x7F80u;
    static __device__ __forceinline__ pair_t upper(float2_t p) { return __builtin_convertvector(p * kBelow, pair_t); }
};

// Two weights, each as hi + lo.
template <class T> __device__ __forceinline__ void split(float2_t p, uint32_t &hi, uint32_t &lo) {
    typedef typename Split<T>::pair_t pair_t;
    const pair_t upper = Split<T>::upper(p);
    hi = __builtin_bit_cast(uint32_t, upper);
    lo = __builtin_bit_cast(uint32_t, __builtin_convertvector(p - __builtin_convertvector(upper, float2_t), pair_t));
}

template <class T, int D> struct Shape {
    static constexpr int kSteps = D / 32;         // K steps of the first product, and 16-byte pieces of V per lane and sub-tile
    static constexpr int kDTiles = D / 16;        // row tiles of O^T
    static constexpr int kRowBytes = 2 * D + 32;  // a row of V in LDS: 32 bytes of padding turn the banks of successive rows
    static constexpr int kRegion = kWaveKeys * kRowBytes;
    static constexpr int kORow = D + 4;           // floats of a column of O in LDS
    static_assert(16 * kORow * 4 <= kRegion, "O takes the place of V");
};

// Piece i * 64 + lane of a sub-tile's 16 rows of D / 8 pieces: its key, its offset in memory and its place in LDS. Where rows are a
// power of two of pieces, piece i lies a constant number of rows behind piece 0.
template <int D> struct Pieces {
    static constexpr int kPerRow = D / 8;
    static constexpr bool kEven = 64 % kPerRow == 0;
    static constexpr int kKept = kEven ? 1 : D / 32;
    int keys[kKept];
    uint32_t offsets[kKept], places[kKept];
    uint32_t step;

    __device__ __forceinline__ Pieces(int lane, uint32_t row_bytes) : step(64 / kPerRow * row_bytes) {
#pragma unroll
        for (int i = 0; i < kKept; ++i) {
            const int piece = i * 64 + lane;
            keys[i] = piece / kPerRow;
            const int c = piece - keys[i] * kPerRow;
            offsets[i] = keys[i] * row_bytes + c * 16;
            places[i] = keys[i] * (2 * D + 32) + c * 16;
        }
    }
    __device__ __forceinline__ int key(int i) const { return kEven ? keys[0] + i * (64 / kPerRow) : keys[i % kKept]; }
    __device__ __forceinline__ uint32_t offset(int i) const { return kEven ? offsets[0] + i * step : offsets[i % kKept]; }
    __device__ __forceinline__ uint32_t lds_offset() const { return kEven ? places[0] : 0; }
    __device__ __forceinline__ uint32_t lds_step(int i) const { return kEven ? i * (64 / kPerRow) * (2 * D + 32) : places[i % kKept]; }
};

// The same, once they are counted, in a launch before.
__device__ __forceinline__ Prompts prompts_known(const PagedAttentionArgs &a, const AttentionPlan &plan) {
    return plan.counted && plan.prompt_rows != 0 ? Prompts{plan.prompt_rows, carve(a.workspace, plan.runs, plan.cols).counts[kChunks]}
                                                 : prompts_of(a, plan.prompt_rows, plan.prompt_slots);
}

// The tiles of each chunk of rows, a workgroup per chunk, and the limit of prompt blocks.
template <bool GROUPED> __global__ void __launch_bounds__(kThreads) count_kernel(PagedAttentionArgs a, AttentionPlan plan) {
    __shared__ int sums[kAttentionWaves];
    Prompts prompts{0, 0};
    if constexpr (GROUPED) {
        prompts = prompts_of(a, plan.prompt_rows, plan.prompt_slots);
    }
    const int rows = static_cast<int>(a.rows), per = (rows + kChunks - 1) / kChunks;
    const int t0 = min(static_cast<int>(blockIdx.x) * per, rows), t1 = min(t0 + per, rows);
    int own = 0;
    for (int i = t0 + threadIdx.x; i < t1; i += kThreads) {
        own += row_of<GROUPED>(a, i, plan.team * kWaveKeys, plan.rows, prompts).tiles;
    }
#pragma unroll
    for (int off = 32; off > 0; off >>= 1) {
        own += __shfl_xor(own, off);
    }
    if ((threadIdx.x & 63) == 0) {
        sums[threadIdx.x >> 6] = own;
    }
    __syncthreads();
    if (threadIdx.x == 0) {
        for (int i = 1; i < kAttentionWaves; ++i) {
            own += sums[i];
        }
        int32_t *counts = carve(a.workspace, plan.runs, plan.cols).counts;
        counts[blockIdx.x] = own;
        if (blockIdx.x == 0) {
            counts[kChunks] = prompts.limit;
        }
    }
}

// TEAM waves of a workgroup (4 or 1) share a run of tiles of TEAM * 32 keys; a workgroup has 4 / TEAM runs. CT: tiles of 16 columns that
// a unit has at most. GROUPED: units of several rows.
template <class T, int D, int TEAM, int CT, bool GROUPED>
__global__ void __launch_bounds__(kThreads, D <= 128 ? 2 : 1) paged_attention_kernel(PagedAttentionArgs a, AttentionPlan plan) {
    using S = Shape<T, D>;
    constexpr int kRuns = kAttentionWaves / TEAM, kTileKeys = TEAM * kWaveKeys;
    __shared__ __attribute__((aligned(16))) uint8_t lds[kAttentionWaves * S::kRegion];
    __shared__ float2 wave_stats[kAttentionWaves][16];
    __shared__ int scan[kAttentionWaves];
    __shared__ int found[kRuns][2];

    const int lane = threadIdx.x & 63, wave = uniform(threadIdx.x >> 6);
    const int member = TEAM == 1 ? 0 : wave; // of its run's waves
    const int col = lane & 15, quad = lane >> 4;
    const int units = plan.units;
    const int w = blockIdx.x * kRuns + (TEAM == 1 ? wave : 0), rows = static_cast<int>(a.rows);

    Prompts prompts{0, 0};
    if constexpr (GROUPED) {
        prompts = prompts_known(a, plan);
    }

    // ---- this run's tiles, [x, x_end) ----
    int x, x_end;
    Runs runs{};
    int t = 0, base = 0; // the row that x lies in, and the row's first tile
    Row r{};
    if (rows <= 64 * kLaneRows) { // each wave finds its place by itself, kLaneRows rows a lane or one
        const int per = rows <= 64 ? 1 : kLaneRows;
        Row mine[kLaneRows];
        int own = 0;
#pragma unroll
        for (int i = 0; i < kLaneRows; ++i) {
            const bool some = i < per && lane * per + i < rows;
            mine[i] = some ? row_of<GROUPED>(a, lane * per + i, kTileKeys, plan.rows, prompts) : Row{};
            own += mine[i].tiles;
        }
        int upto = own;
#pragma unroll
        for (int off = 1; off < 64; off <<= 1) {
            const int v = __shfl_up(upto, off);
            upto += lane >= off ? v : 0;
        }
        runs = Runs::deal(__builtin_amdgcn_readlane(upto, 63) * units, plan.runs);
        x = runs.begin(w);
        x_end = w < plan.runs ? runs.begin(w + 1) : x;
        if (x < x_end) {
            const int from = __builtin_ctzll(__ballot(x < upto * units));
            base = (__builtin_amdgcn_readlane(upto, from) - __builtin_amdgcn_readlane(own, from)) * units;
            t = from * per;
#pragma unroll
            for (int i = 0; i < kLaneRows; ++i) {
                if (i < per) {
                    r = row_of_lane(mine[i], from);
                    if (x < base + r.tiles * units) {
                        break;
                    }
                    base += r.tiles * units;
                    ++t;
                }
            }
        }
    } else {
        const int per = (rows + kChunks - 1) / kChunks;
        const int t0 = min(static_cast<int>(threadIdx.x) * per, rows), t1 = min(t0 + per, rows);
        int own = 0;
        if (plan.counted) {
            own = carve(a.workspace, plan.runs, plan.cols).counts[threadIdx.x];
        } else {
            for (int i = t0; i < t1; ++i) {
                own += row_of<GROUPED>(a, i, kTileKeys, plan.rows, prompts).tiles;
            }
        }
        int upto = own;
#pragma unroll
        for (int off = 1; off < 64; off <<= 1) {
            const int v = __shfl_up(upto, off);
            upto += lane >= off ? v : 0;
        }
        if (lane == 63) {
            scan[wave] = upto;
        }
        __syncthreads();
        int before = upto - own, total = 0;
#pragma unroll
        for (int i = 0; i < kAttentionWaves; ++i) {
            before += i < wave ? scan[i] : 0;
            total += scan[i];
        }
        runs = Runs::deal(uniform(total) * units, plan.runs);
        x = runs.begin(w);
        x_end = w < plan.runs ? runs.begin(w + 1) : x;
#pragma unroll
        for (int j = 0; j < kRuns; ++j) {
            const int xj = runs.begin(blockIdx.x * kRuns + j);
            if (before * units <= xj && xj < (before + own) * units) {
                found[j][0] = t0;
                found[j][1] = before * units;
            }
        }
        __syncthreads();
        if (x < x_end) { // the chunk's rows, 64 at a time
            base = uniform(found[TEAM == 1 ? wave : 0][1]);
            for (int from = uniform(found[TEAM == 1 ? wave : 0][0]); from < rows; from += 64) {
                const Row mine = from + lane < rows ? row_of<GROUPED>(a, from + lane, kTileKeys, plan.rows, prompts) : Row{};
                int to = mine.tiles;
#pragma unroll
                for (int off = 1; off < 64; off <<= 1) {
                    const int v = __shfl_up(to, off);
                    to += lane >= off ? v : 0;
                }
                const uint64_t behind = __ballot(x < base + to * units);
                if (behind != 0) {
                    const int at = __builtin_ctzll(behind);
                    r = row_of_lane(mine, at);
                    base += (__builtin_amdgcn_readlane(to, at) - r.tiles) * units;
                    t = from + at;
                    break;
                }
                base += __builtin_amdgcn_readlane(to, 63) * units;
            }
        }
    }
    AttentionDescriptor begun{0, 0, 0, 0};

    // ---- constants of the lane ----
    const uint32_t row_bytes = static_cast<uint32_t>(a.token_stride) * 2;
    // Pieces of 16 bytes of a sub-tile's rows as the lanes load them, whole rows by neighbouring lanes.
    const Pieces<D> pieces(lane, row_bytes);
    const uint32_t to_lds = wave * S::kRegion + pieces.lds_offset();
    const uint32_t k_lds = wave * S::kRegion + col * S::kRowBytes + quad * 16;
    const uint32_t v_lds = wave * S::kRegion + (4 * quad + (col >> 2)) * S::kRowBytes + (col & 3) * 8;
    const float c_scale = a.scale * 1.4426950408889634f;

    while (x < x_end) {
        while (x >= base + r.tiles * units) { // on to the next row with tiles, 64 at a time
            base = uniform(base + r.tiles * units);
            int from = t + 1;
            uint64_t some = 0;
            for (; from < rows; from += 64) {
                some = __ballot(from + lane < rows && row_of<GROUPED>(a, min(from + lane, rows - 1), kTileKeys, plan.rows, prompts).tiles > 0);
                if (some != 0) {
                    break;
                }
            }
            t = uniform(some != 0 ? from + static_cast<int>(__builtin_ctzll(some)) : rows - 1); // a run ends before the rows do
            r = uniform_row(row_of<GROUPED>(a, t, kTileKeys, plan.rows, prompts));
        }
        const int unit = uniform(static_cast<uint32_t>(x - base) / static_cast<uint32_t>(r.tiles));
        const int tile0 = x - base - unit * r.tiles;
        const int tile1 = min(r.tiles, tile0 + (x_end - x));
        const int columns = plan.columns<GROUPED>(unit, r.count), kv_head = uniform(plan.kv_head(unit));

        u32x4_t q[CT][S::kSteps];
        int first[GROUPED ? CT : 1], end[GROUPED ? CT : 1], row_in_unit[GROUPED ? CT : 1]; // of the lane's column
#pragma unroll
        for (int c = 0; c < CT; ++c) {
            const bool live = 16 * c + col < columns;
            const Column at = plan.column<GROUPED>(unit, live ? 16 * c + col : 0);
            const uint16_t *q_row = a.q + static_cast<int64_t>(t + at.row) * a.ldq + static_cast<int64_t>(at.q_head) * D + 8 * quad;
            if constexpr (GROUPED) {
                first[c] = r.first, end[c] = r.end, row_in_unit[c] = at.row;
                if (!r.bad) {
                    const Keys k = keys_of(a, t + at.row);
                    first[c] = k.first, end[c] = k.end;
                }
            }
#pragma unroll
            for (int s = 0; s < S::kSteps; ++s) {
                q[c][s] = live ? *reinterpret_cast<const u32x4_t *>(q_row + 32 * s) : u32x4_t{0, 0, 0, 0};
            }
        }

        float4_t o[CT][S::kDTiles];
        float m[CT], l[CT];
#pragma unroll
        for (int c = 0; c < CT; ++c) {
#pragma unroll
            for (int i = 0; i < S::kDTiles; ++i) {
                o[c][i] = float4_t{0.0f, 0.0f, 0.0f, 0.0f};
            }
            m[c] = -INFINITY, l[c] = 0.0f;
        }
        bool poisoned[GROUPED ? CT : 1] = {}; // a page outside the cache among those that the column (GROUPED) or the row sees

        u32x4_t k_reg[2][S::kSteps], v_reg[2][S::kSteps];
        const int32_t *table = a.block_table + uniform64((r.bad ? 0 : r.request) * a.ld_table);
        const uint16_t *k_head = a.k + uniform64(kv_head * a.head_stride), *v_head = a.v + uniform64(kv_head * a.head_stride);
        const int64_t page_stride = uniform64(a.page_stride);
        const int shift = uniform(a.page_shift), offset_mask = (1 << shift) - 1;
        const uint32_t pages = uniform(static_cast<int>(a.pages));
        int32_t id[2];
        const auto page_ids = [&](int tile) {
#pragma unroll
            for (int s = 0; s < 2; ++s) {
                const int key = r.start + tile * kTileKeys + member * kWaveKeys + 16 * s;
                id[s] = key < r.end ? table[key >> shift] : 0;
            }
        };
        const auto request = [&](int tile) {
#pragma unroll
            for (int s = 0; s < 2; ++s) {
                const int key = r.start + tile * kTileKeys + member * kWaveKeys + 16 * s;
                const int32_t page = uniform(id[s]);
                int seen = max(0, min(16, r.end - key));
                if (static_cast<uint32_t>(page) >= pages) {
                    if constexpr (GROUPED) {
#pragma unroll
                        for (int c = 0; c < CT; ++c) {
                            poisoned[c] |= key < end[c] && key + 16 > first[c];
                        }
                    } else {
                        poisoned[0] |= seen > 0;
                    }
                    seen = 0;
                }
                // Past the row's last key the buffer ends, and its loads return zero.
                const uint32_t bytes = uniform(seen > 0 ? (seen - 1) * row_bytes + 2 * D : 0);
                const int64_t at = uniform64(seen > 0 ? page * page_stride + static_cast<int64_t>(key & offset_mask) * (row_bytes / 2) : 0);
                const __amdgpu_buffer_rsrc_t kr = buffer_rsrc(k_head + at, bytes), vr = buffer_rsrc(v_head + at, bytes);
#pragma unroll
                for (int i = 0; i < S::kSteps; ++i) {
                    k_reg[s][i] = __builtin_amdgcn_raw_buffer_load_b128(kr, pieces.offset(i), 0, GROUPED ? 0 : kStream);
                }
#pragma unroll
                for (int i = 0; i < S::kSteps; ++i) {
                    v_reg[s][i] = __builtin_amdgcn_raw_buffer_load_b128(vr, pieces.offset(i), 0, GROUPED ? 0 : kStream);
                }
            }
        };
        page_ids(tile0);
        request(tile0);
        page_ids(min(tile0 + 1, tile1 - 1));
        for (int tile = tile0; tile < tile1; ++tile) {
            const int key0 = r.start + tile * kTileKeys + member * kWaveKeys;
            if (key0 >= r.end) {
                break; // only the row's last tile has waves without keys
            }
            if (key0 < r.first) { // values before the window count as zero, whatever they are
#pragma unroll
                for (int s = 0; s < 2; ++s) {
#pragma unroll
                    for (int i = 0; i < S::kSteps; ++i) {
                        if (key0 + 16 * s + pieces.key(i) < r.first) {
                            v_reg[s][i] = u32x4_t{0, 0, 0, 0};
                        }
                    }
                }
            }
            const bool some_masked = key0 < r.all_first || key0 + kWaveKeys > r.all_end;
            // Keys that some of the unit's rows see and others do not: their weight is zero where they are not seen, but zero times an infinity or
            // NaN among the values would still show there. Then the rows go one by one.
            bool apart = false;
            if constexpr (GROUPED) {
                if (some_masked) {
#pragma unroll
                    for (int s = 0; s < 2; ++s) {
#pragma unroll
                        for (int i = 0; i < S::kSteps; ++i) {
#pragma unroll
                            for (int k = 0; k < 4; ++k) {
                                const uint32_t v = v_reg[s][i][k], e = Split<T>::kExponent;
                                apart |= (v & e) == e || (v >> 16 & e) == e;
                            }
                        }
                    }
                    apart = __any(apart);
                }
            }
            // K and then V pass through the wave's own region of LDS; a wave's LDS accesses are carried out in order.
#pragma unroll
            for (int s = 0; s < 2; ++s) {
#pragma unroll
                for (int i = 0; i < S::kSteps; ++i) {
                    *reinterpret_cast<u32x4_t *>(lds + to_lds + pieces.lds_step(i) + s * 16 * S::kRowBytes) = k_reg[s][i];
                }
            }
            float4_t score[CT][2];
#pragma unroll
            for (int c = 0; c < CT; ++c) {
                score[c][0] = score[c][1] = float4_t{0.0f, 0.0f, 0.0f, 0.0f};
            }
#pragma unroll
            for (int i = 0; i < S::kSteps; ++i) {
#pragma unroll
                for (int s = 0; s < 2; ++s) {
                    const uint4 k = *reinterpret_cast<const uint4 *>(lds + k_lds + s * 16 * S::kRowBytes + 64 * i);
#pragma unroll
                    for (int c = 0; c < CT; ++c) {
                        score[c][s] = T::mfma16(k, __builtin_bit_cast(uint4, q[c][i]), score[c][s]);
                    }
                }
            }
#pragma unroll
            for (int s = 0; s < 2; ++s) {
#pragma unroll
                for (int i = 0; i < S::kSteps; ++i) {
                    *reinterpret_cast<u32x4_t *>(lds + to_lds + pieces.lds_step(i) + s * 16 * S::kRowBytes) = v_reg[s][i];
                }
            }
            if (tile + 1 < tile1) {
                request(tile + 1);
                page_ids(min(tile + 2, tile1 - 1));
            }
            u32x4_t hi[CT], lo[CT];
#pragma unroll
            for (int c = 0; c < CT; ++c) {
                float p[8];
#pragma unroll
                for (int e = 0; e < 8; ++e) {
                    p[e] = score[c][e >> 2][e & 3] * c_scale;
                }
                if (some_masked) {
#pragma unroll
                    for (int e = 0; e < 8; ++e) {
                        const int key = key0 + 16 * (e >> 2) + 4 * quad + (e & 3);
                        p[e] = key >= (GROUPED ? first[c] : r.first) && key < (GROUPED ? end[c] : r.end) ? p[e] : -INFINITY;
                    }
                }
                float top = fmaxf(fmaxf(fmaxf(p[0], p[1]), fmaxf(p[2], p[3])), fmaxf(fmaxf(p[4], p[5]), fmaxf(p[6], p[7])));
                top = fmaxf(top, __shfl_xor(top, 16));
                top = fmaxf(top, __shfl_xor(top, 32));
                if (__any(top > m[c])) {
                    const float m_new = fmaxf(m[c], top);
                    const float f = m_new == -INFINITY ? 1.0f : exp2_fast(m[c] - m_new);
                    m[c] = m_new;
                    l[c] *= f;
#pragma unroll
                    for (int i = 0; i < S::kDTiles; ++i) {
                        o[c][i] *= f;
                    }
                }
                const float m_used = m[c] == -INFINITY ? 0.0f : m[c] - Split<T>::kTop;
#pragma unroll
                for (int e = 0; e < 8; ++e) {
                    p[e] = exp2_fast(p[e] - m_used);
                    l[c] += p[e];
                }
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    uint32_t upper, lower;
                    split<T>(float2_t{p[2 * e], p[2 * e + 1]}, upper, lower);
                    hi[c][e] = upper, lo[c][e] = lower;
                }
            }
#pragma unroll
            for (int i = 0; i < S::kDTiles; ++i) {
                uint2 half[2];
#pragma unroll
                for (int s = 0; s < 2; ++s) {
                    half[s] = lds_read_transposed(lds + v_lds + s * 16 * S::kRowBytes + i * 32);
                }
                const uint4 vt = make_uint4(half[0].x, half[0].y, half[1].x, half[1].y);
                if constexpr (GROUPED) {
                    if (apart) {
                        for (int u = 0; u < r.count; ++u) {
                            const Keys seen = keys_of(a, t + u);
                            uint32_t mine[4] = {vt.x, vt.y, vt.z, vt.w};
#pragma unroll
                            for (int k = 0; k < 4; ++k) {
                                const int key = key0 + 16 * (k >> 1) + 4 * quad + 2 * (k & 1);
                                mine[k] &= (key >= seen.first && key < seen.end ? 0xFFFFu : 0u) |
                                           (key + 1 >= seen.first && key + 1 < seen.end ? 0xFFFF0000u : 0u);
                            }
                            const uint4 vu = make_uint4(mine[0], mine[1], mine[2], mine[3]);
#pragma unroll
                            for (int c = 0; c < CT; ++c) {
                                float4_t sum = o[c][i];
                                sum = T::mfma16(vu, __builtin_bit_cast(uint4, hi[c]), sum);
                                sum = T::mfma16(vu, __builtin_bit_cast(uint4, lo[c]), sum);
                                o[c][i] = row_in_unit[c] == u ? sum : o[c][i];
                            }
                        }
                        continue;
                    }
                }
#pragma unroll
                for (int c = 0; c < CT; ++c) {
                    o[c][i] = T::mfma16(vt, __builtin_bit_cast(uint4, hi[c]), o[c][i]);
                    o[c][i] = T::mfma16(vt, __builtin_bit_cast(uint4, lo[c]), o[c][i]);
                }
            }
        }

        // ---- the unit's part, or the whole of it ----
        const bool whole = tile0 == 0 && tile1 == r.tiles;
        const int64_t part = 2 * w + (tile0 == 0 ? 1 : 0);
        const AttentionWorkspace ws = carve(a.workspace, plan.runs, plan.cols);
        const auto out = [&](int j) {
            const Column at = plan.column<GROUPED>(unit, j);
            return a.out + static_cast<int64_t>(t + at.row) * a.ldo + static_cast<int64_t>(at.q_head) * D;
        };
        // What a whole unit's sums are divided by: NaN outside the table; a row that sees no key is zero over one.
        const auto divisor = [&](float sum, int keys_end) { return r.bad ? NAN : keys_end == 0 ? 1.0f : sum; };
#pragma unroll
        for (int c = 0; c < CT; ++c) {
            l[c] += __shfl_xor(l[c], 16);
            l[c] += __shfl_xor(l[c], 32);
            if (poisoned[GROUPED ? c : 0]) {
                l[c] = NAN;
            }
            const int before = 16 * c, used = min(16, columns - before);
            if constexpr (TEAM == 1) {
                if (col < used) {
                    const float over = divisor(l[c], GROUPED ? end[c] : r.end);
                    uint16_t *to = out(before + col);
#pragma unroll
                    for (int i = 0; i < S::kDTiles; ++i) {
                        const int d = 16 * i + 4 * quad;
                        if (whole) {
                            store4<T>(to + d, o[c][i] / over);
                        } else {
                            *reinterpret_cast<float4_t *>(ws.o + (part * plan.cols + before + col) * D + d) = o[c][i];
                        }
                    }
                    if (!whole && quad == 0) {
                        ws.stats[part * plan.cols + before + col] = make_float2(m[c], l[c]);
                    }
                }
            } else {
                if (quad == 0) {
                    wave_stats[wave][col] = make_float2(m[c], l[c]);
                }
                __syncthreads();
                {
                    float top = -INFINITY;
#pragma unroll
                    for (int i = 0; i < TEAM; ++i) {
                        top = fmaxf(top, wave_stats[i][col].x);
                    }
                    const float f = top == -INFINITY ? 0.0f : exp2_fast(m[c] - top);
                    float *mine = reinterpret_cast<float *>(lds + wave * S::kRegion);
                    if (col < used) {
#pragma unroll
                        for (int i = 0; i < S::kDTiles; ++i) {
                            *reinterpret_cast<float4_t *>(mine + col * S::kORow + 16 * i + 4 * quad) = o[c][i] * f;
                        }
                    }
                }
                __syncthreads();
                for (int i = threadIdx.x; i < used * (D / 4); i += kThreads) {
                    const int j = i / (D / 4), d = (i - j * (D / 4)) * 4;
                    float top = -INFINITY, sum = 0.0f;
                    float4_t v = float4_t{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
                    for (int k = 0; k < TEAM; ++k) {
                        top = fmaxf(top, wave_stats[k][j].x);
                    }
#pragma unroll
                    for (int k = 0; k < TEAM; ++k) {
                        const float2 st = wave_stats[k][j];
                        sum += st.y * (top == -INFINITY ? 1.0f : exp2_fast(st.x - top));
                        v += *reinterpret_cast<const float4_t *>(reinterpret_cast<const float *>(lds + k * S::kRegion) + j * S::kORow + d);
                    }
                    if (whole) {
                        const int keys_end = GROUPED && !r.bad ? keys_of(a, t + plan.column<GROUPED>(unit, before + j).row).end : r.end;
                        store4<T>(out(before + j) + d, v / divisor(sum, keys_end));
                    } else {
                        *reinterpret_cast<float4_t *>(ws.o + (part * plan.cols + before + j) * D + d) = v;
                        if (d == 0) {
                            ws.stats[part * plan.cols + before + j] = make_float2(top, sum);
                        }
                    }
                }
                __syncthreads();
            }
        }
        if (tile0 == 0 && !whole) {
            begun = AttentionDescriptor{t, unit, runs.of(x + r.tiles - 1) - w, r.count};
        }
        x = uniform(x + tile1 - tile0);
    }
    if (member == 0 && lane == 0 && w < plan.runs) {
        carve(a.workspace, plan.runs, plan.cols).desc[w] = begun;
    }
}

#include "hm_paged_attention_prompt.hpp"

// The parts of column j of one unit, of runs w .. w + pieces, joined into `out` (zero if the column sees no key): THREADS threads, kLanes parts at a time for each of its
// float4 elements, kAhead of them requested before the first is used.
template <class T, int D, int THREADS>
__device__ __forceinline__ void join_column(uint16_t *out, bool empty, const AttentionWorkspace &ws, int cols, int w, int pieces, int j) {
    constexpr int kItems = D / 4;
    constexpr int kLanes = THREADS / kItems;
    constexpr int kAhead = 8;
    __shared__ float4_t acc[kLanes][kItems];
    __shared__ float2 stat[kLanes];
    const int y = threadIdx.x / kItems, e = threadIdx.x - y * kItems;
    float m = -INFINITY, l = 0.0f;
    float4_t v = float4_t{0.0f, 0.0f, 0.0f, 0.0f};
    if (y < kLanes) {
        for (int i = y; i <= pieces; i += kAhead * kLanes) {
            float2 st[kAhead];
            float4_t o[kAhead];
            float top = m;
#pragma unroll
            for (int k = 0; k < kAhead; ++k) {
                const int p = min(i + k * kLanes, pieces);
                const int64_t part = 2 * (w + p) + (p == 0 ? 1 : 0);
                st[k] = ws.stats[part * cols + j];
                o[k] = *reinterpret_cast<const float4_t *>(ws.o + (part * cols + j) * D + 4 * e);
            }
#pragma unroll
            for (int k = 0; k < kAhead; ++k) {
                top = fmaxf(top, st[k].x); // the last part may count twice here
            }
            const float from = top == -INFINITY ? 0.0f : top; // no finite score yet: weights of zero
            const float f = exp2_fast(m - from);
            v *= f;
            l *= f;
#pragma unroll
            for (int k = 0; k < kAhead; ++k) {
                if (i + k * kLanes <= pieces) {
                    const float g = exp2_fast(st[k].x - from);
                    v += o[k] * g;
                    l += st[k].y * g;
                }
            }
            m = top;
        }
        acc[y][e] = v;
        if (e == 0) {
            stat[y] = make_float2(m, l);
        }
    }
    __syncthreads();
    if (y == 0) {
        float top = -INFINITY, sum = 0.0f;
        float4_t all = float4_t{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll 8
        for (int i = 0; i < kLanes; ++i) {
            top = fmaxf(top, stat[i].x);
        }
#pragma unroll 8
        for (int i = 0; i < kLanes; ++i) {
            const float f = exp2_fast(stat[i].x - (top == -INFINITY ? 0.0f : top));
            all += acc[i][e] * f;
            sum += stat[i].y * f;
        }
        store4<T>(out + 4 * e, empty ? float4_t{0.0f, 0.0f, 0.0f, 0.0f} : all / sum);
    }
    __syncthreads();
}

// Joins the unit that run blockIdx.x began and others went on with: columns blockIdx.y, blockIdx.y + gridDim.y, ... One wave: most find
// nothing to join and leave.
// The joins are a launch of their own: the count of arrivals that would let the last workgroup join in the first launch costs
// as much, since its stores, count and loads each go to memory and back past the XCDs' L2s, one after the other (and with fences of that
// scope instead, which write back and drop a whole L2, 64 rows of 8192 keys took 670 us).
template <class T, int D, bool GROUPED> __global__ void __launch_bounds__(64) join_kernel(PagedAttentionArgs a, AttentionPlan plan) {
    const AttentionWorkspace ws = carve(a.workspace, plan.runs, plan.cols);
    const AttentionDescriptor d = ws.desc[blockIdx.x];
    if (d.pieces == 0) {
        return;
    }
    const int columns = plan.columns<GROUPED>(d.unit, d.count);
    for (int j = blockIdx.y; j < columns; j += gridDim.y) {
        const Column at = plan.column<GROUPED>(d.unit, j);
        const int64_t row = d.row + at.row;
        join_column<T, D, 64>(a.out + row * a.ldo + static_cast<int64_t>(at.q_head) * D, a.positions[row] < 0, ws, plan.cols, blockIdx.x, d.pieces, j);
    }
}

// The same for few units, which have many parts each: a workgroup per unit and column, which finds the parts from the lengths.
constexpr int kFewThreads = 512;
template <class T, int D, bool GROUPED> __global__ void __launch_bounds__(kFewThreads) join_few_kernel(PagedAttentionArgs a, AttentionPlan plan) {
    constexpr int kTileKeys = kAttentionWaves * kWaveKeys; // few units are dealt in tiles of whole workgroups
    const int t = blockIdx.x / plan.units, unit = blockIdx.x - t * plan.units;
    __shared__ int sums[kFewThreads / 64][2];
    const Prompts prompts{0, 0}; // enough rows for them are not few units
    const Row own = row_of<GROUPED>(a, t, kTileKeys, plan.rows, prompts);
    int before = 0, total = 0;
    for (int i = threadIdx.x; i < static_cast<int>(a.rows); i += kFewThreads) {
        const int n = row_of<GROUPED>(a, i, kTileKeys, plan.rows, prompts).tiles;
        before += i < t ? n : 0;
        total += n;
    }
#pragma unroll
    for (int off = 32; off > 0; off >>= 1) {
        before += __shfl_xor(before, off);
        total += __shfl_xor(total, off);
    }
    if ((threadIdx.x & 63) == 0) {
        sums[threadIdx.x >> 6][0] = before;
        sums[threadIdx.x >> 6][1] = total;
    }
    __syncthreads();
    before = total = 0;
#pragma unroll
    for (int i = 0; i < kFewThreads / 64; ++i) {
        before += sums[i][0];
        total += sums[i][1];
    }
    if (own.tiles == 0) {
        return;
    }
    const Runs runs = Runs::deal(total * plan.units, plan.runs);
    const int first = before * plan.units + unit * own.tiles;
    const int w = runs.of(first), pieces = runs.of(first + own.tiles - 1) - w;
    const int j = blockIdx.y;
    if (pieces == 0 || j >= plan.columns<GROUPED>(unit, own.count)) {
        return;
    }
    const Column at = plan.column<GROUPED>(unit, j);
    const int64_t row = t + at.row;
    join_column<T, D, kFewThreads>(a.out + row * a.ldo + static_cast<int64_t>(at.q_head) * D, a.positions[row] < 0,
                                   carve(a.workspace, plan.runs, plan.cols), plan.cols, w, pieces, j);
}

template <class T, int D, int TEAM, int CT, bool GROUPED> hipError_t launch(const PagedAttentionArgs &a, const AttentionPlan &plan, hipStream_t stream) {
    if (plan.counted) {
        hipLaunchKernelGGL((count_kernel<GROUPED>), dim3(kChunks), dim3(kThreads), 0, stream, a, plan);
        const hipError_t e = hipGetLastError();
        if (e != hipSuccess) {
            return e;
        }
    }
    if constexpr (GROUPED) {
        if (plan.prompt_rows != 0) {
            const unsigned prompt_blocks = static_cast<unsigned>(a.rows / plan.prompt_rows * a.kv_heads);
            hipLaunchKernelGGL((prompt_attention_kernel<T, D>), dim3(prompt_blocks), dim3(kThreads), 0, stream, a, plan);
            const hipError_t e = hipGetLastError();
            if (e != hipSuccess) {
                return e;
            }
        }
    }
    const unsigned blocks = static_cast<unsigned>((plan.runs * TEAM + kAttentionWaves - 1) / kAttentionWaves);
    hipLaunchKernelGGL((paged_attention_kernel<T, D, TEAM, CT, GROUPED>), dim3(blocks), dim3(kThreads), 0, stream, a, plan);
    const hipError_t e = hipGetLastError();
    if (e != hipSuccess || !plan.joins) {
        return e;
    }
    if (plan.few_units) {
        hipLaunchKernelGGL((join_few_kernel<T, D, GROUPED>), dim3(static_cast<unsigned>(a.rows * plan.units), static_cast<unsigned>(plan.cols)),
                           dim3(kFewThreads), 0, stream, a, plan);
    } else {
        hipLaunchKernelGGL((join_kernel<T, D, GROUPED>), dim3(static_cast<unsigned>(plan.runs), static_cast<unsigned>(plan.join_cols)), dim3(64), 0,
                           stream, a, plan);
    }
    return hipGetLastError();
}

template <class T, int D> hipError_t launch_d(const PagedAttentionArgs &a, const AttentionPlan &plan, hipStream_t stream) {
    if (plan.rows > 1 || plan.prompt_rows != 0) {
        return plan.team == 1 ? launch<T, D, 1, 1, true>(a, plan, stream) : launch<T, D, 4, 1, true>(a, plan, stream);
    }
    return plan.team == 1     ? launch<T, D, 1, 1, false>(a, plan, stream)
           : plan.cols <= 16 ? launch<T, D, 4, 1, false>(a, plan, stream)
                              : launch<T, D, 4, 2, false>(a, plan, stream);
}

template <class T> hipError_t launch_t(const PagedAttentionArgs &a, const AttentionPlan &plan, hipStream_t stream) {
    switch (a.head_dim) {
    case 64:
        return launch_d<T, 64>(a, plan, stream);
    case 96:
        return launch_d<T, 96>(a, plan, stream);
    case 128:
        return launch_d<T, 128>(a, plan, stream);
    default:
        return launch_d<T, 256>(a, plan, stream);
    }
}

} // namespace
} // namespace hm
