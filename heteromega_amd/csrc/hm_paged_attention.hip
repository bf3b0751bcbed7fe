// Attention of one query token per row over a paged key-value cache: out = softmax(scale q K^T) V per query head.
//
// Bound by memory: every key and value is read once (4 D bytes per key and key head) for 4 D flops per query head on it, and
// the query heads of a key head (G, up to 16 at a time) are the columns of one MFMA tile, so that they share the reads.
//
// A wave takes 32 keys at a time, as two sub-tiles of 16 keys (a page holds whole sub-tiles):
//   S^T [key, q] = K Q^T   v_mfma_f32_16x16x32: A = K, lane L holds key L & 15 and 8 consecutive elements; B = Q^T, kept in
//                          registers.
//   O^T [d, q] += V^T P^T  A = V^T, read from LDS transposed (ds_read_b64_tr_b16); B = P^T.
// Rows of K and V are loaded whole by neighbouring lanes and pass through LDS, K as well as V: loads in A's own order touch 64
// bytes of 16 rows each, and took 394 us instead of 362 (64 rows of 8192 keys, 8 key heads of 128).
// In S^T a lane holds, for one column q = L & 15, keys 4 (L >> 4) + i of each sub-tile. The k index of the second product may
// be dealt in any order that A and B share, so those eight weights are its B operand as they are: no weight crosses
// lanes. O^T keeps one q per lane too, so rescaling by a new maximum is one factor per lane.
// The scores' running maximum m and the sum l of p = 2^(c s - m) (c = scale log2 e) are fp32. p enters the second product as
// hi + lo, two 16-bit floats of which lo holds what hi lacks (to 2^-16 of p in bf16, 2^-22 in fp16): 16-bit weights alone would add
// an error the size of the output's own rounding, and the matrix cores are idle most of the time here.
//
// Rows differ in length, and their lengths are known on the device only. So the work is dealt in tiles of 128 keys (32 per wave of a
// workgroup): all tiles of all (row, key head) units in one line, cut into equal runs, one per workgroup. A run may end inside
// a unit; then each workgroup's part (fp32 O, m, l) goes to the workspace and a second launch joins the parts. Every
// workgroup finds its place by summing the rows' tile counts itself.
#include "hm_device.hpp"
#include "hm_internal.hpp"

#include <algorithm>

namespace hm {
namespace {

constexpr int kWaves = 4;
constexpr int kThreads = 64 * kWaves;
constexpr int kWaveKeys = 32;
constexpr int kTileKeys = kWaveKeys * kWaves;
constexpr int kPerCu = 2; // workgroups per CU
constexpr int kStream = 2; // cache policy of the keys and values, read once: non-temporal

typedef uint32_t u32x4_t __attribute__((ext_vector_type(4)));


struct Descriptor { // of a workgroup's last unit, when it begins there and is not finished
    int32_t row, unit, pieces, pad; // pieces: workgroups behind this one that hold its other parts
};

// The workspace of `groups` workgroups with `cols` columns (query heads of a unit).
struct Workspace {
    Descriptor *desc;
    float2 *stats; // [2 groups][cols]: m, l of each part; part 2 w: of the unit that workgroup w goes on with, 2 w + 1: of the one it begins
    float *o;      // [2 groups][cols][D]
};

__host__ __device__ __forceinline__ Workspace carve(void *p, int64_t groups, int cols) {
    Workspace w;
    uint8_t *b = static_cast<uint8_t *>(p);
    w.desc = reinterpret_cast<Descriptor *>(b);
    b += groups * static_cast<int64_t>(sizeof(Descriptor));
    w.stats = reinterpret_cast<float2 *>(b);
    b += (2 * groups * cols * static_cast<int64_t>(sizeof(float2)) + 15) / 16 * 16;
    w.o = reinterpret_cast<float *>(b);
    return w;
}

// The keys of one row: [first, end) are seen, the tiles begin at start.
struct Row {
    int32_t request, first, start, end, tiles;
    bool bad; // request or position outside the table
};

__device__ __forceinline__ Row row_of(const PagedAttentionArgs &a, int64_t t) {
    Row r;
    r.request = a.requests != nullptr ? a.requests[t] : static_cast<int32_t>(t);
    const int32_t pos = a.positions[t];
    r.bad = r.request >= a.requests_count || pos < -1 || pos >= (a.width << a.page_shift);
    r.end = r.bad ? 0 : pos + 1;
    r.first = a.window > 0 && a.window < r.end ? r.end - static_cast<int32_t>(a.window) : 0;
    r.start = r.first & ~15;
    // A row without keys still has an output to write.
    r.tiles = r.request < 0 ? 0 : max(1, (r.end - r.start + kTileKeys - 1) / kTileKeys);
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
    return Row{uniform(r.request), uniform(r.first), uniform(r.start), uniform(r.end), uniform(r.tiles), uniform(r.bad) != 0};
}

__device__ __forceinline__ float exp2_fast(float x) { return __builtin_amdgcn_exp2f(x); }

template <class T> __device__ __forceinline__ void store4(uint16_t *p, float4_t v) {
    uint2 o;
    o.x = static_cast<uint32_t>(T::from_float(v[0])) | (static_cast<uint32_t>(T::from_float(v[1])) << 16);
    o.y = static_cast<uint32_t>(T::from_float(v[2])) | (static_cast<uint32_t>(T::from_float(v[3])) << 16);
    *reinterpret_cast<uint2 *>(p) = o;
}

// The compiler's types of T, for its conversion instructions, and the power of two that the largest weight has: fp16 loses
// weights below 2^-25, of which a long row can have enough to matter next to a weight of 1; from 2^15 down to its subnormals
// it has 2^40 of range. kBelow keeps hi below p by more than its rounding, so that lo is positive as well: an infinite value
// then gives an infinite output, as p alone would, where a lo of zero or below would make it NaN.
template <class T> struct Split;
template <> struct Split<F16> {
    typedef half8_t vec;
    typedef _Float16 elem;
    static constexpr float kTop = 15.0f;
    static constexpr float kBelow = 1.0f - 0x1p-11f;
};
template <> struct Split<BF16> {
    typedef bf16x8_t vec;
    typedef __bf16 elem;
    static constexpr float kTop = 0.0f;
    static constexpr float kBelow = 1.0f - 0x1p-8f;
};

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

template <class T, int D>
__global__ void __launch_bounds__(kThreads, D <= 128 ? 2 : 1) paged_attention_kernel(PagedAttentionArgs a, int groups, int cols, int col_tiles) {
    using S = Shape<T, D>;
    using vec = typename Split<T>::vec;
    using elem = typename Split<T>::elem;
    __shared__ __attribute__((aligned(16))) uint8_t lds[kWaves * S::kRegion];
    __shared__ float2 wave_stats[kWaves][16];
    __shared__ int scan[kWaves];
    __shared__ int found, found_base;

    const int lane = threadIdx.x & 63, wave = uniform(threadIdx.x >> 6);
    const int col = lane & 15, quad = lane >> 4;
    const int units = a.kv_heads * col_tiles;
    const int w = blockIdx.x, rows = static_cast<int>(a.rows);

    // ---- this workgroup's run of tiles, [x, x_end) ----
    int x, x_end, per_run, longer; // the first `longer` runs have per_run + 1 tiles, the others per_run
    int t = 0, base = 0;           // the row that x lies in, and the row's first tile
    Row r{};
    {
        const int per = (rows + kThreads - 1) / kThreads;
        const int t0 = min(static_cast<int>(threadIdx.x) * per, rows), t1 = min(t0 + per, rows);
        int own = 0;
        for (int i = t0; i < t1; ++i) {
            own += row_of(a, i).tiles;
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
        for (int i = 0; i < kWaves; ++i) {
            before += i < wave ? scan[i] : 0;
            total += scan[i];
        }
        total = uniform(total) * units;
        per_run = static_cast<uint32_t>(total) / static_cast<uint32_t>(groups);
        longer = total - per_run * groups;
        x = w * per_run + min(w, longer);
        x_end = x + per_run + (w < longer ? 1 : 0);
        if (x < x_end && before * units <= x && x < (before + own) * units) {
            int b = before * units;
            for (int i = t0; i < t1; ++i) {
                const int n = (per == 1 ? own : row_of(a, i).tiles) * units;
                if (x < b + n) {
                    found = i;
                    found_base = b;
                    break;
                }
                b += n;
            }
        }
        __syncthreads();
    }
    Descriptor begun{0, 0, 0, 0};
    if (x < x_end) {
        t = uniform(found);
        base = uniform(found_base);
        r = uniform_row(row_of(a, t));
    }

    // ---- constants of the lane ----
    const uint32_t row_bytes = static_cast<uint32_t>(a.token_stride) * 2;
    // Pieces of 16 bytes of a sub-tile's rows as the lanes load them, whole rows by neighbouring lanes.
    const Pieces<D> pieces(lane, row_bytes);
    const uint32_t to_lds = wave * S::kRegion + pieces.lds_offset();
    const uint32_t k_lds = wave * S::kRegion + col * S::kRowBytes + quad * 16;
    const uint32_t v_lds = wave * S::kRegion + (4 * quad + (col >> 2)) * S::kRowBytes + (col & 3) * 8;
    const float c_scale = a.scale * 1.4426950408889634f;
    const int group_heads = a.q_heads / a.kv_heads;

    while (x < x_end) {
        while (x >= base + r.tiles * units) { // on to the next row with tiles, 64 at a time
            base = uniform(base + r.tiles * units);
            int from = t + 1;
            uint64_t some = 0;
            for (; from < rows; from += 64) {
                some = __ballot(from + lane < rows && row_of(a, min(from + lane, rows - 1)).tiles > 0);
                if (some != 0) {
                    break;
                }
            }
            t = uniform(some != 0 ? from + static_cast<int>(__builtin_ctzll(some)) : rows - 1); // a run ends before the rows do
            r = uniform_row(row_of(a, t));
        }
        const int unit = uniform(static_cast<uint32_t>(x - base) / static_cast<uint32_t>(r.tiles));
        const int tile0 = x - base - unit * r.tiles;
        const int tile1 = min(r.tiles, tile0 + (x_end - x));
        const int kv_head = uniform(col_tiles == 1 ? unit : unit / col_tiles);
        const int head_in_group = (unit - kv_head * col_tiles) * 16;
        const int used = min(16, group_heads - head_in_group);
        const int q_head = kv_head * group_heads + head_in_group;

        u32x4_t q[S::kSteps];
        const uint16_t *q_row = a.q + static_cast<int64_t>(t) * a.ldq + static_cast<int64_t>(q_head + (col < used ? col : 0)) * D + 8 * quad;
#pragma unroll
        for (int s = 0; s < S::kSteps; ++s) {
            q[s] = col < used ? *reinterpret_cast<const u32x4_t *>(q_row + 32 * s) : u32x4_t{0, 0, 0, 0};
        }

        float4_t o[S::kDTiles];
#pragma unroll
        for (int i = 0; i < S::kDTiles; ++i) {
            o[i] = float4_t{0.0f, 0.0f, 0.0f, 0.0f};
        }
        float m = -INFINITY, l = 0.0f;
        bool poisoned = false;

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
                const int key = r.start + tile * kTileKeys + wave * kWaveKeys + 16 * s;
                id[s] = key < r.end ? table[key >> shift] : 0;
            }
        };
        const auto request = [&](int tile) {
#pragma unroll
            for (int s = 0; s < 2; ++s) {
                const int key = r.start + tile * kTileKeys + wave * kWaveKeys + 16 * s;
                const int32_t page = uniform(id[s]);
                int seen = max(0, min(16, r.end - key));
                if (static_cast<uint32_t>(page) >= pages) {
                    poisoned |= seen > 0;
                    seen = 0;
                }
                // Past the row's last key the buffer ends, and its loads return zero.
                const uint32_t bytes = uniform(seen > 0 ? (seen - 1) * row_bytes + 2 * D : 0);
                const int64_t at = uniform64(seen > 0 ? page * page_stride + static_cast<int64_t>(key & offset_mask) * (row_bytes / 2) : 0);
                const __amdgpu_buffer_rsrc_t kr = buffer_rsrc(k_head + at, bytes), vr = buffer_rsrc(v_head + at, bytes);
#pragma unroll
                for (int i = 0; i < S::kSteps; ++i) {
                    k_reg[s][i] = __builtin_amdgcn_raw_buffer_load_b128(kr, pieces.offset(i), 0, kStream);
                }
#pragma unroll
                for (int i = 0; i < S::kSteps; ++i) {
                    v_reg[s][i] = __builtin_amdgcn_raw_buffer_load_b128(vr, pieces.offset(i), 0, kStream);
                }
            }
        };
        page_ids(tile0);
        request(tile0);
        page_ids(min(tile0 + 1, tile1 - 1));
        for (int tile = tile0; tile < tile1; ++tile) {
            const int key0 = r.start + tile * kTileKeys + wave * kWaveKeys;
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
            // K and then V pass through the wave's own region of LDS; a wave's LDS accesses are carried out in order.
#pragma unroll
            for (int s = 0; s < 2; ++s) {
#pragma unroll
                for (int i = 0; i < S::kSteps; ++i) {
                    *reinterpret_cast<u32x4_t *>(lds + to_lds + pieces.lds_step(i) + s * 16 * S::kRowBytes) = k_reg[s][i];
                }
            }
            float4_t score[2] = {float4_t{0.0f, 0.0f, 0.0f, 0.0f}, float4_t{0.0f, 0.0f, 0.0f, 0.0f}};
#pragma unroll
            for (int i = 0; i < S::kSteps; ++i) {
#pragma unroll
                for (int s = 0; s < 2; ++s) {
                    const uint4 k = *reinterpret_cast<const uint4 *>(lds + k_lds + s * 16 * S::kRowBytes + 64 * i);
                    score[s] = T::mfma16(k, __builtin_bit_cast(uint4, q[i]), score[s]);
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
            float p[8];
#pragma unroll
            for (int s = 0; s < 2; ++s) {
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    p[4 * s + i] = score[s][i] * c_scale;
                }
            }
            if (key0 < r.first || key0 + kWaveKeys > r.end) {
#pragma unroll
                for (int e = 0; e < 8; ++e) {
                    const int key = key0 + 16 * (e >> 2) + 4 * quad + (e & 3);
                    p[e] = key >= r.first && key < r.end ? p[e] : -INFINITY;
                }
            }
            float top = fmaxf(fmaxf(fmaxf(p[0], p[1]), fmaxf(p[2], p[3])), fmaxf(fmaxf(p[4], p[5]), fmaxf(p[6], p[7])));
            top = fmaxf(top, __shfl_xor(top, 16));
            top = fmaxf(top, __shfl_xor(top, 32));
            if (__any(top > m)) {
                const float m_new = fmaxf(m, top);
                const float f = m_new == -INFINITY ? 1.0f : exp2_fast(m - m_new);
                m = m_new;
                l *= f;
#pragma unroll
                for (int i = 0; i < S::kDTiles; ++i) {
                    o[i] *= f;
                }
            }
            const float m_used = m == -INFINITY ? 0.0f : m - Split<T>::kTop;
            vec hi, lo;
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                p[e] = exp2_fast(p[e] - m_used);
                l += p[e];
                hi[e] = static_cast<elem>(p[e] * Split<T>::kBelow);
                lo[e] = static_cast<elem>(p[e] - static_cast<float>(hi[e]));
            }
#pragma unroll
            for (int i = 0; i < S::kDTiles; ++i) {
                uint2 half[2];
#pragma unroll
                for (int s = 0; s < 2; ++s) {
                    half[s] = lds_read_transposed(lds + v_lds + s * 16 * S::kRowBytes + i * 32);
                }
                const uint4 vt = make_uint4(half[0].x, half[0].y, half[1].x, half[1].y);
                o[i] = T::mfma16(vt, __builtin_bit_cast(uint4, hi), o[i]);
                o[i] = T::mfma16(vt, __builtin_bit_cast(uint4, lo), o[i]);
            }
        }

        // ---- the waves' parts become the workgroup's ----
        l += __shfl_xor(l, 16);
        l += __shfl_xor(l, 32);
        if (poisoned) {
            l = NAN;
        }
        if (quad == 0) {
            wave_stats[wave][col] = make_float2(m, l);
        }
        __syncthreads();
        {
            float top = -INFINITY;
#pragma unroll
            for (int i = 0; i < kWaves; ++i) {
                top = fmaxf(top, wave_stats[i][col].x);
            }
            const float f = top == -INFINITY ? 0.0f : exp2_fast(m - top);
            float *mine = reinterpret_cast<float *>(lds + wave * S::kRegion);
            if (col < used) {
#pragma unroll
                for (int i = 0; i < S::kDTiles; ++i) {
                    *reinterpret_cast<float4_t *>(mine + col * S::kORow + 16 * i + 4 * quad) = o[i] * f;
                }
            }
        }
        __syncthreads();
        const bool whole = tile0 == 0 && tile1 == r.tiles;
        const int64_t part = 2 * w + (tile0 == 0 ? 1 : 0);
        const Workspace ws = carve(a.workspace, groups, cols);
        for (int i = threadIdx.x; i < used * (D / 4); i += kThreads) {
            const int j = i / (D / 4), d = (i - j * (D / 4)) * 4;
            float top = -INFINITY, sum = 0.0f;
            float4_t v = float4_t{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
            for (int k = 0; k < kWaves; ++k) {
                top = fmaxf(top, wave_stats[k][j].x);
            }
#pragma unroll
            for (int k = 0; k < kWaves; ++k) {
                const float2 st = wave_stats[k][j];
                sum += st.y * (top == -INFINITY ? 1.0f : exp2_fast(st.x - top));
                v += *reinterpret_cast<const float4_t *>(reinterpret_cast<const float *>(lds + k * S::kRegion) + j * S::kORow + d);
            }
            if (whole) {
                if (r.bad) {
                    sum = NAN;
                }
                v = r.end == r.first && !r.bad ? float4_t{0.0f, 0.0f, 0.0f, 0.0f} : v / sum;
                store4<T>(a.out + static_cast<int64_t>(t) * a.ldo + static_cast<int64_t>(q_head + j) * D + d, v);
            } else {
                *reinterpret_cast<float4_t *>(ws.o + (part * cols + j) * D + d) = v;
                if (d == 0) {
                    ws.stats[part * cols + j] = make_float2(top, sum);
                }
            }
        }
        __syncthreads();
        if (tile0 == 0 && !whole) {
            const uint32_t last = x + r.tiles - 1; // the unit's last tile, and the workgroup that has it
            const uint32_t long_tiles = longer * (per_run + 1);
            const int last_w = last < long_tiles ? last / (per_run + 1) : longer + (last - long_tiles) / per_run;
            begun = Descriptor{t, unit, last_w - w, 0};
        }
        x = uniform(x + tile1 - tile0);
    }
    if (threadIdx.x == 0) {
        carve(a.workspace, groups, cols).desc[w] = begun;
    }
}

// Joins the parts of the unit that workgroup blockIdx.x began and others went on with: columns blockIdx.y, blockIdx.y + gridDim.y, ...
// A launch of its own: the count of arrivals that would let the last workgroup join in the first launch costs more, since its
// stores, count and loads each go to memory and back past the XCDs' L2s (one row of 1037 keys: 17.5 us instead of 12.3).
template <class T, int D, int THREADS>
__global__ void __launch_bounds__(THREADS) join_kernel(PagedAttentionArgs a, int groups, int cols, int col_tiles) {
    constexpr int kItems = D / 4;            // float4 elements of a column
    constexpr int kLanes = THREADS / kItems; // parts that the workgroup reads at a time, kAhead times
    constexpr int kAhead = 4;
    __shared__ float4_t acc[kLanes][kItems];
    __shared__ float2 stat[kLanes];
    const Workspace ws = carve(a.workspace, groups, cols);
    const int w = blockIdx.x;
    const Descriptor d = ws.desc[w];
    if (d.pieces == 0) {
        return;
    }
    const int kv_head = d.unit / col_tiles;
    const int head_in_group = (d.unit - kv_head * col_tiles) * 16;
    const int group_heads = a.q_heads / a.kv_heads;
    const int used = min(16, group_heads - head_in_group);
    const int y = threadIdx.x / kItems, e = threadIdx.x - y * kItems;
    for (int j = blockIdx.y; j < used; j += gridDim.y) {
        float m = -INFINITY, l = 0.0f;
        float4_t v = float4_t{0.0f, 0.0f, 0.0f, 0.0f};
        if (y < kLanes) {
            for (int i = y; i <= d.pieces; i += kAhead * kLanes) {
                float2 st[kAhead];
                float4_t o[kAhead];
                float top = m;
#pragma unroll
                for (int k = 0; k < kAhead; ++k) {
                    const int p = min(i + k * kLanes, d.pieces);
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
                    if (i + k * kLanes <= d.pieces) {
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
            float4_t out = float4_t{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
            for (int i = 0; i < kLanes; ++i) {
                top = fmaxf(top, stat[i].x);
            }
#pragma unroll
            for (int i = 0; i < kLanes; ++i) {
                const float f = exp2_fast(stat[i].x - (top == -INFINITY ? 0.0f : top));
                out += acc[i][e] * f;
                sum += stat[i].y * f;
            }
            store4<T>(a.out + d.row * a.ldo + static_cast<int64_t>(kv_head * group_heads + head_in_group + j) * D + 4 * e, out / sum);
        }
        __syncthreads();
    }
}

int64_t max_groups() { return kPerCu * device_topology().cus; }

template <class T, int D> hipError_t launch(const PagedAttentionArgs &a, int64_t groups, int cols, int col_tiles, hipStream_t stream) {
    hipLaunchKernelGGL((paged_attention_kernel<T, D>), dim3(static_cast<unsigned>(groups)), dim3(kThreads), 0, stream, a, static_cast<int>(groups),
                       cols, col_tiles);
    const hipError_t e = hipGetLastError();
    if (e != hipSuccess) {
        return e;
    }
    // Most of these workgroups find nothing to join and leave, so one wave each; four where few units have many parts.
    const dim3 grid(static_cast<unsigned>(groups), static_cast<unsigned>(std::min(cols, 4)));
    if (groups <= 16 * a.rows * a.kv_heads * col_tiles) {
        hipLaunchKernelGGL((join_kernel<T, D, 64>), grid, dim3(64), 0, stream, a, static_cast<int>(groups), cols, col_tiles);
    } else {
        hipLaunchKernelGGL((join_kernel<T, D, 256>), grid, dim3(256), 0, stream, a, static_cast<int>(groups), cols, col_tiles);
    }
    return hipGetLastError();
}

template <class T> hipError_t launch_type(const PagedAttentionArgs &a, int64_t groups, int cols, int col_tiles, hipStream_t stream) {
    switch (a.head_dim) {
    case 64:
        return launch<T, 64>(a, groups, cols, col_tiles, stream);
    case 96:
        return launch<T, 96>(a, groups, cols, col_tiles, stream);
    case 128:
        return launch<T, 128>(a, groups, cols, col_tiles, stream);
    default:
        return launch<T, 256>(a, groups, cols, col_tiles, stream);
    }
}

} // namespace

size_t paged_attention_workspace(int64_t q_heads, int64_t kv_heads, int64_t head_dim) {
    const int64_t groups = max_groups(), cols = std::min<int64_t>(16, q_heads / kv_heads);
    return static_cast<size_t>(groups * static_cast<int64_t>(sizeof(Descriptor)) + (2 * groups * cols * 8 + 15) / 16 * 16 + 2 * groups * cols * head_dim * 4);
}

hipError_t launch_paged_attention(const PagedAttentionArgs &a, hipStream_t stream) {
    if (a.rows == 0) {
        return hipSuccess;
    }
    const int64_t per_head = a.q_heads / a.kv_heads;
    const int cols = static_cast<int>(std::min<int64_t>(16, per_head));
    const int col_tiles = static_cast<int>((per_head + 15) / 16);
    const int64_t most = a.rows * a.kv_heads * col_tiles * (((a.width << a.page_shift) + kTileKeys - 1) / kTileKeys + 1);
    const int64_t groups = std::max<int64_t>(1, std::min(max_groups(), most));
    return a.dtype == HM_FP16 ? launch_type<F16>(a, groups, cols, col_tiles, stream) : launch_type<BF16>(a, groups, cols, col_tiles, stream);
}

} // namespace hm
