// Attention over shared pages: the kernels (hm_shared_attention.hip has the mathematics and the launch rules). They take the tiles' shapes, loads and
// weights from hm_paged_attention_kernel.hpp.
#pragma once

#include "hm_paged_attention_kernel.hpp"
#include "hm_shared_attention.hpp"

#include <type_traits>

namespace hm {
namespace {

// A run's segments, the next one on the way: one of its numbers a lane. The one behind the line's last is read too, and not used: other memory of the plan.
struct Segments {
    const ShareSegment *line;
    int at;
    int32_t next;

    __device__ __forceinline__ Segments(const ShareSegment *l, int first) : line(l), at(first) { read(); }
    __device__ __forceinline__ void read() { next = reinterpret_cast<const int32_t *>(line + at)[threadIdx.x & 7]; }
    __device__ __forceinline__ ShareSegment take() const {
        const auto of = [&](int i) { return __builtin_amdgcn_readlane(next, i); };
        return {of(0), of(1), of(2), of(3), of(4), of(5), of(6), of(7)};
    }
    __device__ __forceinline__ void move_on() {
        ++at;
        read();
    }
};
static_assert(sizeof(ShareSegment) == 32, "eight numbers");

// A unit's tiles [tile0, tile1).
struct Work {
    ShareSegment s;
    int kv_head, row, rows; // row: first, behind the segment's
    int tile0, tile1;
    int64_t part; // its first column among the parts
};

// The next work of a run [x, x_end) of a line; moves x on.
template <int LINE> __device__ __forceinline__ Work next_work(const SharedAttentionArgs &a, Segments &segments, int &x, int x_end, int w) {
    Work k;
    k.s = segments.take();
    const int chunks = LINE == 0 ? 1 : k.s.chunks();
    const int unit = uniform(static_cast<uint32_t>(x - k.s.tile0) / static_cast<uint32_t>(k.s.tiles));
    k.kv_head = LINE == 0 ? unit : unit / chunks;
    k.row = LINE == 0 ? 0 : (unit - k.kv_head * chunks) * k.s.chunk;
    k.rows = min(k.s.chunk, k.s.rows - k.row);
    k.tile0 = x - k.s.tile0 - unit * k.s.tiles;
    k.tile1 = min(k.s.tiles, k.tile0 + (x_end - x));
    k.part = k.tile1 == k.s.tiles ? static_cast<int64_t>(k.s.slot0) * a.q_heads + (static_cast<int64_t>(k.kv_head) * k.s.rows + k.row) * a.group_heads
                                  : run_column(a.rows, a.q_heads, a.groups, LINE, w);
    x += k.tile1 - k.tile0;
    if (k.tile1 == k.s.tiles && unit + 1 == a.kv_heads * chunks) {
        segments.move_on();
    }
    return k;
}

// Where a unit's request has its keys.
struct Pages {
    const int32_t *table;
    const uint16_t *k_head, *v_head;
    int64_t page_stride;
    int shift, mask;
    uint32_t pages, row_bytes;
    int capacity;
    bool there;

    // Page numbers are read for up to 2032 keys behind the last one, which may be at the end of 31 bits: the key has 32.
    __device__ __forceinline__ int32_t page_of(uint32_t key, int hi) const {
        return key >= static_cast<uint32_t>(hi) ? 0 : there && key < static_cast<uint32_t>(capacity) ? table[key >> shift] : -1;
    }
    __device__ __forceinline__ Pages(const SharedAttentionArgs &a, int64_t row, int kv_head) {
        // The plan's requests and keys are those of its call, whose table this call's should be: one that is not there is poisoned.
        const int64_t request = a.requests != nullptr ? a.requests[row] : row;
        there = request >= 0 && request < a.requests_count;
        table = a.block_table + uniform64(there ? request * a.ld_table : 0);
        capacity = uniform(static_cast<int>(a.width << a.page_shift));
        k_head = a.k + uniform64(kv_head * a.head_stride), v_head = a.v + uniform64(kv_head * a.head_stride);
        page_stride = uniform64(a.page_stride);
        shift = uniform(a.page_shift), mask = (1 << shift) - 1;
        pages = uniform(static_cast<int>(a.pages));
        row_bytes = static_cast<uint32_t>(a.token_stride) * 2;
    }
    // Bytes and first element of `seen` keys of a page from `key` on.
    template <int D> __device__ __forceinline__ uint32_t bytes(int seen) const { return uniform(seen > 0 ? (seen - 1) * row_bytes + 2 * D : 0); }
    __device__ __forceinline__ int64_t offset(int32_t page, int key, int seen) const {
        return uniform64(seen > 0 ? page * page_stride + static_cast<int64_t>(key & mask) * (row_bytes / 2) : 0);
    }
};

// The pages of 64 sub-tiles of 16 keys, a lane each, from one read of the table for all of them. They stay from a unit to the next, which mostly is of the same rows
// and another key head.
struct PageIds {
    int32_t ids = 0;
    int first = -1, row = -1, start = 0, end = 0; // sub-tile of lane 0, and whose keys
    bool bad = false;                    // a page outside the cache

    __device__ __forceinline__ void read(const Pages &at, const ShareSegment &s, int sub) {
        if (first != sub || row != s.row0 || start != s.start() || end != s.hi) {
            first = sub, row = s.row0, start = s.start(), end = s.hi;
            ids = at.page_of(static_cast<uint32_t>(start) + 16 * (static_cast<uint32_t>(sub) + (threadIdx.x & 63)), s.hi);
            bad = __any(static_cast<uint32_t>(ids) >= at.pages);
        }
    }
    __device__ __forceinline__ int32_t of(int sub) const { return __builtin_amdgcn_readlane(ids, sub - first); }
};

// A unit of up to 16 CT columns, by one wave, 32 keys at a time: with up to 128 units on a CU one after the other, waves go on to their next by themselves.
template <class T, int D, int CT> __device__ __forceinline__ void narrow_work(const SharedAttentionArgs &a, const Work &k, uint8_t *lds, PageIds &ids) {
    using S = Shape<T, D>;
    const int lane = threadIdx.x & 63;
    const int col = lane & 15, quad = lane >> 4;
    const int columns = k.rows * a.group_heads, start = k.s.start(), lo = k.s.lo, hi = k.s.hi;
    const Pages at(a, k.s.row0, k.kv_head);
    const Pieces<D> pieces(lane, at.row_bytes);
    const uint32_t to_lds = pieces.lds_offset();
    const uint32_t k_lds = col * S::kRowBytes + quad * 16;
    const uint32_t v_lds = (4 * quad + (col >> 2)) * S::kRowBytes + (col & 3) * 8;
    const float c_scale = a.scale * 1.4426950408889634f;

    u32x4_t q[CT][S::kSteps];
    float4_t o[CT][S::kDTiles];
    float m[CT], l[CT];
#pragma unroll
    for (int c = 0; c < CT; ++c) {
        const int column = 16 * c + col, row = column / a.group_heads;
        const bool live = column < columns;
        const uint16_t *q_row =
            a.q + (live ? (k.s.row0 + row) * a.ldq + static_cast<int64_t>(k.kv_head * a.group_heads + column - row * a.group_heads) * D : 0) + 8 * quad;
#pragma unroll
        for (int s = 0; s < S::kSteps; ++s) {
            q[c][s] = live ? *reinterpret_cast<const u32x4_t *>(q_row + 32 * s) : u32x4_t{0, 0, 0, 0};
        }
#pragma unroll
        for (int i = 0; i < S::kDTiles; ++i) {
            o[c][i] = float4_t{0.0f, 0.0f, 0.0f, 0.0f};
        }
        m[c] = -INFINITY, l[c] = 0.0f;
    }
    bool poisoned = false; // a page outside the cache

    constexpr int kTilesAhead = D == 64 ? 2 : 1; // 16 KB on the way for each wave keep the memory busy with one workgroup on a CU, 8 KB do not
    u32x4_t k_reg[kTilesAhead][2][S::kSteps], v_reg[kTilesAhead][2][S::kSteps];
    const auto request = [&](int tile, auto &k_reg, auto &v_reg) __attribute__((always_inline)) {
        if (2 * (tile - k.tile0) % 64 == 0) {
            ids.read(at, k.s, 2 * tile);
            poisoned |= ids.bad;
        }
#pragma unroll
        for (int s = 0; s < 2; ++s) {
            const int key = start + tile * kNarrowTile + 16 * s;
            const int32_t page = ids.of(2 * tile + s);
            const int seen = static_cast<uint32_t>(page) < at.pages ? max(0, min(16, hi - key)) : 0;
            const uint32_t bytes = at.bytes<D>(seen);
            const int64_t from = at.offset(page, key, seen);
            const __amdgpu_buffer_rsrc_t kr = buffer_rsrc(at.k_head + from, bytes), vr = buffer_rsrc(at.v_head + from, bytes);
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
    const auto step = [&](int tile, auto &k_reg, auto &v_reg) __attribute__((always_inline)) {
        const int key0 = start + tile * kNarrowTile;
        if (key0 < lo) { // values before the first key count as zero, whatever they are
#pragma unroll
            for (int s = 0; s < 2; ++s) {
#pragma unroll
                for (int i = 0; i < S::kSteps; ++i) {
                    if (key0 + 16 * s + pieces.key(i) < lo) {
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
        float4_t score[CT][2];
#pragma unroll
        for (int c = 0; c < CT; ++c) {
            score[c][0] = score[c][1] = float4_t{0.0f, 0.0f, 0.0f, 0.0f};
        }
#pragma unroll
        for (int i = 0; i < S::kSteps; ++i) {
#pragma unroll
            for (int s = 0; s < 2; ++s) {
                const uint4 kk = *reinterpret_cast<const uint4 *>(lds + k_lds + s * 16 * S::kRowBytes + 64 * i);
#pragma unroll
                for (int c = 0; c < CT; ++c) {
                    score[c][s] = T::mfma16(kk, __builtin_bit_cast(uint4, q[c][i]), score[c][s]);
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
        if (tile + kTilesAhead < k.tile1) {
            request(tile + kTilesAhead, k_reg, v_reg);
        }
        u32x4_t upper[CT], lower[CT];
#pragma unroll
        for (int c = 0; c < CT; ++c) {
            float p[8];
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                p[e] = score[c][e >> 2][e & 3] * c_scale;
            }
            if (key0 < lo || key0 + kNarrowTile > hi) {
#pragma unroll
                for (int e = 0; e < 8; ++e) {
                    const int key = key0 + 16 * (e >> 2) + 4 * quad + (e & 3);
                    p[e] = key >= lo && key < hi ? p[e] : -INFINITY;
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
                uint32_t u, v;
                split<T>(float2_t{p[2 * e], p[2 * e + 1]}, u, v);
                upper[c][e] = u, lower[c][e] = v;
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
#pragma unroll
            for (int c = 0; c < CT; ++c) {
                o[c][i] = T::mfma16(vt, __builtin_bit_cast(uint4, upper[c]), o[c][i]);
                o[c][i] = T::mfma16(vt, __builtin_bit_cast(uint4, lower[c]), o[c][i]);
            }
        }
    };
#pragma unroll
    for (int i = 0; i < kTilesAhead; ++i) {
        if (k.tile0 + i < k.tile1) {
            request(k.tile0 + i, k_reg[i], v_reg[i]);
        }
    }
#pragma unroll 1
    for (int tile = k.tile0; tile < k.tile1; tile += kTilesAhead) {
#pragma unroll
        for (int i = 0; i < kTilesAhead; ++i) {
            if (i == 0 || tile + i < k.tile1) {
                step(tile + i, k_reg[i], v_reg[i]);
            }
        }
    }

    const SharedParts parts = carve_parts(a.workspace, shared_columns(a.rows, a.q_heads, a.groups));
#pragma unroll
    for (int c = 0; c < CT; ++c) {
        const int column = 16 * c + col;
        l[c] += __shfl_xor(l[c], 16);
        l[c] += __shfl_xor(l[c], 32);
        if (column < columns) {
#pragma unroll
            for (int i = 0; i < S::kDTiles; ++i) {
                *reinterpret_cast<float4_t *>(parts.o + (k.part + column) * D + 16 * i + 4 * quad) = o[c][i];
            }
            if (quad == 0) {
                parts.stats[k.part + column] = make_float2(m[c], poisoned ? NAN : l[c]);
            }
        }
    }
}

// Two weights, each as an upper half cut off below it and a lower one that is rounded: less work than split(), for products that bound the time. The lower half has
// 2^-23 of the weight too much, so that it is positive even where the upper one is exact: an infinite value then gives an infinite output.
template <class T> struct Halves;
template <> struct Halves<BF16> {
    static __device__ __forceinline__ void split(float2_t p, uint32_t &upper, uint32_t &lower) {
        const uint32_t p0 = __float_as_uint(p[0]), p1 = __float_as_uint(p[1]);
        upper = __builtin_amdgcn_perm(p1, p0, 0x07060302u);
        const float2_t rest{__builtin_fmaf(p[0], 1.0f + 0x1p-23f, -__uint_as_float(p0 & 0xFFFF0000u)),
                            __builtin_fmaf(p[1], 1.0f + 0x1p-23f, -__uint_as_float(p1 & 0xFFFF0000u))};
        lower = __builtin_bit_cast(uint32_t, __builtin_convertvector(rest, Split<BF16>::pair_t));
    }
};
template <> struct Halves<F16> {
    static __device__ __forceinline__ void split(float2_t p, uint32_t &upper, uint32_t &lower) {
        const Split<F16>::pair_t cut = __builtin_bit_cast(Split<F16>::pair_t, __builtin_amdgcn_cvt_pkrtz(p[0], p[1]));
        upper = __builtin_bit_cast(uint32_t, cut);
        const float2_t rest{__builtin_fmaf(p[0], 1.0f + 0x1p-23f, -static_cast<float>(cut[0])), __builtin_fmaf(p[1], 1.0f + 0x1p-23f, -static_cast<float>(cut[1]))};
        lower = __builtin_bit_cast(uint32_t, __builtin_convertvector(rest, Split<F16>::pair_t));
    }
};

// Rows of keys and values in LDS as transfers leave them, without padding: 16-byte piece c of row r lies at piece c ^ key(r) or c ^ value(r) of its row, so that
// the pieces that 16 lanes read at a time of 16 rows (keys), and 32 or 16 lanes of 4 rows (values), lie in different banks.
template <int D> struct Swizzle {
    static constexpr int kPerRow = D / 8;
    // Operands whose addresses are not a constant apart.
    static constexpr int kKeys = D == 64 ? 4 : D == 96 ? 2 : 8, kValues = D == 64 ? 2 : D == 96 ? 1 : 4;
    static __device__ __forceinline__ int key(int r) { return D == 64 ? (r >> 1) & 7 : D == 96 ? (r >> 2) & 3 : r & 15; }
    static __device__ __forceinline__ int value(int r) { return D == 64 ? 2 * (r & 3) : D == 96 ? r & 2 : 4 * (r & 1) + 5 * (r & 2); }
};

typedef float float16_t __attribute__((ext_vector_type(16)));

// 32 x 32 x 16: lane L has row (or column) L & 31 of the operands, elements 8 (L >> 5) on; of the result column L & 31, rows 8 (i / 4) + 4 (L >> 5) + i % 4.
template <class T> __device__ __forceinline__ float16_t mfma32(uint4 x, uint4 y, float16_t c);
template <> __device__ __forceinline__ float16_t mfma32<F16>(uint4 x, uint4 y, float16_t c) {
    return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(half8_t, x), __builtin_bit_cast(half8_t, y), c, 0, 0, 0);
}
template <> __device__ __forceinline__ float16_t mfma32<BF16>(uint4 x, uint4 y, float16_t c) {
    return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8_t, x), __builtin_bit_cast(bf16x8_t, y), c, 0, 0, 0);
}

// N transfers of lds_dma16 to 1024 bytes each, without the compiler's knowledge: it would have every read of the ring wait for all transfers to it, and which are
// done is counted here. Bytes and addresses are uniform; `to` is an LDS address. M0, which the compiler does not let be named as changed, is left as it was.
// A vector instruction may write the resource right before (the compiler gets spilled scalars back that way), and a load may read it 5 cycles later: the block waits.
template <int N> __device__ __forceinline__ void ring_transfer(u32x4_t resource, uint32_t to, const uint32_t *offset) {
    static_assert(N >= 2 && N <= 4, "of the heads' sizes");
#if defined(__HIP_DEVICE_COMPILE__)
    uint32_t before;
#define HM_FIRST "s_mov_b32 %0, m0\n\ts_mov_b32 m0, %1\n\ts_nop 4\n\tbuffer_load_dwordx4 %3, %2, 0 offen lds\n\t"
#define HM_NEXT(OFFSET) "s_add_u32 m0, m0, 0x400\n\ts_nop 0\n\tbuffer_load_dwordx4 " OFFSET ", %2, 0 offen lds\n\t"
#define HM_LAST "s_mov_b32 m0, %0"
    if constexpr (N == 2) {
        asm volatile(HM_FIRST HM_NEXT("%4") HM_LAST : "=&s"(before) : "s"(to), "s"(resource), "v"(offset[0]), "v"(offset[1]) : "memory", "scc");
    } else if constexpr (N == 3) {
        asm volatile(HM_FIRST HM_NEXT("%4") HM_NEXT("%5") HM_LAST
                     : "=&s"(before)
                     : "s"(to), "s"(resource), "v"(offset[0]), "v"(offset[1]), "v"(offset[2])
                     : "memory", "scc");
    } else {
        asm volatile(HM_FIRST HM_NEXT("%4") HM_NEXT("%5") HM_NEXT("%6") HM_LAST
                     : "=&s"(before)
                     : "s"(to), "s"(resource), "v"(offset[0]), "v"(offset[1]), "v"(offset[2]), "v"(offset[3])
                     : "memory", "scc");
    }
#undef HM_FIRST
#undef HM_NEXT
#undef HM_LAST
#else
    (void)resource, (void)to, (void)offset;
#endif
}

// Tiles of keys and values on the way or in use at once. In step n the first product takes the keys of tile n + 1, the second the values of tile n - 1, and the
// weights of tile n are worked out beside them. What tile x brings is asked for kAhead steps before it is needed: keys in step x - 4, values in step x - 2, into
// the places of tiles that were last read in the step before.
constexpr int kRing = 4, kAhead = 3;
template <int D> constexpr int kRingBytes = kRing * 2 * kWideTile * 2 * D;

// A unit of more columns, up to 128: 32 of each wave. The four waves share tiles of 32 keys, of which two waves bring the keys and two the values into LDS,
// 16 rows each. The matrix cores bound it if the vector instructions run beside them, and for that they have to lie between the products in the program: hence the
// steps above. Products of 32 x 32 leave them more room than those of 16 x 16 (three vector instructions for each 16 cycles of a product take 30 % longer
// than the products alone, next to 16 x 16 ones 20 to 60 %).
//   S^T [key, column] = K Q^T     A = K, 16 elements of 32 keys; B = Q^T, in registers
//   O^T [d, column] += V^T P^T    A = V^T, 32 elements of 16 keys, read transposed; B = P^T, as it leaves S^T: keys 16 t + 4 (L >> 5) + j and 8 behind them
template <class T, int D> __device__ __forceinline__ void wide_work(const SharedAttentionArgs &a, const Work &k, uint8_t *ring) {
    using S = Shape<T, D>;
    using Z = Swizzle<D>;
    constexpr int kRow = 2 * D, kPlane = kWideTile * kRow; // a tile's keys, or values
    constexpr int kKeySteps = D / 16, kBlocks = D / 32;    // of the first product, and of the second's rows
    // The maximum follows only when a score passes it by more than a factor 2^kSlack, and is one of the scores before their factor
    // (hm_paged_attention_prompt.hpp). Weights end at 2^Split::kTop all the same, so that values may be as large as in narrow units: fp16 ones have 2^9 at the maximum
    // and lose what is below 2^-33 of it, bf16 ones 2^-16 and 2^-110.
    constexpr float kSlack = Split<T>::kTop > 0.0f ? 6.0f : 16.0f, kTop = Split<T>::kTop - kSlack;
    const int lane = threadIdx.x & 63, wave = uniform(threadIdx.x >> 6);
    const int col = lane & 31, side = lane >> 5;
    const int columns = k.rows * a.group_heads, start = k.s.start() + k.tile0 * kWideTile, lo = k.s.lo, hi = min(k.s.hi, k.s.start() + k.tile1 * kWideTile);
    const int tiles = k.tile1 - k.tile0;
    const Pages at(a, k.s.row0, k.kv_head);

    // ---- pages and queries ----
    int32_t ids[2]; // of 128 sub-tiles of 16 keys from first_id on, a lane each
    int first_id = 0;
    bool poisoned = false; // a page outside the cache
    const auto read_ids = [&](int first) {
        first_id = first;
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            ids[i] = at.page_of(static_cast<uint32_t>(start) + 16 * static_cast<uint32_t>(first + 64 * i + lane), hi);
        }
    };
    const auto check_ids = [&] { poisoned |= __any(static_cast<uint32_t>(ids[0]) >= at.pages || static_cast<uint32_t>(ids[1]) >= at.pages); };
    read_ids(0);
    // The sign goes to the queries. Not zero: a masked score of -infinity times it must stay one.
    const float c_scale = fmaxf(fabsf(a.scale) * 1.4426950408889634f, 0x1p-126f);
    const float slack = fminf(kSlack / c_scale, 0x1p126f); // of scores without the factor
    const uint32_t sign = a.scale < 0.0f ? 0x80008000u : 0u;
    const int column = 32 * wave + col;
    const bool live = column < columns;
    u32x4_t q[kKeySteps];
    {
        const int row = column / a.group_heads;
        const uint16_t *q_row =
            a.q + (live ? (k.s.row0 + k.row + row) * a.ldq + static_cast<int64_t>(k.kv_head * a.group_heads + column - row * a.group_heads) * D : 0) + 8 * side;
#pragma unroll
        for (int i = 0; i < kKeySteps; ++i) {
            q[i] = live ? *reinterpret_cast<const u32x4_t *>(q_row + 16 * i) ^ sign : u32x4_t{0, 0, 0, 0};
        }
    }
    check_ids();
    wait_vmcnt<0>(); // from here on only transfers are on the way

    // ---- transfers: the wave's 16 rows of keys (waves 0 and 1) or values ----
    const bool of_values = wave >= 2;
    const int sub = wave & 1;
    uint32_t from[S::kSteps]; // piece j * 64 + lane of the rows is the lane's of transfer j
#pragma unroll
    for (int j = 0; j < S::kSteps; ++j) {
        const int r = (j * 64 + lane) / Z::kPerRow, c = (j * 64 + lane) % Z::kPerRow;
        from[j] = r * at.row_bytes + (c ^ (of_values ? Z::value(r) : Z::key(16 * sub + r))) * 16;
    }
    const uint16_t *head = of_values ? at.v_head : at.k_head;
    const uint32_t ring_at = static_cast<uint32_t>(reinterpret_cast<uintptr_t>((__attribute__((address_space(3))) void *)ring)) + (of_values ? kPlane : 0) + sub * 16 * kRow;
    const auto transfer = [&](int tile) { // zeros behind the last key, also of tiles that there are not: the counts stay what they are
        const int key = start + tile * kWideTile + 16 * sub, i = 2 * tile + sub - first_id;
        const int32_t page = i < 64 ? __builtin_amdgcn_readlane(ids[0], i) : __builtin_amdgcn_readlane(ids[1], i & 63);
        const int seen = static_cast<uint32_t>(page) < at.pages ? max(0, min(16, hi - key)) : 0;
        const uint64_t address = reinterpret_cast<uint64_t>(head + at.offset(page, key, seen));
        const u32x4_t resource{static_cast<uint32_t>(uniform(static_cast<int>(address))), static_cast<uint32_t>(uniform(static_cast<int>(address >> 32))) & 0xFFFFu,
                               at.bytes<D>(seen), 0x00020000u};
        constexpr int kAtOnce = S::kSteps < 4 ? S::kSteps : 4;
#pragma unroll
        for (int j = 0; j < S::kSteps; j += kAtOnce) {
            ring_transfer<kAtOnce>(resource, ring_at + (tile % kRing) * 2 * kPlane + j * 1024, from + j);
        }
    };
#pragma unroll
    for (int x = 0; x < kAhead + 1; ++x) { // as if in steps -4 to -1
        if (!of_values || x >= kAhead - 1) {
            transfer(of_values ? x - 2 : x);
        }
    }

    // ---- operands' addresses, and what is summed up ----
    uint32_t k_lds[Z::kKeys], v_lds[Z::kValues];
#pragma unroll
    for (int i = 0; i < Z::kKeys; ++i) {
        k_lds[i] = col * kRow + ((2 * i + side) ^ Z::key(col)) * 16;
    }
#pragma unroll
    for (int i = 0; i < Z::kValues; ++i) {
        const int r = 4 * side + ((lane & 15) >> 2);
        v_lds[i] = kPlane + r * kRow + ((4 * i + 2 * (lane >> 4 & 1) + ((lane & 3) >> 1)) ^ Z::value(r)) * 16 + (lane & 1) * 8;
    }
    float16_t o[kBlocks];
#pragma unroll
    for (int i = 0; i < kBlocks; ++i) {
        o[i] = float16_t{};
    }
    float m = -INFINITY, l = 0.0f;
    struct Weights {
        u32x4_t upper[2], lower[2];
    };
    const auto first_product = [&](int place, float16_t &score) __attribute__((always_inline)) {
        score = float16_t{};
#pragma unroll
        for (int i = 0; i < kKeySteps; ++i) {
            const uint4 kk = *reinterpret_cast<const uint4 *>(ring + place * 2 * kPlane + k_lds[i % Z::kKeys] + i / Z::kKeys * Z::kKeys * 32);
            score = mfma32<T>(kk, __builtin_bit_cast(uint4, q[i]), score);
        }
    };
    const auto second_product = [&](int place, const Weights &w) __attribute__((always_inline)) {
#pragma unroll
        for (int t = 0; t < 2; ++t) {
#pragma unroll
            for (int i = 0; i < kBlocks; ++i) {
                uint2 half[2];
#pragma unroll
                for (int s = 0; s < 2; ++s) {
                    half[s] = lds_read_transposed(ring + place * 2 * kPlane + v_lds[i % Z::kValues] + (16 * t + 8 * s) * kRow + i / Z::kValues * Z::kValues * 64);
                }
                const uint4 vt = make_uint4(half[0].x, half[0].y, half[1].x, half[1].y);
                o[i] = mfma32<T>(vt, __builtin_bit_cast(uint4, w.upper[t]), o[i]);
                o[i] = mfma32<T>(vt, __builtin_bit_cast(uint4, w.lower[t]), o[i]);
            }
        }
    };
    const auto clear_before = [&] { // values before the first key count as zero, whatever they are
        if (lo > start && wave == 2) {
            for (int j = lane; j < (lo - start) * Z::kPerRow; j += 64) {
                *reinterpret_cast<u32x4_t *>(ring + kPlane + j * 16) = u32x4_t{0, 0, 0, 0};
            }
        }
    };
    const bool works = 32 * wave < columns;
    // Step n, with n % kRing = place: scores of tile n in `score`, weights of tile n - 1 in `before`; leaves those of n + 1 and n.
    const auto step = [&](auto first, int n, auto place, float16_t &score, float16_t &next, Weights &before, Weights &weights) __attribute__((always_inline)) {
        constexpr bool kFirst = decltype(first)::value; // tile 0: there is none before
        constexpr int kPlace = decltype(place)::value;
        wait_vmcnt<(kAhead - 1) * S::kSteps>(); // the wave's transfers that this step needs are done, those of two steps may be on the way
        if (n == 1) {
            clear_before();
        }
        lds_barrier();
        const int wanted = n + (of_values ? kAhead - 1 : kAhead + 1);
        if (2 * (wanted + 1) - first_id > 128) { // seldom: the pages of the next 60 tiles
            read_ids(2 * (n + kAhead - 1));
            check_ids();
            wait_vmcnt<0>();
        }
        transfer(wanted);
        if (!works) {
            return;
        }
        const int key0 = start + n * kWideTile;
        if (key0 < lo || key0 + kWideTile > hi) {
            __builtin_amdgcn_sched_barrier(0); // keeps this a branch
#pragma unroll
            for (int e = 0; e < 16; ++e) {
                const int key = key0 + 8 * (e >> 2) + 4 * side + (e & 3);
                score[e] = key < lo || key >= hi ? -INFINITY : score[e];
            }
        }
        float top = score[0];
#pragma unroll
        for (int e = 1; e < 16; ++e) {
            top = fmaxf(top, score[e]);
        }
        if (__any(top > m + slack)) {
            if constexpr (!kFirst) { // what is on the way is relative to the old maximum
                second_product((kPlace + kRing - 1) % kRing, before);
                before = Weights{};
            }
            top = fmaxf(top, __shfl_xor(top, 32));
            const float m_new = fmaxf(m, top);
            const float f = m_new == -INFINITY ? 1.0f : exp2_fast((m - m_new) * c_scale);
            m = m_new;
            l *= f;
#pragma unroll
            for (int i = 0; i < kBlocks; ++i) {
                o[i] *= f;
            }
        }
        first_product((kPlace + 1) % kRing, next); // behind the last tile: of zeros
        const float m_used = m == -INFINITY ? 0.0f : m;
#pragma unroll
        for (int e = 0; e < 16; e += 2) {
            float2_t p;
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                p[i] = exp2_fast(__builtin_fmaf(score[e + i] - m_used, c_scale, kTop));
                l += p[i];
            }
            uint32_t u, v;
            Halves<T>::split(p, u, v);
            weights.upper[e >> 3][(e & 7) / 2] = u, weights.lower[e >> 3][(e & 7) / 2] = v;
        }
        if constexpr (!kFirst) {
            second_product((kPlace + kRing - 1) % kRing, before);
        }
    };
    float16_t score_even, score_odd;
    Weights even{}, odd{};
    wait_vmcnt<kAhead * S::kSteps>(); // of keys: those of the first tile; of values: no more are on the way
    lds_barrier();
    if (works) {
        first_product(0, score_even);
    }
    step(std::true_type{}, 0, std::integral_constant<int, 0>{}, score_even, score_odd, odd, even);
#pragma unroll 1
    for (int n = 1; n < tiles; n += kRing) {
        step(std::false_type{}, n, std::integral_constant<int, 1>{}, score_odd, score_even, even, odd);
        if (n + 1 < tiles) {
            step(std::false_type{}, n + 1, std::integral_constant<int, 2>{}, score_even, score_odd, odd, even);
        }
        if (n + 2 < tiles) {
            step(std::false_type{}, n + 2, std::integral_constant<int, 3>{}, score_odd, score_even, even, odd);
        }
        if (n + 3 < tiles) {
            step(std::false_type{}, n + 3, std::integral_constant<int, 0>{}, score_even, score_odd, odd, even);
        }
    }
    wait_vmcnt<0>();
    if (tiles == 1) {
        clear_before();
    }
    lds_barrier();
    if (works) {
        second_product((tiles - 1) % kRing, (tiles & 1) != 0 ? even : odd);
    }

    const SharedParts parts = carve_parts(a.workspace, shared_columns(a.rows, a.q_heads, a.groups));
    l += __shfl_xor(l, 32);
    if (live) {
#pragma unroll
        for (int i = 0; i < kBlocks; ++i) {
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                *reinterpret_cast<float4_t *>(parts.o + (k.part + column) * D + 32 * i + 8 * e + 4 * side) =
                    float4_t{o[i][4 * e], o[i][4 * e + 1], o[i][4 * e + 2], o[i][4 * e + 3]};
            }
        }
        if (side == 0) {
            // relative to the maximum as narrow units have it: with the factor, and with weights from 2^Split::kTop down
            parts.stats[k.part + column] = make_float2(m * c_scale + (Split<T>::kTop - kTop), poisoned ? NAN : l);
        }
    }
    lds_barrier(); // the next unit takes the ring
}

// The first workgroups have a run of the wide line each, which the matrix cores bound; the waves of the others one each of the narrow line, which the
// memory bounds. Where both are half, a CU has a workgroup of each.
template <class T, int D> __global__ void __launch_bounds__(kThreads, D <= 128 ? 2 : 1) shared_attention_kernel(SharedAttentionArgs a) {
    using S = Shape<T, D>;
    __shared__ __attribute__((aligned(1024))) uint8_t lds[kRingBytes<D>];
    static_assert(kAttentionWaves * S::kRegion <= kRingBytes<D>, "narrow units' regions take the place of the ring");
    const ShareWorkspace plan = carve_share(a.plan, a.rows, a.groups);
    const int wave = uniform(threadIdx.x >> 6);
    const ShareHeader header = *plan.header;
    if (!header.fits(a.rows, a.group_heads, a.kv_heads, a.groups)) {
        return;
    }
    const int wide = uniform(header.wide), group = static_cast<int>(blockIdx.x) - wide;
    if (group < 0) {
        const Runs runs = Runs::deal(uniform(header.tiles[1]), wide);
        // Runs that follow each other go to one XCD: those of a key head's chunks of rows read the same keys at the same time, and its L2 has them for all.
        const int xcd = blockIdx.x % a.xcds, w = xcd * (wide / a.xcds) + min(xcd, wide % a.xcds) + static_cast<int>(blockIdx.x / a.xcds), x_end = runs.begin(w + 1);
        int x = runs.begin(w);
        Segments segments(plan.segments[1], uniform(plan.starts[1][w]));
        while (x < x_end) {
            wide_work<T, D>(a, next_work<1>(a, segments, x, x_end, w), lds);
        }
        return;
    }
    const int groups = a.groups - wide, w = wave * groups + group; // few runs go to as many workgroups
    if (w >= uniform(header.narrow)) {
        return;
    }
    const Runs runs = Runs::deal(uniform(header.tiles[0]), uniform(header.narrow));
    const int x_end = runs.begin(w + 1);
    int x = runs.begin(w);
    if (x == x_end) {
        return;
    }
    Segments segments(plan.segments[0], uniform(plan.starts[0][w]));
    PageIds ids;
    while (x < x_end) {
        const Work k = next_work<0>(a, segments, x, x_end, w);
        if (k.rows * a.group_heads <= 16) {
            narrow_work<T, D, 1>(a, k, lds + wave * S::kRegion, ids);
        } else {
            narrow_work<T, D, 2>(a, k, lds + wave * S::kRegion, ids);
        }
    }
}

// Columns joined, by THREADS threads each: the parts of the segments on the row's path, each of the runs that its unit lies in.
template <class T, int D, int THREADS> __global__ void __launch_bounds__(256) shared_join_kernel(SharedAttentionArgs a) {
    constexpr int kItems = D / 4, kLanes = THREADS / kItems, kAhead = 4, kColumns = 256 / THREADS;
    __shared__ float4_t acc[kColumns][kLanes][kItems];
    __shared__ float2 stat[kColumns][kLanes];
    const int mine = THREADS == 64 ? uniform(threadIdx.x >> 6) : 0, thread = threadIdx.x % THREADS;
    const uint32_t column = blockIdx.x * kColumns + mine; // rows and heads are below 2^12 and 2^17
    const int64_t t = column / static_cast<uint32_t>(a.q_heads);
    if (t >= a.rows) {
        return;
    }
    const int head = static_cast<int>(column - static_cast<uint32_t>(t) * a.q_heads), kv_head = head / a.group_heads, in_group = head - kv_head * a.group_heads;
    const ShareWorkspace plan = carve_share(a.plan, a.rows, a.groups);
    const ShareHeader header = *plan.header;
    const int lane = threadIdx.x & 63;
    const SharePath p = plan.paths[min(lane, kPathEntries - 1) * a.rows + t];
    const Keys keys = keys_of(a, t);
    if (keys.request < 0) {
        return;
    }
    // The parts of each segment's unit, a lane each: of runs w0, w0 + 1 and so on, the last one at `end`.
    int own_count = 0;
    int64_t own_first = 0, own_end = 0;
    if (lane < kPathEntries && p.tiles > 0 && header.fits(a.rows, a.group_heads, a.kv_heads, a.groups)) {
        const Runs runs = Runs::deal(p.line == 0 ? header.tiles[0] : header.tiles[1], header.runs(p.line));
        const int tile = p.tile + kv_head * p.per_head, w0 = runs.of(tile);
        own_count = runs.of(tile + p.tiles - 1) - w0 + 1;
        own_first = run_column(a.rows, a.q_heads, a.groups, p.line, w0) + p.in_chunk * a.group_heads + in_group;
        own_end = static_cast<int64_t>(p.slot0) * a.q_heads + (static_cast<int64_t>(kv_head) * p.rows + p.row) * a.group_heads + in_group;
    }
    const auto of64 = [](int64_t v, int i) {
        const uint32_t low = __builtin_amdgcn_readlane(static_cast<uint32_t>(v), i), high = __builtin_amdgcn_readlane(static_cast<uint32_t>(static_cast<uint64_t>(v) >> 32), i);
        return static_cast<int64_t>(static_cast<uint64_t>(high) << 32 | low);
    };
    int count[kPathEntries], step[kPathEntries], total = 0;
    int64_t first[kPathEntries], end[kPathEntries];
#pragma unroll
    for (int i = 0; i < kPathEntries; ++i) {
        count[i] = __builtin_amdgcn_readlane(own_count, i);
        step[i] = cols_of(__builtin_amdgcn_readlane(p.line, i));
        first[i] = of64(own_first, i), end[i] = of64(own_end, i);
        total += count[i];
    }
    const auto column_of = [&](int part) {
        int64_t at = 0;
#pragma unroll
        for (int i = 0; i < kPathEntries; ++i) {
            if (part >= 0 && part < count[i]) {
                at = part == count[i] - 1 ? end[i] : first[i] + part * step[i];
            }
            part -= count[i];
        }
        return at;
    };
    const SharedParts parts = carve_parts(a.workspace, shared_columns(a.rows, a.q_heads, a.groups));
    const int y = thread / kItems, e = thread - y * kItems;
    float m = -INFINITY, l = 0.0f;
    float4_t v = float4_t{0.0f, 0.0f, 0.0f, 0.0f};
    if (y < kLanes) {
        for (int i = y; i < total; i += kAhead * kLanes) {
            float2 st[kAhead];
            float4_t o[kAhead];
            float top = m;
#pragma unroll
            for (int n = 0; n < kAhead; ++n) {
                const int64_t from = column_of(min(i + n * kLanes, total - 1));
                st[n] = parts.stats[from];
                o[n] = *reinterpret_cast<const float4_t *>(parts.o + from * D + 4 * e);
            }
#pragma unroll
            for (int n = 0; n < kAhead; ++n) {
                top = fmaxf(top, st[n].x); // the last part may count twice here
            }
            const float from = top == -INFINITY ? 0.0f : top; // no finite score yet: weights of zero
            const float f = exp2_fast(m - from);
            v *= f;
            l *= f;
#pragma unroll
            for (int n = 0; n < kAhead; ++n) {
                if (i + n * kLanes < total) {
                    const float g = exp2_fast(st[n].x - from);
                    v += o[n] * g;
                    l += st[n].y * g;
                }
            }
            m = top;
        }
        acc[mine][y][e] = v;
        if (e == 0) {
            stat[mine][y] = make_float2(m, l);
        }
    }
    if constexpr (THREADS > 64) {
        __syncthreads();
    } else {
        __builtin_amdgcn_wave_barrier(); // a wave's LDS accesses are carried out in order
    }
    if (y == 0) {
        float top = -INFINITY, sum = 0.0f;
        float4_t all = float4_t{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
        for (int i = 0; i < kLanes; ++i) {
            top = fmaxf(top, stat[mine][i].x);
        }
#pragma unroll
        for (int i = 0; i < kLanes; ++i) {
            const float f = exp2_fast(stat[mine][i].x - (top == -INFINITY ? 0.0f : top));
            all += acc[mine][i][e] * f;
            sum += stat[mine][i].y * f;
        }
        const float over = keys.bad ? NAN : keys.end == 0 ? 1.0f : sum; // a row that sees no key is zero
        store4<T>(a.out + t * a.ldo + static_cast<int64_t>(head) * D + 4 * e, all / over);
    }
}

template <class T, int D> hipError_t launch_shared(const SharedAttentionArgs &a, hipStream_t stream) {
    hipLaunchKernelGGL((shared_attention_kernel<T, D>), dim3(static_cast<unsigned>(a.groups)), dim3(kThreads), 0, stream, a);
    const hipError_t e = hipGetLastError();
    if (e != hipSuccess) {
        return e;
    }
    // A wave per column where there are enough columns for the card: 128 columns of 1088 keys 11.7 us by workgroups and 14.7 by waves, 512 of 2112 16.4 and 17.0, 1024
    // 21.0 and 18.7, 2048 of 2304 32.5 and 29.1.
    const int64_t columns = a.rows * a.q_heads;
    if (D == 256 || columns <= a.groups) {
        hipLaunchKernelGGL((shared_join_kernel<T, D, 256>), dim3(static_cast<unsigned>(columns)), dim3(256), 0, stream, a);
    } else {
        hipLaunchKernelGGL((shared_join_kernel<T, D, D == 256 ? 256 : 64>), dim3(static_cast<unsigned>((columns + 3) / 4)), dim3(256), 0, stream, a);
    }
    return hipGetLastError();
}

template <class T> hipError_t launch_shared_t(const SharedAttentionArgs &a, hipStream_t stream) {
    switch (a.head_dim) {
    case 64:
        return launch_shared<T, 64>(a, stream);
    case 96:
        return launch_shared<T, 96>(a, stream);
    case 128:
        return launch_shared<T, 128>(a, stream);
    default:
        return launch_shared<T, 256>(a, stream);
    }
}

} // namespace
} // namespace hm
