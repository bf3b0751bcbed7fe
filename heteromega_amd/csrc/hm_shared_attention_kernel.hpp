// Attention over shared pages: the kernels (hm_shared_attention.hip has the mathematics and the launch rules). They take the tiles' shapes, loads and
// weights from hm_paged_attention_kernel.hpp.
#pragma once

#include "hm_paged_attention_kernel.hpp"
#include "hm_shared_attention.hpp"

namespace hm {
namespace {

// The segment that tile x of a line lies in, found by 64 lanes at a time: the last one that begins at x or before it.
__device__ __forceinline__ int segment_at(const ShareSegment *segments, int count, int x) {
    const int lane = threadIdx.x & 63;
    int from = 0;
    while (count > 1) {
        const int step = (count + 63) / 64, at = lane * step;
        const uint64_t who = __ballot(at < count && segments[from + min(at, count - 1)].tile0 <= x); // lane 0's always does
        const int last = 63 - static_cast<int>(__builtin_clzll(who | 1));
        from += last * step;
        count = min(step, count - last * step);
    }
    return uniform(from);
}

__device__ __forceinline__ ShareSegment uniform_segment(const ShareSegment *p) {
    const ShareSegment s = *p;
    return {uniform(s.row0), uniform(s.rows), uniform(s.lo), uniform(s.hi), uniform(s.tile0), uniform(s.tiles), uniform(s.slot0), uniform(s.chunk)};
}

__device__ __forceinline__ bool fits(const ShareWorkspace &plan, const SharedAttentionArgs &a) {
    return plan.header->rows == static_cast<int32_t>(a.rows) && plan.header->group_heads == a.group_heads && plan.header->kv_heads == a.kv_heads;
}

// A unit's tiles [tile0, tile1) as a workgroup works on them.
struct Work {
    ShareSegment s;
    int kv_head, row, rows; // row: first, behind the segment's
    int tile0, tile1;
    int64_t part; // its first column among the parts
};

// The next work of a run [x, x_end) of a line; moves x on.
template <int LINE> __device__ __forceinline__ Work next_work(const SharedAttentionArgs &a, const ShareSegment *segments, int &at, int &x, int x_end, int w) {
    Work k;
    k.s = uniform_segment(segments + at);
    const int chunks = LINE == 0 ? 1 : k.s.chunks();
    const int unit = uniform(static_cast<uint32_t>(x - k.s.tile0) / static_cast<uint32_t>(k.s.tiles));
    k.kv_head = LINE == 0 ? unit : unit / chunks;
    k.row = LINE == 0 ? 0 : (unit - k.kv_head * chunks) * k.s.chunk;
    k.rows = min(k.s.chunk, k.s.rows - k.row);
    k.tile0 = x - k.s.tile0 - unit * k.s.tiles;
    k.tile1 = min(k.s.tiles, k.tile0 + (x_end - x));
    k.part = k.tile1 == k.s.tiles ? static_cast<int64_t>(k.s.slot0) * a.q_heads + (static_cast<int64_t>(k.kv_head) * k.s.rows + k.row) * a.group_heads
                                  : run_column(a.rows, a.q_heads, a.runs, LINE, w);
    x += k.tile1 - k.tile0;
    at += k.tile1 == k.s.tiles && unit + 1 == a.kv_heads * chunks;
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

    __device__ __forceinline__ int32_t page_of(int key, int hi) const { return key >= hi ? 0 : there && key < capacity ? table[key >> shift] : -1; }
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

// A unit of up to 16 columns: each of the four waves takes 32 keys of a tile, and the waves join over LDS.
template <class T, int D> __device__ __forceinline__ void narrow_work(const SharedAttentionArgs &a, const Work &k, uint8_t *lds, float2 (&wave_stats)[kAttentionWaves][16]) {
    using S = Shape<T, D>;
    const int lane = threadIdx.x & 63, wave = uniform(threadIdx.x >> 6);
    const int col = lane & 15, quad = lane >> 4;
    const int columns = k.rows * a.group_heads, start = k.s.start(), lo = k.s.lo, hi = k.s.hi;
    const Pages at(a, k.s.row0, k.kv_head);
    const Pieces<D> pieces(lane, at.row_bytes);
    const uint32_t to_lds = wave * S::kRegion + pieces.lds_offset();
    const uint32_t k_lds = wave * S::kRegion + col * S::kRowBytes + quad * 16;
    const uint32_t v_lds = wave * S::kRegion + (4 * quad + (col >> 2)) * S::kRowBytes + (col & 3) * 8;
    const float c_scale = a.scale * 1.4426950408889634f;

    u32x4_t q[S::kSteps];
    const int row = col / a.group_heads;
    const bool live = col < columns;
    const uint16_t *q_row = a.q + (live ? (k.s.row0 + row) * a.ldq + static_cast<int64_t>(k.kv_head * a.group_heads + col - row * a.group_heads) * D : 0) + 8 * quad;
#pragma unroll
    for (int s = 0; s < S::kSteps; ++s) {
        q[s] = live ? *reinterpret_cast<const u32x4_t *>(q_row + 32 * s) : u32x4_t{0, 0, 0, 0};
    }
    float4_t o[S::kDTiles];
#pragma unroll
    for (int i = 0; i < S::kDTiles; ++i) {
        o[i] = float4_t{0.0f, 0.0f, 0.0f, 0.0f};
    }
    float m = -INFINITY, l = 0.0f;
    bool poisoned = false; // a page outside the cache

    u32x4_t k_reg[2][S::kSteps], v_reg[2][S::kSteps];
    int32_t id[2];
    const auto page_ids = [&](int tile) {
#pragma unroll
        for (int s = 0; s < 2; ++s) {
            const int key = start + tile * kNarrowTile + wave * kWaveKeys + 16 * s;
            id[s] = at.page_of(key, hi);
        }
    };
    const auto request = [&](int tile) {
#pragma unroll
        for (int s = 0; s < 2; ++s) {
            const int key = start + tile * kNarrowTile + wave * kWaveKeys + 16 * s;
            const int32_t page = uniform(id[s]);
            int seen = max(0, min(16, hi - key));
            if (static_cast<uint32_t>(page) >= at.pages) {
                poisoned |= seen > 0;
                seen = 0;
            }
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
    page_ids(k.tile0);
    request(k.tile0);
    page_ids(min(k.tile0 + 1, k.tile1 - 1));
    for (int tile = k.tile0; tile < k.tile1; ++tile) {
        const int key0 = start + tile * kNarrowTile + wave * kWaveKeys;
        if (key0 >= hi) {
            break; // only the segment's last tile has waves without keys
        }
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
        float4_t score[2] = {float4_t{0.0f, 0.0f, 0.0f, 0.0f}, float4_t{0.0f, 0.0f, 0.0f, 0.0f}};
#pragma unroll
        for (int i = 0; i < S::kSteps; ++i) {
#pragma unroll
            for (int s = 0; s < 2; ++s) {
                const uint4 kk = *reinterpret_cast<const uint4 *>(lds + k_lds + s * 16 * S::kRowBytes + 64 * i);
                score[s] = T::mfma16(kk, __builtin_bit_cast(uint4, q[i]), score[s]);
            }
        }
#pragma unroll
        for (int s = 0; s < 2; ++s) {
#pragma unroll
            for (int i = 0; i < S::kSteps; ++i) {
                *reinterpret_cast<u32x4_t *>(lds + to_lds + pieces.lds_step(i) + s * 16 * S::kRowBytes) = v_reg[s][i];
            }
        }
        if (tile + 1 < k.tile1) {
            request(tile + 1);
            page_ids(min(tile + 2, k.tile1 - 1));
        }
        float p[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            p[e] = score[e >> 2][e & 3] * c_scale;
        }
        if (key0 < lo || key0 + kWaveKeys > hi) {
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                const int key = key0 + 16 * (e >> 2) + 4 * quad + (e & 3);
                p[e] = key >= lo && key < hi ? p[e] : -INFINITY;
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
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            p[e] = exp2_fast(p[e] - m_used);
            l += p[e];
        }
        u32x4_t upper, lower;
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            uint32_t u, v;
            split<T>(float2_t{p[2 * e], p[2 * e + 1]}, u, v);
            upper[e] = u, lower[e] = v;
        }
#pragma unroll
        for (int i = 0; i < S::kDTiles; ++i) {
            uint2 half[2];
#pragma unroll
            for (int s = 0; s < 2; ++s) {
                half[s] = lds_read_transposed(lds + v_lds + s * 16 * S::kRowBytes + i * 32);
            }
            const uint4 vt = make_uint4(half[0].x, half[0].y, half[1].x, half[1].y);
            o[i] = T::mfma16(vt, __builtin_bit_cast(uint4, upper), o[i]);
            o[i] = T::mfma16(vt, __builtin_bit_cast(uint4, lower), o[i]);
        }
    }

    // ---- the waves' parts joined ----
    const SharedParts parts = carve_parts(a.workspace, shared_columns(a.rows, a.q_heads, a.runs));
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
        for (int i = 0; i < kAttentionWaves; ++i) {
            top = fmaxf(top, wave_stats[i][col].x);
        }
        const float f = top == -INFINITY ? 0.0f : exp2_fast(m - top);
        float *mine = reinterpret_cast<float *>(lds + wave * S::kRegion);
        if (live) {
#pragma unroll
            for (int i = 0; i < S::kDTiles; ++i) {
                *reinterpret_cast<float4_t *>(mine + col * S::kORow + 16 * i + 4 * quad) = o[i] * f;
            }
        }
    }
    __syncthreads();
    for (int i = threadIdx.x; i < columns * (D / 4); i += kThreads) {
        const int j = i / (D / 4), d = (i - j * (D / 4)) * 4;
        float top = -INFINITY, sum = 0.0f;
        float4_t v = float4_t{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
        for (int w = 0; w < kAttentionWaves; ++w) {
            top = fmaxf(top, wave_stats[w][j].x);
        }
#pragma unroll
        for (int w = 0; w < kAttentionWaves; ++w) {
            const float2 st = wave_stats[w][j];
            sum += st.y * (top == -INFINITY ? 1.0f : exp2_fast(st.x - top));
            v += *reinterpret_cast<const float4_t *>(reinterpret_cast<const float *>(lds + w * S::kRegion) + j * S::kORow + d);
        }
        *reinterpret_cast<float4_t *>(parts.o + (k.part + j) * D + d) = v;
        if (d == 0) {
            parts.stats[k.part + j] = make_float2(top, sum);
        }
    }
    __syncthreads(); // the next unit takes the regions
}

// A unit of more columns: 16 CT of each wave, up to 128 in all; the waves share tiles of 64 keys, of which each brings a quarter into LDS. Two buffers, one
// barrier a tile.
template <class T, int D, int CT> __device__ __forceinline__ void wide_work(const SharedAttentionArgs &a, const Work &k, uint8_t *lds) {
    using S = Shape<T, D>;
    constexpr int kTileBytes = kWideTile * S::kRowBytes; // of keys, or values
    // The maximum follows only when a score passes it by more than a factor 2^kSlack, and is one of the scores before their factor
    // (hm_paged_attention_prompt.hpp).
    constexpr float kSlack = 3.0f, kTop = Split<T>::kTop - (Split<T>::kTop > 0.0f ? kSlack : 0.0f);
    const int lane = threadIdx.x & 63, wave = uniform(threadIdx.x >> 6);
    const int col = lane & 15, quad = lane >> 4;
    const int columns = k.rows * a.group_heads, start = k.s.start(), lo = k.s.lo, hi = k.s.hi;
    const Pages at(a, k.s.row0, k.kv_head);
    const Pieces<D> pieces(lane, at.row_bytes);
    const uint32_t to_lds = wave * 16 * S::kRowBytes + pieces.lds_offset();
    const uint32_t k_lds = col * S::kRowBytes + quad * 16;
    const uint32_t v_lds = (4 * quad + (col >> 2)) * S::kRowBytes + (col & 3) * 8;
    // The sign goes to the queries. Not zero: a masked score of -infinity times it must stay one.
    const float c_scale = fmaxf(fabsf(a.scale) * 1.4426950408889634f, 0x1p-126f);
    const float slack = fminf(kSlack / c_scale, 0x1p126f); // of scores without the factor
    const uint32_t sign = a.scale < 0.0f ? 0x80008000u : 0u;

    u32x4_t q[CT][S::kSteps];
#pragma unroll
    for (int c = 0; c < CT; ++c) {
        const int j = 16 * (wave * CT + c) + col, row = j / a.group_heads;
        const bool live = j < columns;
        const uint16_t *q_row =
            a.q + (live ? (k.s.row0 + k.row + row) * a.ldq + static_cast<int64_t>(k.kv_head * a.group_heads + j - row * a.group_heads) * D : 0) + 8 * quad;
#pragma unroll
        for (int s = 0; s < S::kSteps; ++s) {
            q[c][s] = live ? *reinterpret_cast<const u32x4_t *>(q_row + 32 * s) ^ sign : u32x4_t{0, 0, 0, 0};
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
    bool poisoned = false; // a page outside the cache

    u32x4_t k_reg[S::kSteps], v_reg[S::kSteps];
    int32_t ids = 0; // of sub-tile lane % 4: a vector load, since waits for LDS would wait for a scalar one too
    const auto page_ids = [&](int tile) {
        const int key = start + tile * kWideTile + 16 * (lane % kAttentionWaves);
        ids = at.page_of(key, hi);
    };
    const auto load = [&](int tile) { // the wave's sub-tile
        poisoned |= __any(static_cast<uint32_t>(ids) >= at.pages);
        const int32_t page = __builtin_amdgcn_readlane(ids, wave);
        const int key = start + tile * kWideTile + 16 * wave;
        const int seen = static_cast<uint32_t>(page) < at.pages ? max(0, min(16, hi - key)) : 0;
        const uint32_t bytes = at.bytes<D>(seen);
        const int64_t from = at.offset(page, key, seen);
        const __amdgpu_buffer_rsrc_t kr = buffer_rsrc(at.k_head + from, bytes), vr = buffer_rsrc(at.v_head + from, bytes);
#pragma unroll
        for (int i = 0; i < S::kSteps; ++i) {
            k_reg[i] = __builtin_amdgcn_raw_buffer_load_b128(kr, pieces.offset(i), 0, 0);
        }
#pragma unroll
        for (int i = 0; i < S::kSteps; ++i) {
            v_reg[i] = __builtin_amdgcn_raw_buffer_load_b128(vr, pieces.offset(i), 0, 0);
        }
    };
    const bool works = 16 * wave * CT < columns;
    page_ids(k.tile0);
    load(k.tile0);
    page_ids(min(k.tile0 + 1, k.tile1 - 1));
    for (int tile = k.tile0; tile < k.tile1; ++tile) {
        const int key0 = start + tile * kWideTile;
        uint8_t *k_tile = lds + (tile & 1) * 2 * kTileBytes, *v_tile = k_tile + kTileBytes;
        if (key0 < lo) { // values before the first key count as zero, whatever they are
#pragma unroll
            for (int i = 0; i < S::kSteps; ++i) {
                if (key0 + 16 * wave + pieces.key(i) < lo) {
                    v_reg[i] = u32x4_t{0, 0, 0, 0};
                }
            }
        }
#pragma unroll
        for (int i = 0; i < S::kSteps; ++i) {
            *reinterpret_cast<u32x4_t *>(k_tile + to_lds + pieces.lds_step(i)) = k_reg[i];
            *reinterpret_cast<u32x4_t *>(v_tile + to_lds + pieces.lds_step(i)) = v_reg[i];
        }
        // The buffer's readers of two tiles ago passed the barrier of the last one.
        __syncthreads();
        if (tile + 1 < k.tile1) {
            load(tile + 1);
            page_ids(min(tile + 2, k.tile1 - 1));
        }
        if (!works) {
            continue;
        }
        const bool some_masked = key0 < lo || key0 + kWideTile > hi;
#pragma unroll
        for (int h = 0; h < 2; ++h) { // 32 keys at a time
            const uint32_t half_lds = h * 32 * S::kRowBytes;
            float4_t score[CT][2];
#pragma unroll
            for (int c = 0; c < CT; ++c) {
                score[c][0] = score[c][1] = float4_t{0.0f, 0.0f, 0.0f, 0.0f};
            }
#pragma unroll
            for (int i = 0; i < S::kSteps; ++i) {
#pragma unroll
                for (int s = 0; s < 2; ++s) {
                    const uint4 kk = *reinterpret_cast<const uint4 *>(k_tile + k_lds + half_lds + s * 16 * S::kRowBytes + 64 * i);
#pragma unroll
                    for (int c = 0; c < CT; ++c) {
                        score[c][s] = T::mfma16(kk, __builtin_bit_cast(uint4, q[c][i]), score[c][s]);
                    }
                }
            }
            u32x4_t upper[CT], lower[CT];
#pragma unroll
            for (int c = 0; c < CT; ++c) {
                if (some_masked) {
                    __builtin_amdgcn_sched_barrier(0); // keeps this a branch
#pragma unroll
                    for (int e = 0; e < 8; ++e) {
                        const int key = key0 + 32 * h + 16 * (e >> 2) + 4 * quad + (e & 3);
                        if (key < lo || key >= hi) {
                            score[c][e >> 2][e & 3] = -INFINITY;
                        }
                    }
                }
                float top = score[c][0][0];
#pragma unroll
                for (int e = 1; e < 8; ++e) {
                    top = fmaxf(top, score[c][e >> 2][e & 3]);
                }
                if (__any(top > m[c] + slack)) {
                    top = fmaxf(top, __shfl_xor(top, 16));
                    top = fmaxf(top, __shfl_xor(top, 32));
                    const float m_new = fmaxf(m[c], top);
                    const float f = m_new == -INFINITY ? 1.0f : exp2_fast((m[c] - m_new) * c_scale);
                    m[c] = m_new;
                    l[c] *= f;
#pragma unroll
                    for (int i = 0; i < S::kDTiles; ++i) {
                        o[c][i] *= f;
                    }
                }
                const float m_used = m[c] == -INFINITY ? 0.0f : m[c];
#pragma unroll
                for (int e = 0; e < 8; e += 2) {
                    float2_t p;
#pragma unroll
                    for (int n = 0; n < 2; ++n) {
                        p[n] = exp2_fast(__builtin_fmaf(score[c][e >> 2][(e & 3) + n] - m_used, c_scale, kTop));
                        l[c] += p[n];
                    }
                    uint32_t u, v;
                    split<T>(p, u, v);
                    upper[c][e / 2] = u, lower[c][e / 2] = v;
                }
            }
#pragma unroll
            for (int i = 0; i < S::kDTiles; ++i) {
                uint2 half[2];
#pragma unroll
                for (int s = 0; s < 2; ++s) {
                    half[s] = lds_read_transposed(v_tile + v_lds + half_lds + s * 16 * S::kRowBytes + i * 32);
                }
                const uint4 vt = make_uint4(half[0].x, half[0].y, half[1].x, half[1].y);
#pragma unroll
                for (int c = 0; c < CT; ++c) {
                    o[c][i] = T::mfma16(vt, __builtin_bit_cast(uint4, upper[c]), o[c][i]);
                    o[c][i] = T::mfma16(vt, __builtin_bit_cast(uint4, lower[c]), o[c][i]);
                }
            }
        }
    }

    const SharedParts parts = carve_parts(a.workspace, shared_columns(a.rows, a.q_heads, a.runs));
#pragma unroll
    for (int c = 0; c < CT; ++c) {
        l[c] += __shfl_xor(l[c], 16);
        l[c] += __shfl_xor(l[c], 32);
        const int j = 16 * (wave * CT + c) + col;
        if (j < columns) {
#pragma unroll
            for (int i = 0; i < S::kDTiles; ++i) {
                *reinterpret_cast<float4_t *>(parts.o + (k.part + j) * D + 16 * i + 4 * quad) = o[c][i];
            }
            if (quad == 0) {
                // relative to the maximum as narrow units have it: with the factor, and with weights from 2^Split::kTop down
                parts.stats[k.part + j] = make_float2(m[c] * c_scale + (Split<T>::kTop - kTop), poisoned ? NAN : l[c]);
            }
        }
    }
    __syncthreads(); // the next unit takes the buffers
}

// A run of each line per workgroup. Half of the workgroups begin with the wide line, which the matrix cores bound, half with the
// narrow one, which the memory bounds.
template <class T, int D> __global__ void __launch_bounds__(kThreads, D <= 128 ? 2 : 1) shared_attention_kernel(SharedAttentionArgs a) {
    using S = Shape<T, D>;
    constexpr int kNarrowBytes = kAttentionWaves * S::kRegion, kWideBytes = 4 * kWideTile * S::kRowBytes;
    __shared__ __attribute__((aligned(16))) uint8_t lds[kNarrowBytes > kWideBytes ? kNarrowBytes : kWideBytes];
    __shared__ float2 wave_stats[kAttentionWaves][16];
    const ShareWorkspace plan = carve_share(a.plan, a.rows);
    if (!fits(plan, a)) {
        return;
    }
    const int w = blockIdx.x;
    const bool wide_first = 2 * w < a.runs;
#pragma unroll 1
    for (int turn = 0; turn < 2; ++turn) {
        const int line = (turn == 0) == wide_first ? 1 : 0;
        const ShareLine all{uniform(plan.header->lines[line].segments), uniform(plan.header->lines[line].tiles)};
        const Runs runs = Runs::deal(all.tiles, a.runs);
        int x = runs.begin(w);
        const int x_end = runs.begin(w + 1);
        if (x >= x_end) {
            continue;
        }
        const ShareSegment *segments = line == 1 ? plan.wide : plan.narrow;
        int at = segment_at(segments, all.segments, x);
        while (x < x_end) {
            if (line == 0) {
                narrow_work<T, D>(a, next_work<0>(a, segments, at, x, x_end, w), lds, wave_stats);
            } else {
                const Work k = next_work<1>(a, segments, at, x, x_end, w);
                if (k.rows * a.group_heads > 64) {
                    wide_work<T, D, 2>(a, k, lds);
                } else {
                    wide_work<T, D, 1>(a, k, lds);
                }
            }
        }
    }
}

// A column's parts joined: those of the segments on its row's path, each of the runs that its unit lies in.
template <class T, int D, int THREADS> __global__ void __launch_bounds__(THREADS) shared_join_kernel(SharedAttentionArgs a) {
    constexpr int kItems = D / 4, kLanes = THREADS / kItems, kAhead = 4;
    struct Span { // the parts of one unit: of runs first..last, that of the last at `end`
        int64_t run0, end;
        int count;
    };
    __shared__ Span spans[kPathEntries];
    __shared__ float4_t acc[kLanes][kItems];
    __shared__ float2 stat[kLanes];
    const int64_t t = blockIdx.x / a.q_heads;
    const int head = static_cast<int>(blockIdx.x - t * a.q_heads);
    const Keys keys = keys_of(a, t);
    if (keys.request < 0) {
        return;
    }
    uint16_t *out = a.out + t * a.ldo + static_cast<int64_t>(head) * D;
    const ShareWorkspace plan = carve_share(a.plan, a.rows);
    const SharedParts parts = carve_parts(a.workspace, shared_columns(a.rows, a.q_heads, a.runs));
    if (threadIdx.x < kPathEntries) {
        const int ref = fits(plan, a) ? plan.paths[t * kPathEntries + threadIdx.x] : -1;
        Span span{0, 0, 0};
        if (ref >= 0) {
            const int line = ref & 1;
            const ShareSegment s = (line ? plan.wide : plan.narrow)[ref >> 1];
            const Runs runs = Runs::deal(plan.header->lines[line].tiles, a.runs);
            const int kv_head = head / a.group_heads, row = static_cast<int>(t) - s.row0, chunks = s.chunks(), chunk = row / s.chunk;
            const int tile = s.tile0 + (kv_head * chunks + chunk) * s.tiles;
            const int w0 = runs.of(tile), w1 = runs.of(tile + s.tiles - 1);
            const int in_unit = (row - chunk * s.chunk) * a.group_heads + head - kv_head * a.group_heads;
            span.run0 = run_column(a.rows, a.q_heads, a.runs, line, w0) + in_unit;
            span.end = static_cast<int64_t>(s.slot0) * a.q_heads + (static_cast<int64_t>(kv_head) * s.rows + row) * a.group_heads + head - kv_head * a.group_heads;
            span.count = (w1 - w0 + 1) * 2 + line;
        }
        spans[threadIdx.x] = span;
    }
    __syncthreads();
    int total = 0;
#pragma unroll
    for (int i = 0; i < kPathEntries; ++i) {
        total += spans[i].count >> 1;
    }
    const auto column_of = [&](int p) {
        int64_t column = 0;
#pragma unroll
        for (int i = 0; i < kPathEntries; ++i) {
            const Span &s = spans[i];
            const int n = s.count >> 1;
            if (p >= 0 && p < n) {
                column = p == n - 1 ? s.end : s.run0 + p * ((s.count & 1) ? kWideCols : kNarrowCols);
            }
            p -= n;
        }
        return column;
    };
    const int y = threadIdx.x / kItems, e = threadIdx.x - y * kItems;
    float m = -INFINITY, l = 0.0f;
    float4_t v = float4_t{0.0f, 0.0f, 0.0f, 0.0f};
    if (y < kLanes) {
        for (int i = y; i < total; i += kAhead * kLanes) {
            float2 st[kAhead];
            float4_t o[kAhead];
            float top = m;
#pragma unroll
            for (int n = 0; n < kAhead; ++n) {
                const int64_t column = column_of(min(i + n * kLanes, total - 1));
                st[n] = parts.stats[column];
                o[n] = *reinterpret_cast<const float4_t *>(parts.o + column * D + 4 * e);
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
        acc[y][e] = v;
        if (e == 0) {
            stat[y] = make_float2(m, l);
        }
    }
    __syncthreads();
    if (y == 0) {
        float top = -INFINITY, sum = 0.0f;
        float4_t all = float4_t{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
        for (int i = 0; i < kLanes; ++i) {
            top = fmaxf(top, stat[i].x);
        }
#pragma unroll
        for (int i = 0; i < kLanes; ++i) {
            const float f = exp2_fast(stat[i].x - (top == -INFINITY ? 0.0f : top));
            all += acc[i][e] * f;
            sum += stat[i].y * f;
        }
        const float over = keys.bad ? NAN : keys.end == 0 ? 1.0f : sum; // a row that sees no key is zero
        store4<T>(out + 4 * e, all / over);
    }
}

template <class T, int D> hipError_t launch_shared(const SharedAttentionArgs &a, hipStream_t stream) {
    hipLaunchKernelGGL((shared_attention_kernel<T, D>), dim3(static_cast<unsigned>(a.runs)), dim3(kThreads), 0, stream, a);
    const hipError_t e = hipGetLastError();
    if (e != hipSuccess) {
        return e;
    }
    hipLaunchKernelGGL((shared_join_kernel<T, D, 256>), dim3(static_cast<unsigned>(a.rows * a.q_heads)), dim3(256), 0, stream, a);
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
