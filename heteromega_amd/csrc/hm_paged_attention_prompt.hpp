// Attention over a paged cache for the rows of prompts (hm_paged_attention.hip has the mathematics): a part of
// hm_paged_attention_kernel.hpp, whose types it uses.
//
// Many rows of one request read the same keys, so the matrix cores bound them, not the memory: of their work, a third is the weights'
// lower half. A unit has 64 CT columns (rows of one request times the query heads of a key head), 16 CT of them per wave, and its four
// waves share each tile of 64 keys, of which each brings a quarter into LDS. Against a tile per wave, a key is loaded and stored once
// for four times the columns, and each read of it from LDS feeds CT products. Two buffers, one barrier a tile; the next tile is under way
// while one is worked on. A wave skips tiles that none of its rows sees. Nothing is split over keys; the last rows, the longest of a
// prompt, go first.
//
// 32 query and 8 key heads of 128, bf16: a prompt of 2048 rows 108 us (319 TFLOP/s; 408 us by units of 16 columns), of 8192 rows 849 us
// (648; 4400), the last 2048 of 32768 rows 1.62 ms (656; 8.75 ms). A large matrix product reaches 1199 TFLOP/s, and the lower halves
// make three products of two, so 800 would be all. Steps at 8192 rows: as first built 1211 us; 32 of the tile's 64 keys at a time, for
// the registers, 1176; maximum followed late 1050; masks as branches, paired conversions 1015; page ids by vector loads 990; rows
// counted in a launch before 922 (828 timed as above, and 849 since the maximum is taken from scores without their factor).
#pragma once

constexpr int kPromptTile = 16 * kAttentionWaves;

// A workgroup per key head and aligned block of plan.prompt_rows rows, if that is a prompt block: its rows in runs of one request (mostly
// one run), each a unit.
template <class T, int D> __global__ void __launch_bounds__(kThreads, D <= 128 ? 2 : 1) prompt_attention_kernel(PagedAttentionArgs a, AttentionPlan plan) {
    using S = Shape<T, D>;
    typedef typename Split<T>::elem_t elem4_t __attribute__((ext_vector_type(4)));
    constexpr int CT = prompt_tiles(D), kMostRows = 16 * kAttentionWaves * CT, kSubs = kAttentionWaves;
    // The maximum that weights are relative to follows only when a score passes it by more than a factor 2^kSlack: sums and outputs are
    // rescaled seldom, and weights stay in range by starting that much lower. The maximum is one of the scores as they leave the product, and is taken from them
    // before the factor comes in: a fused score times factor less a maximum that was rounded with its factor is off by half a step of that maximum, in
    // the exponent (infinite fp16 weights from 2^23 on). The subtraction costs 2 %: 8192 rows 828 -> 849 us.
    constexpr float kSlack = 3.0f, kTop = Split<T>::kTop - (Split<T>::kTop > 0.0f ? kSlack : 0.0f);
    constexpr int kTileBytes = kPromptTile * S::kRowBytes; // of keys, or values
    __shared__ __attribute__((aligned(16))) uint8_t lds[2][2][kTileBytes];
    __shared__ int32_t row_request[kMostRows], row_first[kMostRows], row_end[kMostRows]; // end -1: outside the table
    __shared__ int odd[2][kSubs]; // infinities or NaN among the values of a sub-tile

    const int kv_head = blockIdx.x % a.kv_heads, blocks = gridDim.x / a.kv_heads;
    // Longest first; if all are on the card at once, the second of a CU's two is the shorter the longer the first.
    const int place = blockIdx.x / a.kv_heads;
    const int64_t block = blocks > plan.prompt_slots || 2 * place < blocks ? blocks - 1 - place : place - (blocks + 1) / 2;
    if (!of_prompt(a, prompts_known(a, plan), block)) {
        return;
    }
    const int lane = threadIdx.x & 63, wave = uniform(threadIdx.x >> 6);
    const int col = lane & 15, quad = lane >> 4;
    const int rows = plan.prompt_rows, group = plan.group_heads;
    const int64_t t0 = block * rows;
    if (threadIdx.x < static_cast<unsigned>(rows)) {
        const Keys k = keys_of(a, t0 + threadIdx.x);
        row_request[threadIdx.x] = k.request;
        row_first[threadIdx.x] = k.first;
        row_end[threadIdx.x] = k.bad ? -1 : k.end;
    }
    __syncthreads();

    const uint32_t row_bytes = static_cast<uint32_t>(a.token_stride) * 2;
    const Pieces<D> pieces(lane, row_bytes);
    const uint32_t to_lds = wave * 16 * S::kRowBytes + pieces.lds_offset();
    const uint32_t k_lds = col * S::kRowBytes + quad * 16;
    const uint32_t v_lds = (4 * quad + (col >> 2)) * S::kRowBytes + (col & 3) * 8;
    // The sign goes to the queries. Not zero: a masked score of -infinity times it must stay one.
    const float c_scale = fmaxf(fabsf(a.scale) * 1.4426950408889634f, 0x1p-126f);
    const float slack = fminf(kSlack / c_scale, 0x1p126f); // of scores without the factor
    const uint32_t sign = a.scale < 0.0f ? 0x80008000u : 0u;
    const int64_t page_stride = uniform64(a.page_stride);
    const int shift = uniform(a.page_shift), offset_mask = (1 << shift) - 1;
    const uint32_t pages = uniform(static_cast<int>(a.pages));
    const uint16_t *k_head = a.k + uniform64(kv_head * a.head_stride), *v_head = a.v + uniform64(kv_head * a.head_stride);

    int from = 0;
    while (from < rows) {
        const int request = uniform(row_request[from]);
        if (request < 0) {
            ++from;
            continue;
        }
        if (uniform(row_end[from]) < 0) {
            uint16_t *out = a.out + (t0 + from) * a.ldo + static_cast<int64_t>(kv_head) * group * D;
            for (int i = 4 * threadIdx.x; i < group * D; i += 4 * kThreads) {
                store4<T>(out + i, float4_t{NAN, NAN, NAN, NAN});
            }
            ++from;
            continue;
        }
        // ---- the run's rows, [from, stop), and the keys that some and all of them see ----
        int stop = rows;
#pragma unroll
        for (int i = kMostRows - 64; i >= 0; i -= 64) {
            const int at = i + lane;
            const uint64_t other = __ballot(at > from && at < rows && (row_request[at] != request || row_end[at] < 0));
            stop = other != 0 ? i + static_cast<int>(__builtin_ctzll(other)) : stop;
        }
        int first = INT32_MAX, end = 0, all_first = 0, all_end = INT32_MAX;
#pragma unroll
        for (int i = 0; i < kMostRows; i += 64) {
            const int at = i + lane;
            if (at >= from && at < stop) {
                first = min(first, row_first[at]), all_first = max(all_first, row_first[at]);
                end = max(end, row_end[at]), all_end = min(all_end, row_end[at]);
            }
        }
#pragma unroll
        for (int off = 32; off > 0; off >>= 1) {
            first = min(first, __shfl_xor(first, off)), all_first = max(all_first, __shfl_xor(all_first, off));
            end = max(end, __shfl_xor(end, off)), all_end = min(all_end, __shfl_xor(all_end, off));
        }
        first = uniform(first), end = uniform(end), all_first = uniform(all_first), all_end = uniform(all_end);
        const int start = first & ~15, tiles = uniform((max(0, end - start) + kPromptTile - 1) / kPromptTile);

        // ---- the lane's columns, and the keys that some and all of the wave's see ----
        u32x4_t q[CT][S::kSteps];
        int col_first[CT], col_end[CT], col_row[CT]; // of a column that is not there: all keys
        int wave_first = INT32_MAX, wave_end = 0, wave_all_first = 0, wave_all_end = INT32_MAX;
        const int columns = (stop - from) * group;
        const auto head_offset = [&](int c) { // of column c's head in its row
            const int j = 16 * (wave * CT + c) + col;
            return static_cast<int64_t>(kv_head * group + j - (col_row[c] - from) * group) * D;
        };
#pragma unroll
        for (int c = 0; c < CT; ++c) {
            const int j = 16 * (wave * CT + c) + col;
            const bool live = j < columns;
            col_row[c] = live ? from + j / group : stop;
            col_first[c] = live ? row_first[col_row[c]] : 0;
            col_end[c] = live ? row_end[col_row[c]] : INT32_MAX;
            if (live) {
                wave_first = min(wave_first, col_first[c]), wave_all_first = max(wave_all_first, col_first[c]);
                wave_end = max(wave_end, col_end[c]), wave_all_end = min(wave_all_end, col_end[c]);
            }
            const uint16_t *q_row = live ? a.q + (t0 + col_row[c]) * a.ldq + head_offset(c) + 8 * quad : a.q;
#pragma unroll
            for (int s = 0; s < S::kSteps; ++s) {
                q[c][s] = live ? *reinterpret_cast<const u32x4_t *>(q_row + 32 * s) ^ sign : u32x4_t{0, 0, 0, 0};
            }
        }
#pragma unroll
        for (int off = 8; off > 0; off >>= 1) {
            wave_first = min(wave_first, __shfl_xor(wave_first, off)), wave_all_first = max(wave_all_first, __shfl_xor(wave_all_first, off));
            wave_end = max(wave_end, __shfl_xor(wave_end, off)), wave_all_end = min(wave_all_end, __shfl_xor(wave_all_end, off));
        }
        wave_first = uniform(wave_first), wave_end = uniform(wave_end);
        wave_all_first = uniform(wave_all_first), wave_all_end = uniform(wave_all_end);

        float4_t o[CT][S::kDTiles];
        float m[CT], l[CT];
        bool poisoned[CT];
#pragma unroll
        for (int c = 0; c < CT; ++c) {
#pragma unroll
            for (int i = 0; i < S::kDTiles; ++i) {
                o[c][i] = float4_t{0.0f, 0.0f, 0.0f, 0.0f};
            }
            m[c] = -INFINITY, l[c] = 0.0f, poisoned[c] = false;
        }

        u32x4_t k_reg[S::kSteps], v_reg[S::kSteps];
        const int32_t *table = a.block_table + uniform64(request * a.ld_table);
        int32_t ids = 0; // of sub-tile lane % kSubs: a vector load, since waits for LDS would wait for a scalar one too
        const auto page_ids = [&](int tile) {
            const int key = start + tile * kPromptTile + 16 * (lane % kSubs);
            ids = key < end ? table[key >> shift] : 0;
        };
        const auto load = [&](int tile) { // the wave's sub-tile; pages outside the cache are noted for all columns that see them
            if (__any(static_cast<uint32_t>(ids) >= pages)) {
#pragma unroll
                for (int s = 0; s < kSubs; ++s) {
                    const int key = start + tile * kPromptTile + 16 * s;
                    if (static_cast<uint32_t>(__builtin_amdgcn_readlane(ids, s)) >= pages) {
#pragma unroll
                        for (int c = 0; c < CT; ++c) {
                            poisoned[c] |= key < col_end[c] && key + 16 > col_first[c];
                        }
                    }
                }
            }
            const int32_t page = __builtin_amdgcn_readlane(ids, wave);
            const int key = start + tile * kPromptTile + 16 * wave;
            const int seen = static_cast<uint32_t>(page) < pages ? max(0, min(16, end - key)) : 0;
            const uint32_t bytes = uniform(seen > 0 ? (seen - 1) * row_bytes + 2 * D : 0);
            const int64_t at = uniform64(seen > 0 ? page * page_stride + static_cast<int64_t>(key & offset_mask) * (row_bytes / 2) : 0);
            const __amdgpu_buffer_rsrc_t kr = buffer_rsrc(k_head + at, bytes), vr = buffer_rsrc(v_head + at, bytes);
#pragma unroll
            for (int i = 0; i < S::kSteps; ++i) {
                k_reg[i] = __builtin_amdgcn_raw_buffer_load_b128(kr, pieces.offset(i), 0, 0);
            }
#pragma unroll
            for (int i = 0; i < S::kSteps; ++i) {
                v_reg[i] = __builtin_amdgcn_raw_buffer_load_b128(vr, pieces.offset(i), 0, 0);
            }
        };
        if (tiles > 0) {
            page_ids(0);
            load(0);
            page_ids(min(1, tiles - 1));
        }
        for (int tile = 0; tile < tiles; ++tile) {
            const int buffer = tile & 1, key0 = start + tile * kPromptTile;
            uint8_t *k_tile = lds[buffer][0], *v_tile = lds[buffer][1];
            if (key0 < first) { // values before the windows count as zero, whatever they are
#pragma unroll
                for (int i = 0; i < S::kSteps; ++i) {
                    if (key0 + 16 * wave + pieces.key(i) < first) {
                        v_reg[i] = u32x4_t{0, 0, 0, 0};
                    }
                }
            }
            // Keys that some rows see and others do not: a weight of zero does not hide an infinity or NaN among their values. Those go in as zero,
            // and the rows that see them get them at the end of the tile.
            const bool mixed = key0 < all_first || key0 + kPromptTile > all_end;
            if (mixed) {
                bool is_odd = false;
#pragma unroll
                for (int i = 0; i < S::kSteps; ++i) {
#pragma unroll
                    for (int k = 0; k < 4; ++k) {
                        const uint32_t v = v_reg[i][k], e = Split<T>::kExponent;
                        const uint32_t keep = ((v & e) == e ? 0u : 0xFFFFu) | ((v >> 16 & e) == e ? 0u : 0xFFFF0000u);
                        is_odd |= keep != 0xFFFFFFFFu;
                        v_reg[i][k] = v & keep;
                    }
                }
                is_odd = __any(is_odd);
                if (lane == 0) {
                    odd[buffer][wave] = is_odd;
                }
            }
#pragma unroll
            for (int i = 0; i < S::kSteps; ++i) {
                *reinterpret_cast<u32x4_t *>(k_tile + to_lds + pieces.lds_step(i)) = k_reg[i];
                *reinterpret_cast<u32x4_t *>(v_tile + to_lds + pieces.lds_step(i)) = v_reg[i];
            }
            // The buffer's readers of two tiles ago passed the barrier of the last one.
            __syncthreads();
            if (tile + 1 < tiles) {
                load(tile + 1);
                page_ids(min(tile + 2, tiles - 1));
            }
            if (key0 >= wave_end || key0 + kPromptTile <= wave_first) {
                continue;
            }
            const bool some_masked = key0 < wave_all_first || key0 + kPromptTile > wave_all_end;
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
                        const uint4 k = *reinterpret_cast<const uint4 *>(k_tile + k_lds + half_lds + s * 16 * S::kRowBytes + 64 * i);
#pragma unroll
                        for (int c = 0; c < CT; ++c) {
                            score[c][s] = T::mfma16(k, __builtin_bit_cast(uint4, q[c][i]), score[c][s]);
                        }
                    }
                }
                u32x4_t hi[CT], lo[CT];
#pragma unroll
                for (int c = 0; c < CT; ++c) {
                    if (some_masked) {
                        __builtin_amdgcn_sched_barrier(0); // keeps this a branch: as selects it is a sixth of a tile's instructions
#pragma unroll
                        for (int e = 0; e < 8; ++e) {
                            const int key = key0 + 32 * h + 16 * (e >> 2) + 4 * quad + (e & 3);
                            if (key < col_first[c] || key >= col_end[c]) {
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
                        for (int k = 0; k < 2; ++k) {
                            p[k] = exp2_fast(__builtin_fmaf(score[c][e >> 2][(e & 3) + k] - m_used, c_scale, kTop));
                            l[c] += p[k];
                        }
                        uint32_t upper, lower;
                        split<T>(p, upper, lower);
                        hi[c][e / 2] = upper, lo[c][e / 2] = lower;
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
                        o[c][i] = T::mfma16(vt, __builtin_bit_cast(uint4, hi[c]), o[c][i]);
                        o[c][i] = T::mfma16(vt, __builtin_bit_cast(uint4, lo[c]), o[c][i]);
                    }
                }
            }
            if (!mixed) {
                continue;
            }
            for (int s = 0; s < kSubs; ++s) { // infinities and NaN, read again: they show whatever their weight
                const int sub = key0 + 16 * s;
                const int32_t page = sub < end ? uniform(table[sub >> shift]) : -1;
                if (uniform(odd[buffer][s]) == 0 || static_cast<uint32_t>(page) >= pages) {
                    continue;
                }
                for (int key = max(sub, first); key < min(sub + 16, end); ++key) {
                    const uint16_t *v_row = v_head + page * page_stride + static_cast<int64_t>(key & offset_mask) * (row_bytes / 2) + 4 * quad;
#pragma unroll
                    for (int i = 0; i < S::kDTiles; ++i) {
                        const uint2 v = *reinterpret_cast<const uint2 *>(v_row + 16 * i);
#pragma unroll
                        for (int e = 0; e < 4; ++e) {
                            const uint32_t bits = (e < 2 ? v.x : v.y) >> 16 * (e % 2) & 0xFFFFu;
                            const float value = (bits & Split<T>::kExponent) == Split<T>::kExponent ? T::to_float(bits) : 0.0f;
#pragma unroll
                            for (int c = 0; c < CT; ++c) {
                                o[c][i][e] += key >= col_first[c] && key < col_end[c] ? value : 0.0f;
                            }
                        }
                    }
                }
            }
        }

#pragma unroll
        for (int c = 0; c < CT; ++c) {
            l[c] += __shfl_xor(l[c], 16);
            l[c] += __shfl_xor(l[c], 32);
            if (col_row[c] < stop) {
                const float factor = poisoned[c] ? NAN : col_end[c] == 0 ? 1.0f : 1.0f / l[c]; // a row that sees no key is zero
                uint16_t *out = a.out + (t0 + col_row[c]) * a.ldo + head_offset(c);
#pragma unroll
                for (int i = 0; i < S::kDTiles; ++i) {
                    *reinterpret_cast<elem4_t *>(out + 16 * i + 4 * quad) = __builtin_convertvector(o[c][i] * factor, elem4_t);
                }
            }
        }
        __syncthreads(); // the next run's tiles take the buffers
        from = stop;
    }
}
