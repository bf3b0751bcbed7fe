// Rows of a Q/K/V projection made ready for attention: bias, RMSNorm of each query and key head, position rotation, keys and
// values to their cache slots, in one pass over the rows.
//
// A head of D elements is handled by D / 16 lanes (of a group of the next power of two), 16 elements each in two 16-byte
// pieces. A lane takes pieces c of both halves, so that with either pairing both elements
// of a pair are its own and only the norm's sum crosses lanes. The angles depend on the row alone: a workgroup forms cos and sin of its rows once
// (position times frequency in turns in fp64, the fraction of a turn in fp32, so that far positions lose nothing) and all
// heads read them from LDS.
//
// Bound by memory: each element is read and written once (4 bytes of traffic, about 10 fp32 operations). 8192 rows of 32 + 2 * 8 heads of
// 128, normed: 201 MB in 39.4 us (5.1 TB/s; a copy of 4 GB runs at 4.75). One row: 3.1 us, a launch.
#include "hm_device.hpp"
#include "hm_internal.hpp"

#include <algorithm>

namespace hm {
namespace {

constexpr int kThreads = 256;
constexpr int kMaxRows = 2; // rows of one workgroup (8192 rows, with plain loads and stores: 44 us, with 1 row 45, with 4 and 8 rows 48)

template <class T> __device__ __forceinline__ void unpack8(const uint4 v, float o[8]) {
    const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        o[2 * i] = T::to_float(w[i] & 0xFFFFu);
        o[2 * i + 1] = T::to_float(w[i] >> 16);
    }
}

template <class T> __device__ __forceinline__ uint4 pack8(const float v[8]) {
    uint32_t w[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        w[i] = static_cast<uint32_t>(T::from_float(v[2 * i])) | (static_cast<uint32_t>(T::from_float(v[2 * i + 1])) << 16);
    }
    return make_uint4(w[0], w[1], w[2], w[3]);
}

typedef uint32_t u32x4_t __attribute__((ext_vector_type(4)));

__device__ __forceinline__ uint4 load16(const uint16_t *p) { return *reinterpret_cast<const uint4 *>(p); }

// The rows are read once. Many rows' results outgrow the L2s before anyone reads them, so they are not kept there either (STREAM: 44.6 to
// 40.9 us at 8192 rows of 48 heads of 128); a few rows' queries are read next from the L2.
__device__ __forceinline__ uint4 load16_once(const uint16_t *p) {
    return __builtin_bit_cast(uint4, __builtin_nontemporal_load(reinterpret_cast<const u32x4_t *>(p)));
}

template <bool STREAM> __device__ __forceinline__ void store16(uint16_t *p, const uint4 v) {
    if constexpr (STREAM) {
        __builtin_nontemporal_store(__builtin_bit_cast(u32x4_t, v), reinterpret_cast<u32x4_t *>(p));
    } else {
        *reinterpret_cast<uint4 *>(p) = v;
    }
}

// rows_per_block rows by heads_per_block heads; items (row, head) go round the lane groups. The next item's pieces are
// requested before the present one is worked on.
template <class T, bool INTERLEAVED, bool STREAM>
__global__ void __launch_bounds__(kThreads) qk_norm_rope_kernel(QkNormRopeArgs a, int rows_per_block, int heads_per_block, int group_log) {
    extern __shared__ float2 turn[]; // [rows_per_block][rotary_dim / 2]
    __shared__ int64_t cache_row[kMaxRows]; // offset of the row's slot in the cache, -1: none
    __shared__ int32_t present[kMaxRows];
    const int D = a.head_dim, rd = a.rotary_dim, half = rd / 2;
    const int group = 1 << group_log, groups = kThreads >> group_log;
    const int c = threadIdx.x & (group - 1);
    const int64_t row0 = static_cast<int64_t>(blockIdx.x) * rows_per_block;
    const int rows = static_cast<int>(min(static_cast<int64_t>(rows_per_block), a.rows - row0));
    const int head0 = blockIdx.y * heads_per_block;
    const int heads = min(heads_per_block, a.heads - head0);
    const int items = rows * heads;
    const bool lane_used = c < D / 16;
    const bool rotated = 16 * c < rd;
    // A lane's two pieces lie half of its part of the head apart (the rotated part or the rest): neighbouring lanes load neighbouring pieces.
    const int part = rotated ? 0 : rd, part_c = rotated ? c : c - rd / 16;
    const int off_a = part + 8 * part_c;
    const int off_b = off_a + (rotated ? half : (D - rd) / 2);

    int item = threadIdx.x >> group_log;
    uint4 next_a = {}, next_b = {};
    const auto request = [&](int i) {
        if (i < items && lane_used) {
            const int r = i / heads, h = head0 + i - r * heads;
            const uint16_t *p = a.qkv + (row0 + r) * a.ldqkv + static_cast<int64_t>(h) * D;
            next_a = load16_once(p + off_a);
            next_b = load16_once(p + off_b);
        }
    };
    request(item);
    uint4 qw_a = {}, qw_b = {}, kw_a = {}, kw_b = {};
    if (lane_used && a.q_weight != nullptr) {
        qw_a = load16(a.q_weight + off_a), qw_b = load16(a.q_weight + off_b);
    }
    if (lane_used && a.k_weight != nullptr) {
        kw_a = load16(a.k_weight + off_a), kw_b = load16(a.k_weight + off_b);
    }

    for (int i = threadIdx.x; i < rows * half; i += kThreads) {
        const int r = i / half;
        const double turns = static_cast<double>(a.positions[row0 + r]) * (a.frequencies[i - r * half] * 0.15915494309189535);
        float s, co;
        sincospif(2.0f * static_cast<float>(turns - rint(turns)), &s, &co);
        turn[i] = make_float2(co, s);
    }
    if (threadIdx.x < static_cast<unsigned>(rows)) {
        present[threadIdx.x] = a.positions[row0 + threadIdx.x] >= 0;
        int64_t at = -1;
        if (a.slots != nullptr) {
            const int64_t slot = a.slots[row0 + threadIdx.x];
            if (slot >= 0 && slot >> a.page_shift < a.pages) {
                at = (slot >> a.page_shift) * a.page_stride + (slot & ((int64_t(1) << a.page_shift) - 1)) * a.token_stride;
            }
        }
        cache_row[threadIdx.x] = at;
    }
    __syncthreads();

    for (; item < items; item += groups) {
        const uint4 in_a = next_a, in_b = next_b;
        request(item + groups);
        const int r = item / heads, h = head0 + item - r * heads;
        if (!present[r]) { // the same for the whole lane group: its shuffles stay among themselves
            continue;
        }
        const bool is_q = h < a.q_heads, is_k = !is_q && h < a.q_heads + a.kv_heads;
        uint16_t *dest;
        if (is_q) {
            dest = a.q + (row0 + r) * a.ldq + static_cast<int64_t>(h) * D;
        } else if (a.slots == nullptr) {
            dest = a.k + (row0 + r) * a.ldk + static_cast<int64_t>(h - a.q_heads) * D;
        } else if (cache_row[r] < 0) {
            continue;
        } else {
            dest = (is_k ? a.cache_k + (h - a.q_heads) * a.head_stride : a.cache_v + (h - a.q_heads - a.kv_heads) * a.head_stride) + cache_row[r];
        }
        if (!is_q && !is_k && a.bias == nullptr) { // values without a bias: a copy
            if (lane_used) {
                store16<STREAM>(dest + off_a, in_a);
                store16<STREAM>(dest + off_b, in_b);
            }
            continue;
        }
        float x[8], y[8];
        unpack8<T>(in_a, x);
        unpack8<T>(in_b, y);
        if (a.bias != nullptr && lane_used) {
            float b[8];
            unpack8<T>(load16(a.bias + static_cast<int64_t>(h) * D + off_a), b);
#pragma unroll
            for (int k = 0; k < 8; ++k) {
                x[k] += b[k];
            }
            unpack8<T>(load16(a.bias + static_cast<int64_t>(h) * D + off_b), b);
#pragma unroll
            for (int k = 0; k < 8; ++k) {
                y[k] += b[k];
            }
        }
        if (is_q ? a.q_weight != nullptr : is_k && a.k_weight != nullptr) {
            float sum = 0.0f;
            if (lane_used) {
#pragma unroll
                for (int k = 0; k < 8; ++k) {
                    sum += x[k] * x[k] + y[k] * y[k];
                }
            }
            for (int off = group >> 1; off > 0; off >>= 1) {
                sum += __shfl_xor(sum, off);
            }
            const float scale = 1.0f / sqrtf(sum / static_cast<float>(D) + a.eps);
            float w[8];
            unpack8<T>(is_q ? qw_a : kw_a, w);
#pragma unroll
            for (int k = 0; k < 8; ++k) {
                x[k] *= scale * w[k];
            }
            unpack8<T>(is_q ? qw_b : kw_b, w);
#pragma unroll
            for (int k = 0; k < 8; ++k) {
                y[k] *= scale * w[k];
            }
        }
        if (!lane_used) {
            continue;
        }
        if (rotated && (is_q || is_k)) {
            // The pairs of pieces a and b: pair 8 c + k across them, or, interleaved, pairs 4 c + k of a and half / 2 + 4 c + k of b.
            const float2 *t = turn + r * half + (INTERLEAVED ? 4 : 8) * c;
#pragma unroll
            for (int k = 0; k < 8; ++k) {
                const float2 cs = INTERLEAVED ? (k < 4 ? t[k] : t[half / 2 + k - 4]) : t[k];
                float &p = INTERLEAVED ? (k < 4 ? x[2 * k] : y[2 * k - 8]) : x[k];
                float &q = INTERLEAVED ? (k < 4 ? x[2 * k + 1] : y[2 * k - 7]) : y[k];
                const float p0 = p, q0 = q;
                p = p0 * cs.x - q0 * cs.y;
                q = q0 * cs.x + p0 * cs.y;
            }
        }
        store16<STREAM>(dest + off_a, pack8<T>(x));
        store16<STREAM>(dest + off_b, pack8<T>(y));
    }
}

template <class T> auto kernel_of(bool interleaved, bool stream) {
    return interleaved ? (stream ? qk_norm_rope_kernel<T, true, true> : qk_norm_rope_kernel<T, true, false>)
                       : (stream ? qk_norm_rope_kernel<T, false, true> : qk_norm_rope_kernel<T, false, false>);
}

} // namespace

hipError_t launch_qk_norm_rope(const QkNormRopeArgs &a, hipStream_t stream) {
    if (a.rows == 0) {
        return hipSuccess;
    }
    int group_log = 0;
    while ((1 << group_log) < a.head_dim / 16) {
        ++group_log;
    }
    const int groups = kThreads >> group_log;
    // Few rows: one pass of the lane groups per workgroup, so that the heads spread over the CUs.
    const int64_t spread = a.rows * ((a.heads + groups - 1) / groups);
    const bool few = spread < 8 * device_topology().cus;
    const int rows_per_block = few ? 1 : kMaxRows;
    const int heads_per_block = few ? std::min<int>(a.heads, groups) : a.heads;
    const dim3 grid(static_cast<unsigned>((a.rows + rows_per_block - 1) / rows_per_block),
                    static_cast<unsigned>((a.heads + heads_per_block - 1) / heads_per_block));
    const size_t lds = static_cast<size_t>(rows_per_block) * (a.rotary_dim / 2) * sizeof(float2);
    auto kern = a.dtype == HM_FP16 ? kernel_of<F16>(a.interleaved, !few) : kernel_of<BF16>(a.interleaved, !few);
    hipLaunchKernelGGL(kern, grid, dim3(kThreads), lds, stream, a, rows_per_block, heads_per_block, group_log);
    return hipGetLastError();
}

} // namespace hm
