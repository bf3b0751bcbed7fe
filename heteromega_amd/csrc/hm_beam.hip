// Beam search's selection: of the continuations of a request's beams the k best, by score + logit - log(sum of exp(logits)).
//
// Bound by memory: the logits are read once (2 bytes each in 16 bits), 64 requests of 4 beams and 152064 tokens 78 MB. A wave takes 64 bytes a lane of one row
// into registers and works out its maximum, the sum of exp relative to it and its k best tokens; a second launch, a workgroup per request, joins the
// waves' sums in fp64 and picks the k best of all their candidates. Candidates of one row are compared by their logits, which are exact; those of
// different rows by fp64 scores, since their sums' errors (about 1e-8 relative: fp32 sums of 32 terms, joined in fp64) should not decide which comes first.
//
// The k best of a wave's 2048: the k-th largest of the 64 lanes' maxima, found by sorting them over the lanes, is a bound that at least k elements reach and
// seldom many more; those go to a list in LDS and are ranked by counting who comes before. Many equal or badly spread elements overflow the list;
// then the best are taken one after the other.
#include "hm_device.hpp"
#include "hm_internal.hpp"

namespace hm {
namespace {

constexpr int kVectors = 4;    // 16-byte loads of a lane
constexpr int kList = 192;     // candidates that a wave's list holds
constexpr int kJoinThreads = 256;
constexpr int kJoinList = 1024;

struct Fp32 {
    static __device__ __forceinline__ float to_float(uint32_t bits) { return __uint_as_float(bits); }
};

template <class T> struct Elements {
    static constexpr int kOf16Bytes = 8;
    static __device__ __forceinline__ float get(const uint4 &v, int i) {
        const uint32_t w = i < 2 ? v.x : i < 4 ? v.y : i < 6 ? v.z : v.w;
        return T::to_float(i & 1 ? w >> 16 : w & 0xFFFFu);
    }
};
template <> struct Elements<Fp32> {
    static constexpr int kOf16Bytes = 4;
    static __device__ __forceinline__ float get(const uint4 &v, int i) { return __uint_as_float(i == 0 ? v.x : i == 1 ? v.y : i == 2 ? v.z : v.w); }
};

template <class T> constexpr int wave_elements() { return 64 * kVectors * Elements<T>::kOf16Bytes; }

struct Candidate {
    float logit;
    int32_t token;
};

struct BeamWorkspace {
    float2 *stats;         // [rows][parts]: maximum, and sum of exp(logit - maximum)
    Candidate *candidates; // [rows][parts][k], best first; tokens of -1 behind the last
};

__host__ __device__ __forceinline__ BeamWorkspace carve_beam(void *p, int64_t rows, int64_t parts) {
    float2 *stats = static_cast<float2 *>(p);
    return {stats, reinterpret_cast<Candidate *>(stats + rows * parts)};
}

// Whether a row has candidates from its logits.
__device__ __forceinline__ bool is_open(const BeamSelectArgs &a, int64_t row) {
    return (a.ended == nullptr || a.ended[row] == 0) && fabsf(a.scores[row]) < INFINITY;
}

// The k-th largest value of the lanes': sorted downwards over the lanes.
__device__ __forceinline__ float kth_of_lanes(float v, int k) {
    const int lane = threadIdx.x & 63;
#pragma unroll
    for (int size = 2; size <= 64; size <<= 1) {
#pragma unroll
        for (int step = size >> 1; step > 0; step >>= 1) {
            const float other = __shfl_xor(v, step);
            const bool keep_more = ((lane & step) == 0) == ((lane & size) == 0 || size == 64);
            v = keep_more ? fmaxf(v, other) : fminf(v, other);
        }
    }
    return __shfl(v, k - 1);
}

__device__ __forceinline__ bool before(float v, int32_t token, float w, int32_t other) { return v > w || (v == w && token < other); }

template <class T> __global__ void __launch_bounds__(256) beam_parts_kernel(BeamSelectArgs a) {
    using E = Elements<T>;
    constexpr int kOne = E::kOf16Bytes, kMine = kVectors * kOne;
    __shared__ Candidate list[4][kList];
    const int lane = threadIdx.x & 63, wave = uniform(threadIdx.x >> 6);
    const int64_t row = blockIdx.y;
    const int part = static_cast<int>(blockIdx.x) * 4 + wave;
    if (part >= a.parts || !is_open(a, row)) {
        return;
    }
    // 16-byte pieces from the one on that holds the row's first element: what lies around the row's elements in its first and last piece is read, not used.
    const int64_t bytes = 16 / kOne, start = reinterpret_cast<int64_t>(a.logits) + row * a.ld * bytes;
    const int skip = static_cast<int>(start & 15) / static_cast<int>(bytes);
    const uint4 *pieces = reinterpret_cast<const uint4 *>(start & ~int64_t(15));
    const int vocabulary = static_cast<int>(a.vocabulary), last_piece = (vocabulary + skip - 1) / kOne;
    const int first = part * (64 * kVectors);
    uint4 raw[kVectors];
#pragma unroll
    for (int i = 0; i < kVectors; ++i) {
        const int piece = first + i * 64 + lane;
        raw[i] = piece <= last_piece ? pieces[piece] : uint4{};
    }
    float x[kMine];
#pragma unroll
    for (int i = 0; i < kVectors; ++i) {
#pragma unroll
        for (int e = 0; e < kOne; ++e) {
            x[i * kOne + e] = E::get(raw[i], e);
        }
    }
    const auto token_of = [&](int j) { return (first + j / kOne * 64 + lane) * kOne + j % kOne - skip; };
    if (first == 0 || first + kVectors * 64 > last_piece) { // elements that are not the row's
#pragma unroll
        for (int j = 0; j < kMine; ++j) {
            const int token = token_of(j);
            x[j] = token >= 0 && token < vocabulary ? x[j] : -INFINITY;
        }
    }
    float most = x[0];
#pragma unroll
    for (int j = 1; j < kMine; ++j) {
        most = fmaxf(most, x[j]);
    }
    float top = most;
#pragma unroll
    for (int off = 32; off > 0; off >>= 1) {
        top = fmaxf(top, __shfl_xor(top, off));
    }
    // An infinity or NaN among the logits makes the sum NaN.
    const float from = top == -INFINITY ? 0.0f : top;
    float sum = 0.0f;
#pragma unroll
    for (int j = 0; j < kMine; ++j) {
        sum += __builtin_amdgcn_exp2f((x[j] - from) * 1.4426950408889634f);
    }
#pragma unroll
    for (int off = 32; off > 0; off >>= 1) {
        sum += __shfl_xor(sum, off);
    }
    const BeamWorkspace ws = carve_beam(a.workspace, a.rows, a.parts);
    const int64_t at = row * a.parts + part;
    if (lane == 0) {
        ws.stats[at] = make_float2(top, sum);
    }
    const int k = a.k;
    Candidate *out = ws.candidates + at * k;
    const float bound = fmaxf(kth_of_lanes(most, k), -3.4028234663852886e38f); // -infinity is no candidate
    Candidate *mine = list[wave];
    int count = 0;
#pragma unroll
    for (int j = 0; j < kMine; ++j) {
        const bool in = x[j] >= bound;
        const uint64_t who = __ballot(in);
        if (who != 0) {
            const int place = count + __popcll(who & ((uint64_t(1) << lane) - 1));
            if (in && place < kList) {
                mine[place] = Candidate{x[j], token_of(j)};
            }
            count += __popcll(who);
        }
    }
    __builtin_amdgcn_wave_barrier(); // a wave's LDS accesses are carried out in order
    if (count <= kList) {
        for (int i = lane; i < count; i += 64) {
            const Candidate c = mine[i];
            int rank = 0;
            for (int j = 0; j < count; ++j) {
                const Candidate d = mine[j];
                rank += before(d.logit, d.token, c.logit, c.token);
            }
            if (rank < k) {
                out[rank] = c;
            }
        }
        for (int i = count + lane; i < k; i += 64) {
            out[i] = Candidate{-INFINITY, -1};
        }
        return;
    }
    float last = INFINITY;
    int32_t last_token = -1;
    for (int i = 0; i < k; ++i) { // the best behind the last one taken
        float best = -INFINITY;
        int32_t token = INT32_MAX;
#pragma unroll
        for (int j = 0; j < kMine; ++j) {
            const int32_t t = token_of(j);
            if (before(last, last_token, x[j], t) && before(x[j], t, best, token)) {
                best = x[j], token = t;
            }
        }
#pragma unroll
        for (int off = 32; off > 0; off >>= 1) {
            const float v = __shfl_xor(best, off);
            const int32_t t = __shfl_xor(token, off);
            if (before(v, t, best, token)) {
                best = v, token = t;
            }
        }
        if (lane == 0) {
            out[i] = best == -INFINITY ? Candidate{-INFINITY, -1} : Candidate{best, token};
        }
        last = best, last_token = token;
    }
}

struct Scored {
    double score;
    int32_t beam;
    float logit;
    int32_t token;
};

// Where the scores' rounding makes equals of a row's logits (next to a sum of 1e38, say), these still tell them apart.
__device__ __forceinline__ bool before(const Scored &a, const Scored &b) {
    return a.score > b.score || (a.score == b.score && (a.beam < b.beam || (a.beam == b.beam && before(a.logit, a.token, b.logit, b.token))));
}

constexpr Scored kNone{-INFINITY, INT32_MAX, -INFINITY, INT32_MAX};

// A workgroup per request.
__global__ void __launch_bounds__(kJoinThreads) beam_join_kernel(BeamSelectArgs a) {
    __shared__ double norm[HM_BEAM_MAX_BEAMS], base[HM_BEAM_MAX_BEAMS]; // base NaN: the row has no candidates from its logits
    __shared__ uint8_t was_ended[HM_BEAM_MAX_BEAMS];
    __shared__ double maxima[kJoinThreads];
    __shared__ Scored list[kJoinList];
    __shared__ Scored wave_best[kJoinThreads / 64];
    __shared__ int listed;
    __shared__ double bound_at;
    const int lane = threadIdx.x & 63, wave = uniform(threadIdx.x >> 6);
    const int beams = a.beams, k = a.k, parts = a.parts;
    const int64_t row0 = static_cast<int64_t>(blockIdx.x) * beams;
    const BeamWorkspace ws = carve_beam(a.workspace, a.rows, parts);
    for (int beam = wave; beam < beams; beam += kJoinThreads / 64) {
        const int64_t row = row0 + beam;
        const bool open = is_open(a, row);
        float top = -INFINITY;
        bool odd = false;
        for (int i = lane; open && i < parts; i += 64) {
            const float2 st = ws.stats[row * parts + i];
            top = fmaxf(top, st.x);
            odd |= !(st.y < INFINITY);
        }
#pragma unroll
        for (int off = 32; off > 0; off >>= 1) {
            top = fmaxf(top, __shfl_xor(top, off));
        }
        double sum = 0.0;
        for (int i = lane; open && i < parts; i += 64) {
            const float2 st = ws.stats[row * parts + i];
            sum += st.y == 0.0f ? 0.0 : static_cast<double>(st.y) * exp(static_cast<double>(st.x) - static_cast<double>(top));
        }
#pragma unroll
        for (int off = 32; off > 0; off >>= 1) {
            sum += __shfl_xor(sum, off);
        }
        odd = __any(odd) || !(fabsf(top) < INFINITY);
        if (lane == 0) {
            const float score = a.scores[row];
            const bool ended = a.ended != nullptr && a.ended[row] != 0;
            norm[beam] = static_cast<double>(top) + log(sum);
            base[beam] = open && odd ? NAN : fabsf(score) < INFINITY ? static_cast<double>(score) : NAN;
            was_ended[beam] = ended;
        }
    }
    if (threadIdx.x == 0) {
        listed = 0;
    }
    __syncthreads();
    // Candidate i of the request's, all rows' parts' k; one that is not there has a score of -infinity.
    const int per_row = parts * k;
    const int64_t all = static_cast<int64_t>(beams) * per_row;
    const auto scored = [&](int64_t i) {
        const int beam = static_cast<int>(i / per_row);
        Scored s = kNone;
        if (base[beam] != base[beam]) {
            return s;
        }
        const int in_row = static_cast<int>(i - static_cast<int64_t>(beam) * per_row);
        if (was_ended[beam] != 0) { // goes on as it is, once
            if (in_row == 0) {
                s = Scored{base[beam], beam, 0.0f, a.end_token};
            }
            return s;
        }
        const Candidate c = ws.candidates[(row0 + beam) * per_row + in_row];
        if (c.token >= 0) {
            s = Scored{base[beam] + (static_cast<double>(c.logit) - norm[beam]), beam, c.logit, c.token};
        }
        return s;
    };
    double most = -INFINITY;
    for (int64_t i = threadIdx.x; i < all; i += kJoinThreads) {
        most = fmax(most, scored(i).score);
    }
    maxima[threadIdx.x] = most;
    __syncthreads();
    {
        // The k-th largest of the threads' maxima, ties counted one by one: a bound that at least k candidates reach.
        int rank = 0;
        for (int i = 0; i < kJoinThreads; ++i) {
            rank += maxima[i] > most || (maxima[i] == most && i < static_cast<int>(threadIdx.x));
        }
        if (rank == k - 1) {
            bound_at = most;
        }
    }
    __syncthreads();
    const double bound = bound_at;
    for (int64_t i = threadIdx.x; i < all; i += kJoinThreads) {
        const Scored s = scored(i);
        if (s.score >= bound && s.score > -INFINITY) {
            const int place = atomicAdd(&listed, 1);
            if (place < kJoinList) {
                list[place] = s;
            }
        }
    }
    __syncthreads();
    const auto put = [&](int rank, const Scored &s) {
        const int64_t to = static_cast<int64_t>(blockIdx.x) * k + rank;
        const bool some = s.score > -INFINITY;
        a.parents[to] = some ? static_cast<int32_t>(row0) + s.beam : -1;
        a.tokens[to] = some ? s.token : -1;
        a.scores_out[to] = some ? static_cast<float>(s.score) : -INFINITY;
        a.ended_out[to] = !some || was_ended[s.beam] != 0 || s.token == a.end_token;
    };
    const int count = listed;
    if (count <= kJoinList) {
        for (int i = threadIdx.x; i < count; i += kJoinThreads) {
            const Scored s = list[i];
            int rank = 0;
            for (int j = 0; j < count; ++j) {
                rank += before(list[j], s);
            }
            if (rank < k) {
                put(rank, s);
            }
        }
        for (int i = count + threadIdx.x; i < k; i += kJoinThreads) {
            put(i, kNone);
        }
        return;
    }
    Scored last{INFINITY, -1, INFINITY, -1};
    for (int i = 0; i < k; ++i) { // the best behind the last one taken
        Scored best = kNone;
        for (int64_t j = threadIdx.x; j < all; j += kJoinThreads) {
            const Scored s = scored(j);
            if (before(last, s) && before(s, best)) {
                best = s;
            }
        }
#pragma unroll
        for (int off = 32; off > 0; off >>= 1) {
            const Scored other{__shfl_xor(best.score, off), __shfl_xor(best.beam, off), __shfl_xor(best.logit, off), __shfl_xor(best.token, off)};
            best = before(other, best) ? other : best;
        }
        if (lane == 0) {
            wave_best[wave] = best;
        }
        __syncthreads();
#pragma unroll
        for (int w = 0; w < kJoinThreads / 64; ++w) {
            best = before(wave_best[w], best) ? wave_best[w] : best;
        }
        if (threadIdx.x == 0) {
            put(i, best);
        }
        last = best;
        __syncthreads();
    }
}

int64_t parts_of(int64_t vocabulary, int dtype) { // the row may begin within a piece
    const int64_t one = dtype == HM_LOGITS_FP32 ? 4 : 8;
    return (vocabulary + one - 1 + 64 * kVectors * one - 1) / (64 * kVectors * one);
}

} // namespace

size_t beam_select_workspace(int64_t rows, int64_t vocabulary, int64_t k, int dtype) {
    return static_cast<size_t>(rows * parts_of(vocabulary, dtype)) * (sizeof(float2) + static_cast<size_t>(k) * sizeof(Candidate));
}

hipError_t launch_beam_select(BeamSelectArgs a, hipStream_t stream) {
    a.parts = static_cast<int>(parts_of(a.vocabulary, a.dtype));
    const dim3 grid(static_cast<unsigned>((a.parts + 3) / 4), static_cast<unsigned>(a.rows));
    switch (a.dtype) {
    case HM_FP16:
        hipLaunchKernelGGL((beam_parts_kernel<F16>), grid, dim3(256), 0, stream, a);
        break;
    case HM_BF16:
        hipLaunchKernelGGL((beam_parts_kernel<BF16>), grid, dim3(256), 0, stream, a);
        break;
    default:
        hipLaunchKernelGGL((beam_parts_kernel<Fp32>), grid, dim3(256), 0, stream, a);
    }
    const hipError_t e = hipGetLastError();
    if (e != hipSuccess) {
        return e;
    }
    hipLaunchKernelGGL(beam_join_kernel, dim3(static_cast<unsigned>(a.rows / a.beams)), dim3(kJoinThreads), 0, stream, a);
    return hipGetLastError();
}

} // namespace hm
