// Beam search's selection: of the continuations of a request's beams the k best, by score + logit - log(sum of exp(logits)).
//
// Bound by memory and, nearly as much, by the instructions of a first launch, which reads the logits once: 64 requests of 4 beams and 152064 tokens have 78 MB of
// them in 16 bits. A wave takes 32 elements a lane of one row into registers and works out its maximum, the sum of exp relative to it and its k best tokens. A
// second launch, a workgroup per request, joins the waves' sums and picks the k best of their candidates. It is bound by latency: of the waves' best ones only
// those that reach the k-th score's bound are looked at closely. With all candidates compared it took 26 to 34 us, so 5.5. Candidates of one row are compared by their
// logits, which are exact; those of different rows by fp64 scores, so that rounding adds no ties. Nor may it take any away: which lane sums which tokens, and in
// which order the sums are joined, goes by the token alone, whichever beam a row is and wherever it begins in memory, so that equal rows have one sum, to the last bit.
//
// The k best of a wave's 2048: the k-th largest of the 64 lanes' maxima (above k = 32, of 128 halves' maxima), found by sorting them over the lanes, is a bound that at
// least k elements reach and seldom many more; those go to a list in LDS and are ranked by counting who comes before. (The least of k or more groups' maxima is
// quicker to find, but almost three times as many reach it: 37 us instead of 21 for the case above. 64 elements a lane, with fewer sorts, took 25 at three waves a
// SIMD; 8 or 16 of them for few logits gain less here than the second launch loses by more parts.) Many equal or badly spread elements overflow the list; then the
// best are taken one after the other. A request's candidates are ranked in the same way, after a second and third bound where there are many.
#include "hm_device.hpp"
#include "hm_internal.hpp"

namespace hm {
namespace {

constexpr int kElements = 32;    // of a lane
constexpr float kLowest = -3.4028234663852886e38f;
constexpr int kList = 256;       // candidates that a wave's list holds
constexpr int kJoinList = 1024;  // and that of a request
constexpr int kJoinParts = 1024; // parts that are looked at at once
constexpr int kRanked = 128;     // candidates that are ranked without a look for a better bound

typedef uint32_t u32x4_t __attribute__((ext_vector_type(4)));
struct __attribute__((packed)) Unaligned {
    u32x4_t v;
};

struct Fp32 {
    static __device__ __forceinline__ float to_float(uint32_t bits) { return __uint_as_float(bits); }
};

template <class T> struct Elements {
    static constexpr int kOf16Bytes = 8;
    static __device__ __forceinline__ float get(const u32x4_t &v, int i) { return T::to_float(i & 1 ? v[i / 2] >> 16 : v[i / 2] & 0xFFFFu); }
    // Element `at` of a row in the place of the i-th, which was zero.
    static __device__ __forceinline__ void put(u32x4_t &v, int i, const uint8_t *row, int at) {
        v[i / 2] |= static_cast<uint32_t>(reinterpret_cast<const uint16_t *>(row)[at]) << (i & 1 ? 16 : 0);
    }
};
template <> struct Elements<Fp32> {
    static constexpr int kOf16Bytes = 4;
    static __device__ __forceinline__ float get(const u32x4_t &v, int i) { return __uint_as_float(v[i]); }
    static __device__ __forceinline__ void put(u32x4_t &v, int i, const uint8_t *row, int at) { v[i] = reinterpret_cast<const uint32_t *>(row)[at]; }
};

// A logit and its token as one whole number, in the order of candidates of a row: larger logits first (zeros of either sign are equal), of equal ones lower tokens.
// 0: none.
typedef uint64_t Candidate;
__device__ __forceinline__ uint32_t ordered(float v) {
    const uint32_t bits = __float_as_uint(v + 0.0f);
    return bits ^ ((bits >> 31) != 0 ? 0xFFFFFFFFu : 0x80000000u);
}
__device__ __forceinline__ float value_of(uint32_t key) { return __uint_as_float((key >> 31) != 0 ? key ^ 0x80000000u : ~key); }
__device__ __forceinline__ Candidate candidate(float logit, int32_t token) { return static_cast<uint64_t>(ordered(logit)) << 32 | ~static_cast<uint32_t>(token); }

struct BeamWorkspace {
    float2 *stats;         // [rows][parts]: maximum, and sum of exp(logit - maximum)
    Candidate *candidates; // [rows][parts][k], best first
};

__host__ __device__ __forceinline__ BeamWorkspace carve_beam(void *p, int64_t rows, int64_t parts) {
    float2 *stats = static_cast<float2 *>(p);
    return {stats, reinterpret_cast<Candidate *>(stats + rows * parts)};
}

// Whether a row has candidates from its logits.
__device__ __forceinline__ bool is_open(const BeamSelectArgs &a, int64_t row) {
    return (a.ended == nullptr || a.ended[row] == 0) && fabsf(a.scores[row]) < INFINITY;
}

template <int CTRL> __device__ __forceinline__ int dpp(int v) { return __builtin_amdgcn_mov_dpp(v, CTRL, 0xF, 0xF, true); }

// The values of a lane and of the one whose number has bit STEP changed, in either order, without passing through LDS.
template <int STEP> __device__ __forceinline__ int2 both(int v) {
    if constexpr (STEP <= 8) { // quad_perm, row_half_mirror (^ 7) of quad_perm (^ 3), row_ror
        return make_int2(v, STEP == 1 ? dpp<0xB1>(v) : STEP == 2 ? dpp<0x4E>(v) : STEP == 4 ? dpp<0x141>(dpp<0x1B>(v)) : dpp<0x128>(v));
    } else {
        typedef unsigned pair_t __attribute__((ext_vector_type(2)));
        const unsigned bits = static_cast<unsigned>(v);
        const pair_t p = STEP == 16 ? __builtin_bit_cast(pair_t, __builtin_amdgcn_permlane16_swap(bits, bits, false, false))
                                    : __builtin_bit_cast(pair_t, __builtin_amdgcn_permlane32_swap(bits, bits, false, false));
        return make_int2(static_cast<int>(p.x), static_cast<int>(p.y));
    }
}

template <int STEP = 1> __device__ __forceinline__ double sum_over_lanes(double v) {
    const int2 low = both<STEP>(__double2loint(v)), high = both<STEP>(__double2hiint(v));
    v = __hiloint2double(high.x, low.x) + __hiloint2double(high.y, low.y);
    if constexpr (STEP < 32) {
        v = sum_over_lanes<2 * STEP>(v);
    }
    return v;
}

template <int STEP = 1, class F> __device__ __forceinline__ float over_lanes(float v, F f) {
    const int2 p = both<STEP>(__float_as_int(v));
    v = f(__int_as_float(p.x), __int_as_float(p.y));
    if constexpr (STEP < 32) {
        v = over_lanes<2 * STEP>(v, f);
    }
    return v;
}

// Steps of a bitonic sort downwards over the lanes: runs of SIZE sorted, from pairs STEP lanes apart.
template <int SIZE, int STEP> __device__ __forceinline__ int sort_steps(int v, int lane) {
    const int2 p = both<STEP>(v);
    const int more = max(p.x, p.y), less = min(p.x, p.y);
    v = ((lane & STEP) == 0) == ((lane & SIZE) == 0 || SIZE == 64) ? more : less;
    if constexpr (STEP > 1) {
        return sort_steps<SIZE, STEP / 2>(v, lane);
    } else if constexpr (SIZE < 64) {
        return sort_steps<2 * SIZE, SIZE>(v, lane);
    } else {
        return v;
    }
}

// The lanes' values sorted downwards, as whole numbers of the same order: those take one instruction each where floats are made quiet first.
struct Sorted {
    int keys;

    static __device__ __forceinline__ int key_of(int bits) { return bits ^ (bits >> 31 & 0x7FFFFFFF); }
    __device__ __forceinline__ explicit Sorted(float v) : keys(sort_steps<2, 1>(key_of(__float_as_int(v)), threadIdx.x & 63)) {}
    __device__ __forceinline__ float at(int i) const { return __int_as_float(key_of(__builtin_amdgcn_readlane(keys, i))); }
};

// A wave per part of a row.
template <class T> __global__ void __launch_bounds__(256) beam_parts_kernel(BeamSelectArgs a) {
    using E = Elements<T>;
    constexpr int kOne = E::kOf16Bytes, V = kElements / kOne;
    __shared__ Candidate list[4][kList];
    const int lane = threadIdx.x & 63, wave = uniform(threadIdx.x >> 6);
    const int64_t row = blockIdx.y;
    const int part = static_cast<int>(blockIdx.x) * 4 + wave;
    if (part >= a.parts) {
        return;
    }
    if (!is_open(a, row)) {
        return;
    }
    // Pieces of 16 bytes from the row's first element on, which is aligned to its type alone: loads of any alignment take no longer (64 requests of 4 beams, bf16:
    // 152 061 tokens 25.5 us, 152 064 26.0).
    const int vocabulary = static_cast<int>(a.vocabulary), first = part * (64 * V);
    const uint8_t *const from_row = static_cast<const uint8_t *>(a.logits) + row * a.ld * (16 / kOne);
    int first_token = (first + lane) * kOne;
    const auto token_of = [&](int j) { return first_token + j / kOne * 64 * kOne + j % kOne; };
    const auto piece_of = [&](int i) __attribute__((always_inline)) { // zeros behind the row's end
        const int token = token_of(i * kOne);
        u32x4_t piece{0, 0, 0, 0};
        if (token + kOne <= vocabulary) {
            piece = reinterpret_cast<const Unaligned *>(from_row + static_cast<int64_t>(token) * (16 / kOne))->v;
        } else if (token < vocabulary) {
#pragma unroll
            for (int e = 0; e < kOne - 1; ++e) {
                if (token + e < vocabulary) {
                    E::put(piece, e, from_row, token + e);
                }
            }
        }
        return piece;
    };
    const bool inside = (first + 64 * V) * kOne <= vocabulary;
    u32x4_t raw[V];
    if (inside) {
        const Unaligned *pieces = reinterpret_cast<const Unaligned *>(from_row + static_cast<int64_t>(first) * 16) + lane;
#pragma unroll
        for (int i = 0; i < V; ++i) {
            raw[i] = pieces[64 * i].v;
        }
    } else {
#pragma unroll
        for (int i = 0; i < V; ++i) {
            raw[i] = piece_of(i);
        }
    }
    float x[kElements];
#pragma unroll
    for (int i = 0; i < V; ++i) {
#pragma unroll
        for (int e = 0; e < kOne; ++e) {
            x[i * kOne + e] = E::get(raw[i], e);
        }
    }
    if (!inside) {
#pragma unroll
        for (int j = 0; j < kElements; ++j) {
            x[j] = token_of(j) < vocabulary ? x[j] : -INFINITY;
        }
    }
    float half[2] = {x[0], x[kOne / 2]}; // of the halves of each 16 bytes, so that short rows have both
#pragma unroll
    for (int j = 1; j < kElements; ++j) {
        half[j % kOne / (kOne / 2)] = fmaxf(half[j % kOne / (kOne / 2)], x[j]);
    }
    const int k = a.k;
    Sorted best(fmaxf(half[0], half[1]));
    const float top = best.at(0);
    if (k > 32) { // the best 64 of the lanes' halves' maxima: the bound that 64 of 64 maxima give is reached by 300 elements, this one by 90
        const Sorted first(half[0]), second(half[1]);
        best.keys = sort_steps<2, 1>(max(first.keys, __shfl(second.keys, 63 - lane)), lane);
    }
    // An infinity or NaN among the logits makes the sum NaN.
    const float from = top == -INFINITY ? 0.0f : top;
    float sum = 0.0f;
#pragma unroll
    for (int i = 0; i < V; ++i) {
        float some = 0.0f;
#pragma unroll
        for (int e = 0; e < kOne; ++e) {
            some += __builtin_amdgcn_exp2f((x[i * kOne + e] - from) * 1.4426950408889634f);
        }
        sum += some;
    }
    sum = over_lanes(sum, [](float v, float w) { return v + w; });
    const BeamWorkspace ws = carve_beam(a.workspace, a.rows, a.parts);
    const int64_t at = row * a.parts + part;
    if (lane == 0) {
        ws.stats[at] = make_float2(top, sum);
    }
    Candidate *out = ws.candidates + at * k;
    const float bound = fmaxf(best.at(k - 1), kLowest); // -infinity is no candidate
    Candidate *mine = list[wave];
#if defined(__HIP_DEVICE_COMPILE__)
    asm volatile("" : "+v"(first_token)); // the tokens are worked out again rather than kept in registers
#endif
    int count = 0;
#pragma unroll
    for (int j = 0; j < kElements; ++j) {
        const bool in = x[j] >= bound;
        const uint64_t who = __ballot(in);
        if (who != 0) {
            const int place = count + __popcll(who & ((uint64_t(1) << lane) - 1));
            if (in && place < kList) {
                mine[place] = candidate(x[j], token_of(j));
            }
            count += __popcll(who);
        }
    }
    __builtin_amdgcn_wave_barrier(); // a wave's LDS accesses are carried out in order
    for (int i = count + lane; i < k; i += 64) {
        out[i] = 0;
    }
    if (count <= 64) {
        const Candidate c = lane < count ? mine[lane] : 0;
        const uint32_t upper = static_cast<uint32_t>(c >> 32), lower = static_cast<uint32_t>(c);
        int rank = 0;
        for (int j = 0; j < count; ++j) {
            const uint32_t u = __builtin_amdgcn_readlane(upper, j), v = __builtin_amdgcn_readlane(lower, j);
            rank += (static_cast<uint64_t>(u) << 32 | v) > c;
        }
        if (lane < count && rank < k) {
            out[rank] = c;
        }
        return;
    }
    if (count <= kList) {
        Candidate own[kList / 64];
        int rank[kList / 64];
#pragma unroll
        for (int i = 0; i < kList / 64; ++i) {
            own[i] = 64 * i + lane < count ? mine[64 * i + lane] : 0;
            rank[i] = 0;
        }
#pragma unroll 2
        for (int j = 0; j < count; ++j) {
            const Candidate c = mine[j];
#pragma unroll
            for (int i = 0; i < kList / 64; ++i) {
                if (64 * i < count) {
                    rank[i] += c > own[i];
                }
            }
        }
#pragma unroll
        for (int i = 0; i < kList / 64; ++i) {
            if (64 * i + lane < count && rank[i] < k) {
                out[rank[i]] = own[i];
            }
        }
        return;
    }
    Candidate last = ~Candidate(0);
    for (int i = 0; i < k; ++i) { // the best behind the last one taken, from memory: seldom, and little code
        Candidate best = 0;
#pragma unroll 1
        for (int j = 0; j < V; ++j) {
            const u32x4_t piece = piece_of(j);
#pragma unroll
            for (int e = 0; e < kOne; ++e) {
                const int32_t t = token_of(j * kOne + e);
                const float v = t < vocabulary ? E::get(piece, e) : -INFINITY;
                const Candidate c = v > -INFINITY ? candidate(v, t) : 0;
                best = c < last && c > best ? c : best;
            }
        }
#pragma unroll
        for (int off = 32; off > 0; off >>= 1) {
            const Candidate other = __shfl_xor(static_cast<unsigned long long>(best), off);
            best = other > best ? other : best;
        }
        if (lane == 0) {
            out[i] = best;
        }
        last = best;
    }
}

// A request's candidate in the order of the results: by score, then lower beams first, then as candidates of a row, which rounded scores may make equal (next to a
// sum of 1e38, say). {0, 0}: none.
struct alignas(16) Scored {
    uint64_t score, rest; // rest: 8 bits of the beam, 32 of the logit, 24 of the token

    static __device__ __forceinline__ Scored of(double score, int beam, float logit, int32_t token) {
        const uint64_t bits = static_cast<uint64_t>(__double_as_longlong(score + 0.0));
        return {bits ^ ((bits >> 63) != 0 ? ~uint64_t(0) : uint64_t(1) << 63),
                static_cast<uint64_t>(255 - beam) << 56 | static_cast<uint64_t>(ordered(logit)) << 24 | (0xFFFFFFu - static_cast<uint32_t>(token))};
    }
    __device__ __forceinline__ double value() const { return __longlong_as_double(static_cast<long long>((score >> 63) != 0 ? score ^ uint64_t(1) << 63 : ~score)); }
    __device__ __forceinline__ int beam() const { return 255 - static_cast<int>(rest >> 56); }
    __device__ __forceinline__ int32_t token() const { return static_cast<int32_t>(0xFFFFFFu - (static_cast<uint32_t>(rest) & 0xFFFFFFu)); }
    __device__ __forceinline__ bool some() const { return score != 0; }
};
static_assert(HM_BEAM_MAX_BEAMS <= 256, "a beam has 8 bits");

__device__ __forceinline__ bool before(const Scored &a, const Scored &b) { return a.score > b.score || (a.score == b.score && a.rest > b.rest); }

__device__ __forceinline__ Scored better(const Scored &a, const Scored &b) { // by fields: the whole would be picked in memory
    const bool first = before(a, b);
    return Scored{first ? a.score : b.score, first ? a.rest : b.rest};
}

// Scores as fp32 in their order, none above its score but for those below fp32's range, which are kLowest: -infinity stands for none.
__device__ __forceinline__ float rounded_down(double v) {
    const float f = static_cast<float>(v);
    return v > -INFINITY ? fmaxf(static_cast<double>(f) > v ? nextafterf(f, -INFINITY) : f, kLowest) : -INFINITY;
}

// The bound that such a score is.
__device__ __forceinline__ double bound_of(float v) { return v > kLowest ? static_cast<double>(v) : -INFINITY; }

// A workgroup per request. The scores of the parts' best candidates bound the k-th score from below, and only parts whose best one reaches that bound are looked at
// more closely: about k of them.
template <int THREADS> __global__ void __launch_bounds__(THREADS) beam_join_kernel(BeamSelectArgs a) {
    constexpr int kWaves = THREADS / 64, kHeld = 2;
    __shared__ double norm[HM_BEAM_MAX_BEAMS], base[HM_BEAM_MAX_BEAMS]; // base NaN: the row has no candidates from its logits
    __shared__ uint8_t was_ended[HM_BEAM_MAX_BEAMS];
    __shared__ float maxima[kWaves][64];
    __shared__ float best_of[kJoinParts]; // parts' best scores, rounded down; of the first ones
    __shared__ int32_t work[kJoinParts];
    __shared__ Scored list[kJoinList];
    __shared__ Scored wave_best[kWaves];
    __shared__ int listed, works;
    __shared__ double next_bound;
    const int lane = threadIdx.x & 63, wave = uniform(threadIdx.x >> 6);
    const int beams = a.beams, k = a.k, parts = a.parts;
    const int64_t row0 = static_cast<int64_t>(blockIdx.x) * beams;
    const BeamWorkspace ws = carve_beam(a.workspace, a.rows, parts);
    float own = -INFINITY; // the best of those parts that are the lane's: part i of all beams' is lane i % 64's
    for (int beam = wave; beam < beams; beam += kWaves) {
        const int64_t row = row0 + beam;
        const float2 *stats = ws.stats + row * parts;
        float2 held[kHeld];
#pragma unroll
        for (int n = 0; n < kHeld; ++n) { // of a row that is not open they are not there, and not used
            const int i = lane + 64 * n;
            held[n] = stats[min(i, parts - 1)];
            held[n] = i < parts ? held[n] : make_float2(-INFINITY, 0.0f);
        }
        const float score = a.scores[row];
        const bool ended = a.ended != nullptr && a.ended[row] != 0, open = !ended && fabsf(score) < INFINITY;
        float top = -INFINITY;
        bool odd = false;
        const auto each = [&](auto f) __attribute__((always_inline)) {
#pragma unroll
            for (int n = 0; n < kHeld; ++n) {
                f(lane + 64 * n, held[n]);
            }
            for (int i = lane + 64 * kHeld; i < parts; i += 64) {
                f(i, stats[i]);
            }
        };
        double sum = 0.0;
        if (open) {
            each([&](int, float2 st) {
                top = fmaxf(top, st.x);
                odd |= !(st.y < INFINITY);
            });
            top = over_lanes(top, [](float v, float w) { return fmaxf(v, w); });
            each([&](int, float2 st) { sum += st.y == 0.0f ? 0.0f : st.y * __builtin_amdgcn_exp2f((st.x - top) * 1.4426950408889634f); });
            sum = sum_over_lanes(sum);
            odd = __any(odd) || !(fabsf(top) < INFINITY);
        }
        const double of_row = static_cast<double>(top) + log(sum), from = (open && odd) || !(fabsf(score) < INFINITY) ? NAN : static_cast<double>(score);
        if (lane == 0) {
            norm[beam] = of_row;
            base[beam] = from;
            was_ended[beam] = ended;
        }
        float best = -INFINITY;
        const auto put_best = [&](int i, float v) {
            best = fmaxf(best, v);
            if (beam * parts + i < kJoinParts) {
                best_of[beam * parts + i] = v;
            }
        };
        each([&](int i, float2 st) {
            if (i < parts) {
                // an ended beam goes on as it is, once
                put_best(i, from != from ? -INFINITY : ended ? (i == 0 ? score : -INFINITY) : rounded_down(from + (static_cast<double>(st.x) - of_row)));
            }
        });
        own = fmaxf(own, __shfl(best, (lane - beam * parts) & 63));
    }
    maxima[wave][lane] = own;
    __syncthreads();
#pragma unroll
    for (int w = 0; w < kWaves; ++w) {
        own = fmaxf(own, maxima[w][lane]);
    }
    const int all = beams * parts;
    const auto best_score = [&](int i) {
        if (i < kJoinParts) {
            return best_of[i];
        }
        const int beam = i / parts, part = i - beam * parts;
        return base[beam] != base[beam]    ? -INFINITY
               : was_ended[beam] != 0 ? (part == 0 ? static_cast<float>(base[beam]) : -INFINITY)
                                      : rounded_down(base[beam] + (static_cast<double>(ws.stats[(row0 + beam) * parts + part].x) - norm[beam]));
    };
    // Candidate `place` of a part, as the rows' sums have it, or none.
    const auto scored = [&](int i, int place) {
        const int beam = i / parts, part = i - beam * parts;
        if (base[beam] != base[beam]) {
            return Scored{0, 0};
        }
        if (was_ended[beam] != 0) {
            return part == 0 && place == 0 ? Scored::of(base[beam], beam, 0.0f, a.end_token) : Scored{0, 0};
        }
        const Candidate c = ws.candidates[((row0 + beam) * parts + part) * k + place];
        const float logit = value_of(static_cast<uint32_t>(c >> 32));
        return c != 0 ? Scored::of(base[beam] + (static_cast<double>(logit) - norm[beam]), beam, logit, static_cast<int32_t>(~static_cast<uint32_t>(c))) : Scored{0, 0};
    };
    const auto put = [&](int rank, const Scored &s) {
        const int64_t to = static_cast<int64_t>(blockIdx.x) * k + rank;
        const bool some = s.some();
        a.parents[to] = some ? static_cast<int32_t>(row0) + s.beam() : -1;
        a.tokens[to] = some ? s.token() : -1;
        a.scores_out[to] = some ? static_cast<float>(s.value()) : -INFINITY;
        a.ended_out[to] = !some || was_ended[s.beam()] != 0 || s.token() == a.end_token;
    };
    if (all < 64) { // so few parts that their second, third and further best ones count
        const int place = lane / all;
        const Scored s = place < k ? scored(lane - place * all, place) : Scored{0, 0};
        own = s.some() ? rounded_down(s.value()) : -INFINITY;
    }
    double bound = bound_of(Sorted(own).at(k - 1));
    for (;;) {
        __syncthreads(); // the list's last readers are done
        if (threadIdx.x == 0) {
            listed = 0;
        }
        for (int i0 = 0; i0 < all; i0 += kJoinParts) {
            if (threadIdx.x == 0) {
                works = 0;
            }
            __syncthreads();
            for (int i = i0 + threadIdx.x; i < min(all, i0 + kJoinParts); i += THREADS) {
                const float v = best_score(i);
                if (v > -INFINITY && static_cast<double>(v) >= rounded_down(bound)) {
                    work[atomicAdd(&works, 1)] = i;
                }
            }
            __syncthreads();
            for (int i = threadIdx.x; i < works * k; i += THREADS) {
                const int w = i / k;
                const Scored s = scored(work[w], i - w * k);
                if (s.some() && s.value() >= bound) {
                    const int place = atomicAdd(&listed, 1);
                    if (place < kJoinList) {
                        list[place] = s;
                    }
                }
            }
            __syncthreads();
        }
        const int count = min(listed, kJoinList);
        const bool whole = listed <= kJoinList;
        if (count > kRanked + 4 * k) { // ranking takes the square of the number: the k-th of the lanes' best ones listed is a better bound, unless there are many equal ones
            float most = -INFINITY;
            for (int i = threadIdx.x; i < count; i += THREADS) {
                most = fmaxf(most, rounded_down(list[i].value()));
            }
            maxima[wave][lane] = most;
            __syncthreads();
#pragma unroll
            for (int w = 0; w < kWaves; ++w) {
                most = fmaxf(most, maxima[w][lane]);
            }
            const double next = bound_of(Sorted(most).at(k - 1));
            if (next > bound) {
                bound = next;
                continue;
            }
        }
        for (int i = threadIdx.x; i < count; i += THREADS) {
            const Scored s = list[i];
            int rank = 0;
#pragma unroll 2
            for (int j = 0; j < count; ++j) {
                rank += before(list[j], s);
            }
            if (whole && rank < k) {
                put(rank, s);
            }
            if (!whole && rank == k - 1) {
                next_bound = s.value();
            }
        }
        if (whole) {
            for (int i = count + threadIdx.x; i < k; i += THREADS) {
                put(i, Scored{0, 0});
            }
            return;
        }
        // Too many: the k-th best of those listed is a better bound, unless they are equal.
        __syncthreads();
        if (!(next_bound > bound)) {
            break;
        }
        bound = next_bound;
    }
    Scored last{~uint64_t(0), ~uint64_t(0)};
    for (int i = 0; i < k; ++i) { // the best behind the last one taken
        Scored best{0, 0};
        for (int64_t j = threadIdx.x; j < static_cast<int64_t>(all) * k; j += THREADS) {
            const int part = static_cast<int>(j / k);
            const Scored s = scored(part, static_cast<int>(j - static_cast<int64_t>(part) * k));
            if (before(last, s)) {
                best = better(s, best);
            }
        }
#pragma unroll
        for (int off = 32; off > 0; off >>= 1) {
            const Scored other{__shfl_xor(static_cast<unsigned long long>(best.score), off), __shfl_xor(static_cast<unsigned long long>(best.rest), off)};
            best = better(other, best);
        }
        if (lane == 0) {
            wave_best[wave] = best;
        }
        __syncthreads();
#pragma unroll
        for (int w = 0; w < kWaves; ++w) {
            best = better(wave_best[w], best);
        }
        if (threadIdx.x == 0) {
            put(i, best);
        }
        last = best;
        __syncthreads();
    }
}

int64_t parts_of(int64_t vocabulary) { return (vocabulary + 64 * kElements - 1) / (64 * kElements); }

} // namespace

size_t beam_select_workspace(int64_t rows, int64_t vocabulary, int64_t k) {
    return static_cast<size_t>(rows * parts_of(vocabulary)) * (sizeof(float2) + static_cast<size_t>(k) * sizeof(Candidate));
}

hipError_t launch_beam_select(BeamSelectArgs a, hipStream_t stream) {
    a.parts = static_cast<int>(parts_of(a.vocabulary));
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
    const dim3 requests(static_cast<unsigned>(a.rows / a.beams));
    // A wave for each beam of a search, or sixteen: 64 requests of 4 beams 14.2 us with four waves and 14.8 with sixteen, of 8 18.5 either way, 16 of 16 beams 20.3
    // and 18.6.
    if (a.beams <= 4) {
        hipLaunchKernelGGL((beam_join_kernel<256>), requests, dim3(256), 0, stream, a);
    } else {
        hipLaunchKernelGGL((beam_join_kernel<1024>), requests, dim3(1024), 0, stream, a);
    }
    return hipGetLastError();
}

} // namespace hm
