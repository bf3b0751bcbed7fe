// A C++ host over the C ABI alone (include/hm_w4a16.h; no Python, no torch) as a serving loop over a paged key-value cache calls it: each
// step plans its pages (hm_page_plan), makes its Q/K/V rows ready and writes keys and values to the cache (hm_qk_norm_rope) and attends
// (hm_paged_attention), over steps in which requests start, decode, end and make room for others. Every output row is checked against a
// float64 evaluation of its request's whole history. Prints PASS and exits 0 on success; exits 2 when no GPU is visible.
#include "hm_w4a16.h"

#include <hip/hip_runtime.h>

#include <cmath>
#include <cstdint>
#include <cstdio>
#include <cstring>
#include <random>
#include <vector>

namespace {

uint16_t bf16_bits(float f) { // round to nearest even (finite inputs)
    uint32_t u;
    std::memcpy(&u, &f, 4);
    u += 0x7FFFu + ((u >> 16) & 1u);
    return static_cast<uint16_t>(u >> 16);
}

float bf16_value(uint16_t b) {
    const uint32_t u = static_cast<uint32_t>(b) << 16;
    float f;
    std::memcpy(&f, &u, 4);
    return f;
}

#define CHECK_HM(call)                                                                                   \
    do {                                                                                                 \
        const hm_status st_ = (call);                                                                    \
        if (st_ != HM_OK) {                                                                              \
            std::fprintf(stderr, "%s: status %d: %s\n", #call, static_cast<int>(st_), hm_last_error()); \
            return 1;                                                                                    \
        }                                                                                                \
    } while (0)

#define CHECK_HIP(call)                                                                       \
    do {                                                                                      \
        const hipError_t e_ = (call);                                                         \
        if (e_ != hipSuccess) {                                                               \
            std::fprintf(stderr, "%s: %s\n", #call, hipGetErrorString(e_));                   \
            return 1;                                                                         \
        }                                                                                     \
    } while (0)

template <class T> T *device_copy(const std::vector<T> &v) {
    T *p = nullptr;
    if (hipMalloc(&p, v.size() * sizeof(T)) != hipSuccess || hipMemcpy(p, v.data(), v.size() * sizeof(T), hipMemcpyHostToDevice) != hipSuccess) {
        std::fprintf(stderr, "no device memory\n");
        std::exit(1);
    }
    return p;
}

constexpr int QHeads = 8, KvHeads = 2, D = 64, PageSize = 16, Pages = 24, R = 4, W = 8, Rows = 48, Cols = (QHeads + 2 * KvHeads) * D;

// A head rotated at `position`, as a row holds it after its rounding.
std::vector<double> rotated(const uint16_t *x, int position, const std::vector<double> &frequencies) {
    std::vector<double> y(D);
    for (int i = 0; i < D / 2; ++i) {
        const double a = bf16_value(x[i]), b = bf16_value(x[i + D / 2]), c = std::cos(position * frequencies[i]), s = std::sin(position * frequencies[i]);
        y[i] = bf16_value(bf16_bits(static_cast<float>(a * c - b * s)));
        y[i + D / 2] = bf16_value(bf16_bits(static_cast<float>(b * c + a * s)));
    }
    return y;
}

} // namespace

int main() {
    int devices = 0;
    if (hipGetDeviceCount(&devices) != hipSuccess || devices == 0) {
        std::fprintf(stderr, "no GPU\n");
        return 2;
    }
    std::vector<double> frequencies(D / 2);
    for (int i = 0; i < D / 2; ++i) {
        frequencies[i] = std::pow(10000.0, -2.0 * i / D);
    }
    std::vector<int32_t> ring(Pages);
    for (int i = 0; i < Pages; ++i) {
        ring[i] = (7 * i + 3) % Pages;
    }
    hm_kv_cache cache{};
    CHECK_HIP(hipMalloc(&cache.k, static_cast<size_t>(Pages) * KvHeads * PageSize * D * 2));
    CHECK_HIP(hipMalloc(&cache.v, static_cast<size_t>(Pages) * KvHeads * PageSize * D * 2));
    cache.pages = Pages, cache.page_size = PageSize;
    cache.page_stride = KvHeads * PageSize * D, cache.head_stride = PageSize * D, cache.token_stride = D;
    cache.kv_heads = KvHeads, cache.head_dim = D, cache.dtype = HM_BF16;

    int32_t *lengths = device_copy(std::vector<int32_t>(R, 0)), *added = device_copy(std::vector<int32_t>(R, 0));
    int32_t *table = device_copy(std::vector<int32_t>(R * W, -1)), *free_pages = device_copy(ring);
    int64_t *queue = device_copy(std::vector<int64_t>{0, Pages, 0, 0}), *slots = device_copy(std::vector<int64_t>(Rows));
    int32_t *positions = device_copy(std::vector<int32_t>(Rows)), *requests = device_copy(std::vector<int32_t>(Rows));
    int32_t *starts = device_copy(std::vector<int32_t>(R + 1));
    uint16_t *qkv = device_copy(std::vector<uint16_t>(Rows * Cols)), *out = device_copy(std::vector<uint16_t>(Rows * QHeads * D));
    double *freq = device_copy(frequencies);
    const size_t bytes = hm_paged_attention_workspace_bytes(&cache, QHeads);
    void *ws = nullptr;
    CHECK_HIP(hipMalloc(&ws, bytes));
    hipStream_t s;
    CHECK_HIP(hipStreamCreate(&s));

    std::mt19937 rng(5);
    std::normal_distribution<float> normal(0.0f, 1.0f);
    std::vector<std::vector<std::vector<uint16_t>>> history(R); // each request's rows
    const int steps[][R] = {{5, 0, 33, 0}, {1, 17, 1, 0}, {1, 1, 1, 9}, {-1, 1, 1, 1}, {30, 1, -1, 1}, {1, 1, 7, 1}};
    for (const auto &step : steps) {
        std::vector<uint16_t> x(Rows * Cols, bf16_bits(3.0f));
        int used = 0;
        for (int r = 0; r < R; ++r) {
            if (step[r] < 0) {
                history[r].clear();
            }
            for (int i = 0; i < step[r]; ++i, ++used) {
                for (int c = 0; c < Cols; ++c) {
                    x[used * Cols + c] = bf16_bits(normal(rng));
                }
                history[r].emplace_back(x.begin() + used * Cols, x.begin() + (used + 1) * Cols);
            }
        }
        CHECK_HIP(hipMemcpy(added, step, sizeof(step), hipMemcpyHostToDevice));
        CHECK_HIP(hipMemcpy(qkv, x.data(), x.size() * 2, hipMemcpyHostToDevice));

        // once per step: pages, slots and positions of its rows; lengths and queue advance in place
        CHECK_HM(hm_page_plan(lengths, added, R, table, W, W, PageSize, free_pages, Pages, queue, slots, positions, requests, Rows, starts, lengths, queue, s));
        // each layer: queries in place, keys and values to their slots
        hm_qk_norm_rope_args rope{};
        rope.qkv = qkv, rope.ldqkv = Cols, rope.q = qkv, rope.ldq = Cols;
        rope.frequencies = freq, rope.positions = positions, rope.slots = slots;
        rope.rows = Rows, rope.q_heads = QHeads, rope.kv_heads = KvHeads, rope.head_dim = D, rope.rotary_dim = D, rope.dtype = HM_BF16;
        CHECK_HM(hm_qk_norm_rope(&rope, &cache, s));
        CHECK_HM(hm_paged_attention(&cache, out, QHeads * D, qkv, Cols, Rows, QHeads, table, W, R, W, positions, requests, 1.0f / std::sqrt(static_cast<float>(D)),
                                    0, ws, bytes, s));
        CHECK_HIP(hipStreamSynchronize(s));

        std::vector<uint16_t> got(Rows * QHeads * D);
        int64_t counters[4];
        CHECK_HIP(hipMemcpy(got.data(), out, got.size() * 2, hipMemcpyDeviceToHost));
        CHECK_HIP(hipMemcpy(counters, queue, sizeof(counters), hipMemcpyDeviceToHost));
        if (counters[2] != 0 || counters[3] != used) {
            std::fprintf(stderr, "plan: %lld refused, %lld rows\n", static_cast<long long>(counters[2]), static_cast<long long>(counters[3]));
            return 1;
        }
        double err2 = 0.0, ref2 = 0.0;
        int row = 0;
        for (int r = 0; r < R; ++r) {
            for (int i = 0; i < step[r]; ++i, ++row) {
                const int last = static_cast<int>(history[r].size()) - step[r] + i;
                for (int h = 0; h < QHeads; ++h) {
                    const int kv = h / (QHeads / KvHeads);
                    const std::vector<double> q = rotated(&history[r][last][h * D], last, frequencies);
                    std::vector<double> sum(D);
                    double weights = 0.0;
                    for (int j = 0; j <= last; ++j) { // scores of order 1: exp needs no maximum
                        const std::vector<double> k = rotated(&history[r][j][(QHeads + kv) * D], j, frequencies);
                        double dot = 0.0;
                        for (int d = 0; d < D; ++d) {
                            dot += q[d] * k[d];
                        }
                        const double p = std::exp(dot / std::sqrt(static_cast<double>(D)));
                        weights += p;
                        for (int d = 0; d < D; ++d) {
                            sum[d] += p * bf16_value(history[r][j][(QHeads + KvHeads + kv) * D + d]);
                        }
                    }
                    for (int d = 0; d < D; ++d) {
                        const double ref = sum[d] / weights, off = bf16_value(got[(row * QHeads + h) * D + d]) - ref;
                        err2 += off * off;
                        ref2 += ref * ref;
                    }
                }
            }
        }
        // Half steps of bf16 (2^-8), each at most that much of the whole: a query or key whose rounding falls on the other side than here, through scores
        // of order 1 (2), and the output's rounding.
        const double rel = std::sqrt(err2 / ref2);
        std::printf("%d rows: rel_l2=%.3e\n", used, rel);
        if (!(rel <= 3.0 / 256.0)) {
            std::fprintf(stderr, "outside tolerance\n");
            return 1;
        }
    }
    CHECK_HIP(hipStreamDestroy(s));
    for (void *p : {cache.k, cache.v, static_cast<void *>(lengths), static_cast<void *>(added), static_cast<void *>(table), static_cast<void *>(free_pages),
                    static_cast<void *>(queue), static_cast<void *>(slots), static_cast<void *>(positions), static_cast<void *>(requests),
                    static_cast<void *>(starts), static_cast<void *>(qkv), static_cast<void *>(out), static_cast<void *>(freq), ws}) {
        CHECK_HIP(hipFree(p));
    }
    std::printf("PASS\n");
    return 0;
}
