// C ABI of the attention operators over a paged cache (include/hm_w4a16.h): validation and dispatch.
#include "../../include/hm_w4a16.h"
#include "hm_internal.hpp"

#include <cmath>

namespace {

using hm::set_error;

bool aligned(const void *p, size_t a) { return (reinterpret_cast<uintptr_t>(p) % a) == 0; }

hm_status launched(hipError_t e, const char *what) {
    return e == hipSuccess ? HM_OK : set_error(HM_HIP_ERROR, "%s launch: %s", what, hipGetErrorString(e));
}

int log2_of(int64_t v) { return 63 - __builtin_clzll(static_cast<unsigned long long>(v)); }

hm_status check_page_size(int64_t page_size, const char *what) {
    if (page_size < 16 || page_size > (int64_t(1) << 30) || (page_size & (page_size - 1)) != 0) {
        return set_error(HM_INVALID_ARGUMENT, "%s: page_size must be a power of two from 16 to 2^30, got %lld", what, static_cast<long long>(page_size));
    }
    return HM_OK;
}

hm_status check_dtype(int32_t dtype, const char *what) {
    if (dtype != HM_BF16 && dtype != HM_FP16) {
        return set_error(HM_INVALID_ARGUMENT, "%s: dtype must be HM_BF16 or HM_FP16, got %d", what, static_cast<int>(dtype));
    }
    return HM_OK;
}

hm_status check_cache(const hm_kv_cache *c, const char *what) {
    if (c == nullptr) {
        return set_error(HM_INVALID_ARGUMENT, "%s: null cache", what);
    }
    hm_status st = check_dtype(c->dtype, what);
    if (st != HM_OK || (st = check_page_size(c->page_size, what)) != HM_OK) {
        return st;
    }
    if (c->k == nullptr || c->v == nullptr || !aligned(c->k, 16) || !aligned(c->v, 16)) {
        return set_error(HM_INVALID_ARGUMENT, "%s: keys and values must be 16-byte aligned device pointers", what);
    }
    if (c->pages <= 0 || c->pages > INT32_MAX || c->kv_heads <= 0 || c->head_dim <= 0 || c->head_dim % 16) {
        return set_error(HM_INVALID_ARGUMENT, "%s: a cache has 1 to 2^31 - 1 pages, heads, and a head_dim that is a multiple of 16, got %lld, %d, %d", what,
                         static_cast<long long>(c->pages), static_cast<int>(c->kv_heads), static_cast<int>(c->head_dim));
    }
    if (c->page_stride < c->head_dim || c->head_stride < c->head_dim || c->token_stride < c->head_dim || c->page_stride % 8 || c->head_stride % 8 ||
        c->token_stride % 8) {
        return set_error(HM_INVALID_ARGUMENT, "%s: cache strides must be multiples of 8 and at least head_dim, got %lld, %lld, %lld", what,
                         static_cast<long long>(c->page_stride), static_cast<long long>(c->head_stride), static_cast<long long>(c->token_stride));
    }
    // 2^30 elements: the kernels' byte offsets within a page's head fit 31 bits
    if (c->token_stride > (int64_t(1) << 30) / c->page_size) {
        return set_error(HM_UNSUPPORTED, "%s: a page's tokens of one head must span less than 2 GiB", what);
    }
    return HM_OK;
}

hm_status check_rows(const void *p, int64_t ld, int64_t width, const char *what, const char *name) {
    if (p == nullptr || !aligned(p, 16) || ld % 8 || ld < width) {
        return set_error(HM_INVALID_ARGUMENT, "%s: %s must be 16-byte aligned with a leading dimension that is a multiple of 8 and >= %lld (got %lld)",
                         what, name, static_cast<long long>(width), static_cast<long long>(ld));
    }
    return HM_OK;
}

hm_status check_table(const int32_t *table, int64_t ld, int64_t R, int64_t W, int64_t page_size, const char *what) {
    if (table == nullptr || R <= 0 || R > INT32_MAX || W <= 0 || ld < W) {
        return set_error(HM_INVALID_ARGUMENT, "%s: block_table must be [R > 0, W > 0] with a leading dimension >= W, got [%lld, %lld], %lld", what,
                         static_cast<long long>(R), static_cast<long long>(W), static_cast<long long>(ld));
    }
    // Positions are 32-bit; the attention's tiles may begin up to 15 tokens early and end up to 127 late.
    if (W > (INT32_MAX - 256) / page_size) {
        return set_error(HM_UNSUPPORTED, "%s: W * page_size must stay below 2^31 - 256 tokens, got %lld * %lld", what, static_cast<long long>(W),
                         static_cast<long long>(page_size));
    }
    return HM_OK;
}

} // namespace

extern "C" {

hm_status hm_page_plan(const int32_t *lengths, const int32_t *added, int64_t R, int32_t *block_table, int64_t ld_table, int64_t W,
                       int64_t page_size, int32_t *free_pages, int64_t Q, const int64_t *queue_in, int64_t *slots, int32_t *positions,
                       int32_t *requests, int64_t rows, int32_t *starts, int32_t *lengths_out, int64_t *queue_out, void *stream) {
    const char *what = "hm_page_plan";
    hm_status st = check_page_size(page_size, what);
    if (st != HM_OK || (st = check_table(block_table, ld_table, R, W, page_size, what)) != HM_OK) {
        return st;
    }
    if (R > HM_PAGE_PLAN_MAX_REQUESTS) {
        return set_error(HM_UNSUPPORTED, "%s: at most %d requests, got %lld", what, HM_PAGE_PLAN_MAX_REQUESTS, static_cast<long long>(R));
    }
    if (lengths == nullptr || added == nullptr || free_pages == nullptr || queue_in == nullptr || starts == nullptr || lengths_out == nullptr ||
        queue_out == nullptr || rows < 0 || (rows > 0 && (slots == nullptr || positions == nullptr || requests == nullptr))) {
        return set_error(HM_INVALID_ARGUMENT, "%s: null pointer or negative rows", what);
    }
    if (rows > INT32_MAX || Q <= 0 || Q > INT32_MAX) {
        return set_error(HM_INVALID_ARGUMENT, "%s: rows and the ring's size must fit 31 bits, the ring must not be empty (got %lld, %lld)", what,
                         static_cast<long long>(rows), static_cast<long long>(Q));
    }
    const hm::PagePlanArgs a{lengths, added, R, block_table, ld_table, W, log2_of(page_size), free_pages, Q, queue_in, slots, positions, requests,
                             rows, starts, lengths_out, queue_out};
    return launched(hm::launch_page_plan(a, reinterpret_cast<hipStream_t>(stream)), what);
}

hm_status hm_qk_norm_rope(const hm_qk_norm_rope_args *args, const hm_kv_cache *cache, void *stream) {
    const char *what = "hm_qk_norm_rope";
    if (args == nullptr) {
        return set_error(HM_INVALID_ARGUMENT, "%s: null arguments", what);
    }
    const hm_qk_norm_rope_args &p = *args;
    hm_status st = check_dtype(p.dtype, what);
    if (st != HM_OK || (cache != nullptr && (st = check_cache(cache, what)) != HM_OK)) {
        return st;
    }
    if (p.rows < 0 || p.rows > INT32_MAX || p.q_heads <= 0 || p.kv_heads <= 0 || p.q_heads > 65536 || p.kv_heads > 65536) {
        return set_error(HM_INVALID_ARGUMENT, "%s: rows must fit 31 bits, heads lie in 1..65536, got %lld, %d, %d", what, static_cast<long long>(p.rows),
                         static_cast<int>(p.q_heads), static_cast<int>(p.kv_heads));
    }
    if (p.rows > int64_t(1) << 24) { // a launch has less than 2^32 threads, 128 a row
        return set_error(HM_UNSUPPORTED, "%s: at most 2^24 rows, got %lld", what, static_cast<long long>(p.rows));
    }
    if (p.head_dim <= 0 || p.head_dim % 16 || p.head_dim > 512 || p.rotary_dim < 0 || p.rotary_dim % 16 || p.rotary_dim > p.head_dim) {
        return set_error(HM_INVALID_ARGUMENT, "%s: head_dim must be a multiple of 16 up to 512 and rotary_dim one within it, got %d, %d", what,
                         static_cast<int>(p.head_dim), static_cast<int>(p.rotary_dim));
    }
    if (cache != nullptr && (cache->dtype != p.dtype || cache->kv_heads != p.kv_heads || cache->head_dim != p.head_dim)) {
        return set_error(HM_INVALID_ARGUMENT, "%s: the cache holds %d heads of %d (dtype %d), the rows %d of %d (dtype %d)", what,
                         static_cast<int>(cache->kv_heads), static_cast<int>(cache->head_dim), static_cast<int>(cache->dtype),
                         static_cast<int>(p.kv_heads), static_cast<int>(p.head_dim), static_cast<int>(p.dtype));
    }
    if (!(p.eps >= 0.0f)) {
        return set_error(HM_INVALID_ARGUMENT, "%s: eps must not be negative", what);
    }
    if (p.rows == 0) {
        return HM_OK;
    }
    const int64_t d = p.head_dim;
    if ((st = check_rows(p.qkv, p.ldqkv, (p.q_heads + 2 * static_cast<int64_t>(p.kv_heads)) * d, what, "qkv")) != HM_OK ||
        (st = check_rows(p.q, p.ldq, p.q_heads * d, what, "q")) != HM_OK ||
        (cache == nullptr && (st = check_rows(p.k, p.ldk, p.kv_heads * d, what, "k")) != HM_OK)) {
        return st;
    }
    if (p.positions == nullptr || (p.rotary_dim > 0 && p.frequencies == nullptr) || (cache != nullptr && p.slots == nullptr) ||
        !aligned(p.bias, 16) || !aligned(p.q_weight, 16) || !aligned(p.k_weight, 16)) {
        return set_error(HM_INVALID_ARGUMENT, "%s: positions, frequencies and (with a cache) slots must be given, bias and weights 16-byte aligned", what);
    }
    hm::QkNormRopeArgs a{};
    a.qkv = static_cast<const uint16_t *>(p.qkv);
    a.ldqkv = p.ldqkv;
    a.q = static_cast<uint16_t *>(p.q);
    a.ldq = p.ldq;
    a.k = static_cast<uint16_t *>(p.k);
    a.ldk = p.ldk;
    a.bias = static_cast<const uint16_t *>(p.bias);
    a.q_weight = static_cast<const uint16_t *>(p.q_weight);
    a.k_weight = static_cast<const uint16_t *>(p.k_weight);
    a.frequencies = p.frequencies;
    a.positions = p.positions;
    if (cache != nullptr) {
        a.slots = p.slots;
        a.cache_k = static_cast<uint16_t *>(cache->k);
        a.cache_v = static_cast<uint16_t *>(cache->v);
        a.pages = cache->pages;
        a.page_stride = cache->page_stride;
        a.head_stride = cache->head_stride;
        a.token_stride = cache->token_stride;
        a.page_shift = log2_of(cache->page_size);
    }
    a.rows = p.rows;
    a.q_heads = p.q_heads;
    a.kv_heads = p.kv_heads;
    a.heads = p.q_heads + (cache != nullptr ? 2 : 1) * p.kv_heads;
    a.head_dim = p.head_dim;
    a.rotary_dim = p.rotary_dim;
    a.eps = p.eps;
    a.interleaved = p.interleaved != 0;
    a.dtype = p.dtype;
    return launched(hm::launch_qk_norm_rope(a, reinterpret_cast<hipStream_t>(stream)), what);
}

size_t hm_paged_attention_workspace_bytes(const hm_kv_cache *cache, int64_t q_heads) {
    if (cache == nullptr || cache->kv_heads <= 0 || cache->head_dim <= 0 || q_heads <= 0 || q_heads % cache->kv_heads) {
        return 0;
    }
    return hm::paged_attention_workspace(q_heads, cache->kv_heads, cache->head_dim);
}

hm_status hm_paged_attention(const hm_kv_cache *cache, void *out, int64_t ldo, const void *q, int64_t ldq, int64_t rows, int64_t q_heads,
                             const int32_t *block_table, int64_t ld_table, int64_t R, int64_t W, const int32_t *positions,
                             const int32_t *requests, float scale, int64_t window, void *workspace, size_t workspace_bytes, void *stream) {
    const char *what = "hm_paged_attention";
    hm_status st = check_cache(cache, what);
    if (st != HM_OK || (st = check_table(block_table, ld_table, R, W, cache->page_size, what)) != HM_OK) {
        return st;
    }
    const int64_t d = cache->head_dim;
    if (d != 64 && d != 96 && d != 128 && d != 256) {
        return set_error(HM_UNSUPPORTED, "%s: head_dim must be 64, 96, 128 or 256, got %lld", what, static_cast<long long>(d));
    }
    if (rows < 0 || rows > INT32_MAX || q_heads <= 0 || q_heads > 65536 || q_heads % cache->kv_heads) {
        return set_error(HM_INVALID_ARGUMENT, "%s: rows must fit 31 bits, query heads (up to 65536) be a multiple of the %d key heads, got %lld, %lld", what,
                         static_cast<int>(cache->kv_heads), static_cast<long long>(rows), static_cast<long long>(q_heads));
    }
    if (!std::isfinite(scale) || window < 0) {
        return set_error(HM_INVALID_ARGUMENT, "%s: scale must be finite and window not negative", what);
    }
    if (requests == nullptr && rows > R) {
        return set_error(HM_INVALID_ARGUMENT, "%s: %lld rows need `requests` or a table row each, the table has %lld", what, static_cast<long long>(rows),
                         static_cast<long long>(R));
    }
    // The tiles of all rows and heads are counted in 32 bits.
    const int64_t units = cache->kv_heads * ((q_heads / cache->kv_heads + 15) / 16);
    const int64_t tiles = (W * cache->page_size / 128 + 2) * units;
    if (tiles > INT32_MAX || rows > INT32_MAX / tiles) {
        return set_error(HM_UNSUPPORTED, "%s: rows * key heads * (W * page_size / 128 + 2) must stay below 2^31 (fewer rows per call)", what);
    }
    if (rows == 0) {
        return HM_OK;
    }
    if ((st = check_rows(q, ldq, q_heads * d, what, "q")) != HM_OK || (st = check_rows(out, ldo, q_heads * d, what, "out")) != HM_OK) {
        return st;
    }
    if (positions == nullptr) {
        return set_error(HM_INVALID_ARGUMENT, "%s: null positions", what);
    }
    const size_t need = hm::paged_attention_workspace(q_heads, cache->kv_heads, d);
    if (workspace == nullptr || workspace_bytes < need) {
        return set_error(HM_WORKSPACE_TOO_SMALL, "%s: workspace of %zu bytes, need %zu", what, workspace == nullptr ? size_t(0) : workspace_bytes, need);
    }
    if (!aligned(workspace, 16)) {
        return set_error(HM_INVALID_ARGUMENT, "%s: the workspace must be 16-byte aligned", what);
    }
    hm::PagedAttentionArgs a{};
    a.k = static_cast<const uint16_t *>(cache->k);
    a.v = static_cast<const uint16_t *>(cache->v);
    a.pages = cache->pages;
    a.page_stride = cache->page_stride;
    a.head_stride = cache->head_stride;
    a.token_stride = cache->token_stride;
    a.page_shift = log2_of(cache->page_size);
    a.out = static_cast<uint16_t *>(out);
    a.ldo = ldo;
    a.q = static_cast<const uint16_t *>(q);
    a.ldq = ldq;
    a.rows = rows;
    a.q_heads = static_cast<int>(q_heads);
    a.kv_heads = cache->kv_heads;
    a.head_dim = cache->head_dim;
    a.block_table = block_table;
    a.ld_table = ld_table;
    a.requests_count = R;
    a.width = W;
    a.positions = positions;
    a.requests = requests;
    a.scale = scale;
    a.window = window;
    a.workspace = workspace;
    a.dtype = cache->dtype;
    return launched(hm::launch_paged_attention(a, reinterpret_cast<hipStream_t>(stream)), what);
}

} // extern "C"
