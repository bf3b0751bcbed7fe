// Checks of arguments that the C ABI's calls on a paged cache share (hm_attention_api.cpp, hm_branch_api.cpp).
#pragma once

#include "../../include/hm_w4a16.h"
#include "hm_internal.hpp"

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
    // Positions are 32-bit; the attention's tiles may begin up to 15 tokens early and end up to 160 late.
    if (W > (INT32_MAX - 256) / page_size) {
        return set_error(HM_UNSUPPORTED, "%s: W * page_size must stay below 2^31 - 256 tokens, got %lld * %lld", what, static_cast<long long>(W),
                         static_cast<long long>(page_size));
    }
    return HM_OK;
}

// What the attention calls have in common; the window is 0.
void fill_attention_args(hm::PagedAttentionArgs &a, const hm_kv_cache &cache, void *out, int64_t ldo, const void *q, int64_t ldq, int64_t rows, int64_t q_heads,
                         const int32_t *block_table, int64_t ld_table, int64_t R, int64_t W, const int32_t *positions, const int32_t *requests, float scale,
                         void *workspace) {
    a.k = static_cast<const uint16_t *>(cache.k);
    a.v = static_cast<const uint16_t *>(cache.v);
    a.pages = cache.pages;
    a.page_stride = cache.page_stride;
    a.head_stride = cache.head_stride;
    a.token_stride = cache.token_stride;
    a.page_shift = log2_of(cache.page_size);
    a.out = static_cast<uint16_t *>(out);
    a.ldo = ldo;
    a.q = static_cast<const uint16_t *>(q);
    a.ldq = ldq;
    a.rows = rows;
    a.q_heads = static_cast<int>(q_heads);
    a.kv_heads = cache.kv_heads;
    a.head_dim = cache.head_dim;
    a.block_table = block_table;
    a.ld_table = ld_table;
    a.requests_count = R;
    a.width = W;
    a.positions = positions;
    a.requests = requests;
    a.scale = scale;
    a.window = 0;
    a.workspace = workspace;
    a.dtype = cache.dtype;
}

} // namespace
