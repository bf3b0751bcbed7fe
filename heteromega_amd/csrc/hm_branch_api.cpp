// C ABI of the operators for requests that branch over a paged cache (include/hm_w4a16.h): validation and dispatch.
#include "hm_cache_checks.hpp"
#include "hm_shared_attention.hpp"

#include <algorithm>
#include <cmath>

namespace {

hm_status check_ring(const int32_t *free_pages, int64_t Q, const int64_t *queue_in, const int64_t *queue_out, const char *what) {
    if (free_pages == nullptr || queue_in == nullptr || queue_out == nullptr || Q <= 0 || Q > INT32_MAX) {
        return set_error(HM_INVALID_ARGUMENT, "%s: the ring of free pages and its counters must be given, with 1 to 2^31 - 1 entries, got %lld", what,
                         static_cast<long long>(Q));
    }
    return HM_OK;
}

hm_status check_workspace(const void *workspace, size_t bytes, size_t need, const char *what) {
    if (workspace == nullptr || bytes < need) {
        return set_error(HM_WORKSPACE_TOO_SMALL, "%s: workspace of %zu bytes, need %zu", what, workspace == nullptr ? size_t(0) : bytes, need);
    }
    if (!aligned(workspace, 16)) {
        return set_error(HM_INVALID_ARGUMENT, "%s: the workspace must be 16-byte aligned", what);
    }
    return HM_OK;
}

hm_status check_beams(int64_t R, int64_t beams, int64_t V, int64_t k, int32_t logits_dtype, const char *what) {
    if (logits_dtype != HM_BF16 && logits_dtype != HM_FP16 && logits_dtype != HM_LOGITS_FP32) {
        return set_error(HM_INVALID_ARGUMENT, "%s: logits must be HM_BF16, HM_FP16 or HM_LOGITS_FP32, got %d", what, static_cast<int>(logits_dtype));
    }
    if (R <= 0 || beams <= 0 || V <= 0 || k <= 0 || beams > HM_BEAM_MAX_BEAMS || k > HM_BEAM_MAX_K) {
        return set_error(HM_INVALID_ARGUMENT, "%s: needs requests, 1 to %d beams, a vocabulary and k of 1 to %d, got %lld, %lld, %lld, %lld", what,
                         HM_BEAM_MAX_BEAMS, HM_BEAM_MAX_K, static_cast<long long>(R), static_cast<long long>(beams), static_cast<long long>(V),
                         static_cast<long long>(k));
    }
    if (V > int64_t(1) << 24 || R > 65535 / beams) { // a launch's grid, and 31-bit places of a request's candidates
        return set_error(HM_UNSUPPORTED, "%s: at most 65535 rows and 2^24 tokens, got %lld x %lld, %lld", what, static_cast<long long>(R),
                         static_cast<long long>(beams), static_cast<long long>(V));
    }
    return HM_OK;
}

// Rows and heads that a plan of shared pages takes, with a table of W blocks.
hm_status check_share(int64_t rows, int64_t q_heads, int64_t kv_heads, int64_t W, int64_t page_size, const char *what) {
    if (rows < 0 || rows > HM_SHARE_MAX_ROWS) {
        return set_error(rows < 0 ? HM_INVALID_ARGUMENT : HM_UNSUPPORTED, "%s: at most %d rows, got %lld", what, HM_SHARE_MAX_ROWS, static_cast<long long>(rows));
    }
    if (kv_heads <= 0 || q_heads <= 0 || q_heads > 65536 || q_heads % kv_heads) {
        return set_error(HM_INVALID_ARGUMENT, "%s: query heads (up to 65536) must be a multiple of key heads, got %lld and %lld", what,
                         static_cast<long long>(q_heads), static_cast<long long>(kv_heads));
    }
    if (q_heads / kv_heads > hm::kWideCols) {
        return set_error(HM_UNSUPPORTED, "%s: at most %d query heads to a key head, got %lld", what, hm::kWideCols, static_cast<long long>(q_heads / kv_heads));
    }
    static_assert(hm::kNarrowTile == 32 && hm::kWideTile == 32, "the refusal names their length");
    const int64_t tiles = (W * page_size / 32 + 2) * kv_heads; // all tiles are counted in 32 bits
    if (tiles > INT32_MAX || 5 * rows > INT32_MAX / tiles) {
        return set_error(HM_UNSUPPORTED, "%s: 5 * rows * key heads * (W * page_size / 32 + 2) must stay below 2^31 (fewer rows per call)", what);
    }
    return HM_OK;
}

// A table that is read and one that is written, which are apart or one and the same.
hm_status check_tables(const int32_t *in, int64_t ld_in, const int32_t *out, int64_t ld_out, int64_t R, int64_t W, int64_t page_size, const char *what) {
    const hm_status st = check_table(in, ld_in, R, W, page_size, what);
    if (st != HM_OK) {
        return st;
    }
    if (out == nullptr || ld_out < W || (out == in && ld_out != ld_in)) {
        return set_error(HM_INVALID_ARGUMENT, "%s: table_out must be a table of the same size, or block_table itself", what);
    }
    return HM_OK;
}

} // namespace

extern "C" {

size_t hm_beam_select_workspace_bytes(int64_t R, int64_t beams, int64_t V, int64_t k, int32_t logits_dtype) {
    if (check_beams(R, beams, V, k, logits_dtype, "hm_beam_select_workspace_bytes") != HM_OK) {
        return 0;
    }
    return hm::beam_select_workspace(R * beams, V, k);
}

hm_status hm_beam_select(const void *logits, int64_t ld, int32_t logits_dtype, const float *scores, const uint8_t *ended, int64_t end_token, int64_t R,
                         int64_t beams, int64_t V, int64_t k, int32_t *parents, int32_t *tokens, float *scores_out, uint8_t *ended_out, void *workspace,
                         size_t workspace_bytes, void *stream) {
    const char *what = "hm_beam_select";
    hm_status st = check_beams(R, beams, V, k, logits_dtype, what);
    if (st != HM_OK) {
        return st;
    }
    if (logits == nullptr || scores == nullptr || parents == nullptr || tokens == nullptr || scores_out == nullptr || ended_out == nullptr || ld < V ||
        !aligned(logits, logits_dtype == HM_LOGITS_FP32 ? 4 : 2)) {
        return set_error(HM_INVALID_ARGUMENT, "%s: null pointer, logits that are not aligned to their type, or a leading dimension below %lld (got %lld)", what,
                         static_cast<long long>(V), static_cast<long long>(ld));
    }
    if (end_token < (ended == nullptr ? -1 : 0) || end_token >= V) {
        return set_error(HM_INVALID_ARGUMENT, "%s: end_token must be one of %lld tokens (or, without `ended`, -1), got %lld", what, static_cast<long long>(V),
                         static_cast<long long>(end_token));
    }
    if (k != beams && (scores_out == scores || ended_out == ended)) {
        return set_error(HM_INVALID_ARGUMENT, "%s: results may take the place of scores and ended only where k is the number of beams", what);
    }
    if ((st = check_workspace(workspace, workspace_bytes, hm::beam_select_workspace(R * beams, V, k), what)) != HM_OK) {
        return st;
    }
    const hm::BeamSelectArgs a{logits, ld, logits_dtype, scores, ended, static_cast<int32_t>(end_token), R * beams, static_cast<int>(beams), V,
                               static_cast<int>(k), parents, tokens, scores_out, ended_out, workspace, 0};
    return launched(hm::launch_beam_select(a, reinterpret_cast<hipStream_t>(stream)), what);
}

size_t hm_page_fork_workspace_bytes(int64_t R, int64_t W) { return R <= 0 || W <= 0 ? 0 : hm::page_fork_workspace(R); }

hm_status hm_page_fork(const int32_t *sources, const int32_t *keep, const int32_t *lengths, int64_t R, const int32_t *block_table, int64_t ld_table,
                       int32_t *table_out, int64_t ld_out, int64_t W, int64_t page_size, int32_t *free_pages, int64_t Q, const int64_t *queue_in,
                       int32_t *copies, int32_t *lengths_out, int64_t *queue_out, void *workspace, size_t workspace_bytes, void *stream) {
    const char *what = "hm_page_fork";
    hm_status st = check_page_size(page_size, what);
    if (st != HM_OK || (st = check_tables(block_table, ld_table, table_out, ld_out, R, W, page_size, what)) != HM_OK ||
        (st = check_ring(free_pages, Q, queue_in, queue_out, what)) != HM_OK) {
        return st;
    }
    if (R > HM_PAGE_PLAN_MAX_REQUESTS) {
        return set_error(HM_UNSUPPORTED, "%s: at most %d requests, got %lld", what, HM_PAGE_PLAN_MAX_REQUESTS, static_cast<long long>(R));
    }
    if (sources == nullptr || lengths == nullptr || copies == nullptr || lengths_out == nullptr) {
        return set_error(HM_INVALID_ARGUMENT, "%s: null pointer", what);
    }
    if ((st = check_workspace(workspace, workspace_bytes, hm::page_fork_workspace(R), what)) != HM_OK) {
        return st;
    }
    const hm::PageForkArgs a{sources, keep, lengths, R, block_table, ld_table, table_out, ld_out, W, log2_of(page_size), free_pages, Q, queue_in,
                             copies, lengths_out, queue_out, workspace, 0};
    return launched(hm::launch_page_fork(a, reinterpret_cast<hipStream_t>(stream)), what);
}

size_t hm_page_compact_workspace_bytes(int64_t pages) { return pages <= 0 ? 0 : hm::page_compact_workspace(pages); }

hm_status hm_page_compact(int64_t pages, int64_t limit, const int32_t *lengths, int64_t R, const int32_t *block_table, int64_t ld_table, int32_t *table_out,
                          int64_t ld_out, int64_t W, int64_t page_size, int32_t *free_pages, int64_t Q, const int64_t *queue_in, int32_t *copies, int64_t n,
                          int64_t *queue_out, void *workspace, size_t workspace_bytes, void *stream) {
    const char *what = "hm_page_compact";
    hm_status st = check_page_size(page_size, what);
    if (st != HM_OK || (st = check_tables(block_table, ld_table, table_out, ld_out, R, W, page_size, what)) != HM_OK ||
        (st = check_ring(free_pages, Q, queue_in, queue_out, what)) != HM_OK) {
        return st;
    }
    if (pages <= 0 || pages > INT32_MAX - 64 || limit < 0 || limit > pages) {
        return set_error(HM_INVALID_ARGUMENT, "%s: a cache has 1 to 2^31 - 65 pages and the limit lies within them, got %lld, %lld", what,
                         static_cast<long long>(pages), static_cast<long long>(limit));
    }
    if (lengths == nullptr || copies == nullptr || n < std::max<int64_t>(1, std::min(limit, pages - limit))) {
        return set_error(HM_INVALID_ARGUMENT, "%s: lengths and copies must be given, copies with an entry for each page that may move (%lld), got %lld", what,
                         static_cast<long long>(std::max<int64_t>(1, std::min(limit, pages - limit))), static_cast<long long>(n));
    }
    if ((st = check_workspace(workspace, workspace_bytes, hm::page_compact_workspace(pages), what)) != HM_OK) {
        return st;
    }
    const hm::PageCompactArgs a{pages, limit, lengths, R, block_table, ld_table, table_out, ld_out, W, log2_of(page_size), free_pages, Q, queue_in,
                                copies, n, queue_out, workspace};
    return launched(hm::launch_page_compact(a, reinterpret_cast<hipStream_t>(stream)), what);
}

hm_status hm_copy_pages(const hm_kv_cache *from, const hm_kv_cache *to, int64_t layers, const int32_t *copies, int64_t n, void *stream) {
    const char *what = "hm_copy_pages";
    if (from == nullptr || layers <= 0 || n < 0 || n > INT32_MAX || (n > 0 && copies == nullptr)) {
        return set_error(HM_INVALID_ARGUMENT, "%s: caches and copies must be given (up to 2^31 - 1), got %lld layers, %lld copies", what,
                         static_cast<long long>(layers), static_cast<long long>(n));
    }
    to = to != nullptr ? to : from;
    for (int64_t i = 0; i < layers; ++i) {
        for (const hm_kv_cache *c : {from + i, to + i}) {
            const hm_status st = check_cache(c, what);
            if (st != HM_OK) {
                return st;
            }
            const hm_kv_cache &first = c == from + i ? from[0] : to[0];
            if (c->kv_heads != from[0].kv_heads || c->head_dim != from[0].head_dim || c->dtype != from[0].dtype || c->page_size != from[0].page_size) {
                return set_error(HM_INVALID_ARGUMENT, "%s: the caches must be alike in heads, type and page size", what);
            }
            if (c->pages != first.pages || c->page_stride != first.page_stride || c->head_stride != first.head_stride || c->token_stride != first.token_stride) {
                return set_error(HM_INVALID_ARGUMENT, "%s: the layers' caches must be alike in pages and strides", what);
            }
        }
    }
    hm::CopyPagesArgs a{};
    a.from_pages = from->pages, a.from_page = from->page_stride, a.from_head = from->head_stride, a.from_token = from->token_stride;
    a.to_pages = to->pages, a.to_page = to->page_stride, a.to_head = to->head_stride, a.to_token = to->token_stride;
    a.kv_heads = from->kv_heads, a.head_dim = from->head_dim, a.page_shift = log2_of(from->page_size);
    a.copies = copies;
    a.count = n;
    for (int64_t at = 0; n > 0 && at < layers; at += a.layers) {
        a.layers = static_cast<int>(std::min<int64_t>(hm::kCopyLayers, layers - at));
        for (int i = 0; i < a.layers; ++i) {
            a.from_k[i] = static_cast<const uint16_t *>(from[at + i].k), a.from_v[i] = static_cast<const uint16_t *>(from[at + i].v);
            a.to_k[i] = static_cast<uint16_t *>(to[at + i].k), a.to_v[i] = static_cast<uint16_t *>(to[at + i].v);
        }
        const hm_status st = launched(hm::launch_copy_pages(a, reinterpret_cast<hipStream_t>(stream)), what);
        if (st != HM_OK) {
            return st;
        }
    }
    return HM_OK;
}

size_t hm_share_plan_bytes(int64_t rows) { return rows < 0 || rows > HM_SHARE_MAX_ROWS ? 0 : hm::share_plan_workspace(rows); }

hm_status hm_share_plan(const int32_t *block_table, int64_t ld_table, int64_t R, int64_t W, int64_t page_size, const int32_t *positions, const int32_t *requests,
                        int64_t rows, int64_t q_heads, int64_t kv_heads, int64_t window, int32_t *shared, void *plan, size_t plan_bytes, void *stream) {
    const char *what = "hm_share_plan";
    hm_status st = check_page_size(page_size, what);
    if (st != HM_OK || (st = check_table(block_table, ld_table, R, W, page_size, what)) != HM_OK ||
        (st = check_share(rows, q_heads, kv_heads, W, page_size, what)) != HM_OK) {
        return st;
    }
    if (window < 0) {
        return set_error(HM_INVALID_ARGUMENT, "%s: window must not be negative", what);
    }
    if (requests == nullptr && rows > R) {
        return set_error(HM_INVALID_ARGUMENT, "%s: %lld rows need `requests` or a table row each, the table has %lld", what, static_cast<long long>(rows),
                         static_cast<long long>(R));
    }
    if (rows == 0) {
        return HM_OK;
    }
    if (positions == nullptr || shared == nullptr) {
        return set_error(HM_INVALID_ARGUMENT, "%s: null pointer", what);
    }
    if ((st = check_workspace(plan, plan_bytes, hm::share_plan_workspace(rows), what)) != HM_OK) {
        return st;
    }
    const hm::SharePlanArgs a{block_table, ld_table, R, W, log2_of(page_size), positions, requests, rows, static_cast<int>(q_heads / kv_heads),
                              static_cast<int>(kv_heads), window, shared, plan, 0};
    return launched(hm::launch_share_plan(a, reinterpret_cast<hipStream_t>(stream)), what);
}

size_t hm_shared_attention_workspace_bytes(const hm_kv_cache *cache, int64_t q_heads, int64_t rows) {
    if (cache == nullptr || cache->kv_heads <= 0 || cache->head_dim <= 0 || q_heads <= 0 || q_heads % cache->kv_heads || rows < 0 || rows > HM_SHARE_MAX_ROWS) {
        return 0;
    }
    return hm::shared_attention_workspace(rows, q_heads, cache->head_dim);
}

hm_status hm_shared_attention(const hm_kv_cache *cache, void *out, int64_t ldo, const void *q, int64_t ldq, int64_t rows, int64_t q_heads,
                              const int32_t *block_table, int64_t ld_table, int64_t R, int64_t W, const int32_t *positions, const int32_t *requests, float scale,
                              const void *plan, size_t plan_bytes, void *workspace, size_t workspace_bytes, void *stream) {
    const char *what = "hm_shared_attention";
    hm_status st = check_cache(cache, what);
    if (st != HM_OK || (st = check_table(block_table, ld_table, R, W, cache->page_size, what)) != HM_OK) {
        return st;
    }
    const int64_t d = cache->head_dim;
    if (d != 64 && d != 96 && d != 128 && d != 256) {
        return set_error(HM_UNSUPPORTED, "%s: head_dim must be 64, 96, 128 or 256, got %lld", what, static_cast<long long>(d));
    }
    if ((st = check_share(rows, q_heads, cache->kv_heads, W, cache->page_size, what)) != HM_OK) {
        return st;
    }
    if (!std::isfinite(scale)) {
        return set_error(HM_INVALID_ARGUMENT, "%s: scale must be finite", what);
    }
    if (requests == nullptr && rows > R) {
        return set_error(HM_INVALID_ARGUMENT, "%s: %lld rows need `requests` or a table row each, the table has %lld", what, static_cast<long long>(rows),
                         static_cast<long long>(R));
    }
    if (rows == 0) {
        return HM_OK;
    }
    if ((st = check_rows(q, ldq, q_heads * d, what, "q")) != HM_OK || (st = check_rows(out, ldo, q_heads * d, what, "out")) != HM_OK) {
        return st;
    }
    if (positions == nullptr || plan == nullptr || plan_bytes < hm::share_plan_workspace(rows) || !aligned(plan, 16)) {
        return set_error(HM_INVALID_ARGUMENT, "%s: positions and a plan of %lld rows (16-byte aligned) must be given", what, static_cast<long long>(rows));
    }
    if ((st = check_workspace(workspace, workspace_bytes, hm::shared_attention_workspace(rows, q_heads, d), what)) != HM_OK) {
        return st;
    }
    hm::SharedAttentionArgs a{};
    fill_attention_args(a, *cache, out, ldo, q, ldq, rows, q_heads, block_table, ld_table, R, W, positions, requests, scale, workspace);
    a.plan = const_cast<void *>(plan);
    a.group_heads = static_cast<int>(q_heads / cache->kv_heads);
    return launched(hm::launch_shared_attention(a, reinterpret_cast<hipStream_t>(stream)), what);
}

} // extern "C"
