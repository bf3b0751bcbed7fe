// The Python calls' host side of the operators for requests that branch (heteromega_amd/branches.py): argument checks on torch tensors and the C ABI calls, as
// hm_attention_host.cpp has them for the attention operators. Host code only.
#include "hm_host_checks.hpp"

#include <vector>

namespace {

using namespace hm_host;

decltype(&hm_beam_select) c_beam_select = nullptr;
decltype(&hm_page_fork) c_page_fork = nullptr;
decltype(&hm_page_compact) c_page_compact = nullptr;
decltype(&hm_copy_pages) c_copy_pages = nullptr;
decltype(&hm_share_plan) c_share_plan = nullptr;
decltype(&hm_shared_attention) c_shared_attention = nullptr;

void bind_branches(uintptr_t beam_select, uintptr_t page_fork, uintptr_t page_compact, uintptr_t copy_pages, uintptr_t share_plan, uintptr_t shared_attention) {
    c_beam_select = reinterpret_cast<decltype(c_beam_select)>(beam_select);
    c_page_fork = reinterpret_cast<decltype(c_page_fork)>(page_fork);
    c_page_compact = reinterpret_cast<decltype(c_page_compact)>(page_compact);
    c_copy_pages = reinterpret_cast<decltype(c_copy_pages)>(copy_pages);
    c_share_plan = reinterpret_cast<decltype(c_share_plan)>(share_plan);
    c_shared_attention = reinterpret_cast<decltype(c_shared_attention)>(shared_attention);
}

// Address of a contiguous [rows, columns] array.
void *matrix(const at::Tensor &t, at::ScalarType type, int64_t rows, int64_t columns, int device, const char *what, const char *name) {
    if (t.scalar_type() != type || t.dim() != 2 || t.size(0) != rows || t.size(1) != columns || !t.is_contiguous() || !t.is_cuda() || t.get_device() != device) {
        refuse(what, ": ", name, " must be a contiguous ", type, " [", rows, ", ", columns, "] on cuda:", device, ", got ", described(t));
    }
    return t.data_ptr();
}

int32_t *ints(const at::Tensor &t, int64_t n, int device, const char *what, const char *name, bool more = false) {
    return static_cast<int32_t *>(vector(t, at::kInt, n, device, what, name, more));
}

int64_t *counters(const at::Tensor &t, int device, const char *what, const char *name) {
    return static_cast<int64_t *>(vector(t, at::kLong, 4, device, what, name));
}

// The table that is written: the one that is read, or another of its size.
Table table_out_of(const std::optional<at::Tensor> &t, const Table &in, int device, const char *what) {
    if (!t.has_value()) {
        return in;
    }
    const Table out = table_of(*t, device, what);
    if (out.requests != in.requests || out.width != in.width) {
        refuse(what, ": table_out must be [", in.requests, ", ", in.width, "], got ", described(*t));
    }
    return out;
}

int beam_select(const at::Tensor &parents, const at::Tensor &tokens, const at::Tensor &scores_out, const at::Tensor &ended_out, const at::Tensor &workspace,
                int64_t requests, int64_t beams, int64_t vocabulary, int64_t k, const at::Tensor &logits, const at::Tensor &scores,
                const std::optional<at::Tensor> &ended, int64_t end_token, py::handle stream) {
    const char *what = "beam_select";
    const int device = device_of(logits, what);
    const at::ScalarType type = logits.scalar_type();
    const int64_t rows = requests * beams;
    if ((type != at::kHalf && type != at::kBFloat16 && type != at::kFloat) || logits.dim() != 2 || logits.size(0) != rows || logits.size(1) != vocabulary ||
        (vocabulary > 1 && logits.stride(1) != 1)) {
        refuse("beam_select: logits must be float16, bfloat16 or float32 [", rows, ", ", vocabulary, "] with contiguous rows, got ", described(logits));
    }
    const Workspace ws = workspace_of(workspace, device, what);
    auto *parents_at = static_cast<int32_t *>(matrix(parents, at::kInt, requests, k, device, what, "the step's parents"));
    auto *tokens_at = static_cast<int32_t *>(matrix(tokens, at::kInt, requests, k, device, what, "the step's tokens"));
    auto *scores_at = static_cast<float *>(matrix(scores_out, at::kFloat, requests, k, device, what, "the step's scores"));
    auto *ended_at = static_cast<uint8_t *>(matrix(ended_out, at::kBool, requests, k, device, what, "the step's ended"));
    void *s = stream_of(stream, device);
    const OnDevice on(device);
    return c_beam_select(logits.data_ptr(), rows > 1 ? logits.stride(0) : vocabulary, type == at::kHalf ? HM_FP16 : type == at::kBFloat16 ? HM_BF16 : HM_LOGITS_FP32,
                         static_cast<const float *>(vector(scores, at::kFloat, rows, device, what, "scores")),
                         static_cast<const uint8_t *>(vector(ended, at::kBool, rows, device, what, "ended")), end_token, requests, beams, vocabulary, k, parents_at,
                         tokens_at, scores_at, ended_at, ws.p, ws.bytes, s);
}

int page_fork(const at::Tensor &copies, const at::Tensor &fork_lengths, const at::Tensor &fork_queue, const at::Tensor &workspace, int64_t page_size,
              const at::Tensor &sources, const at::Tensor &lengths, const at::Tensor &block_table, const at::Tensor &free_pages, const at::Tensor &queue,
              const std::optional<at::Tensor> &keep, const std::optional<at::Tensor> &table_out, const std::optional<at::Tensor> &lengths_out,
              const std::optional<at::Tensor> &queue_out, py::handle stream) {
    const char *what = "page_fork";
    const int device = device_of(lengths, what);
    const Table table = table_of(block_table, device, what), to = table_out_of(table_out, table, device, what);
    const int64_t n = table.requests;
    const Workspace ws = workspace_of(workspace, device, what);
    const auto *source_at = ints(sources, n, device, what, "sources");
    const auto *keep_at = keep.has_value() ? ints(*keep, n, device, what, "keep") : nullptr;
    const auto *lengths_at = ints(lengths, n, device, what, "lengths");
    auto *ring = ints(free_pages, 1, device, what, "free_pages", true);
    const auto *queue_at = counters(queue, device, what, "queue");
    auto *copies_at = static_cast<int32_t *>(matrix(copies, at::kInt, n, 3, device, what, "the fork's copies"));
    auto *lengths_to = ints(lengths_out.has_value() ? *lengths_out : fork_lengths, n, device, what, "lengths_out");
    auto *queue_to = counters(queue_out.has_value() ? *queue_out : fork_queue, device, what, "queue_out");
    void *s = stream_of(stream, device);
    const OnDevice on(device);
    return c_page_fork(source_at, keep_at, lengths_at, n, table.p, table.ld, to.p, to.ld, table.width, page_size, ring, free_pages.size(0), queue_at, copies_at,
                       lengths_to, queue_to, ws.p, ws.bytes, s);
}

int page_compact(const at::Tensor &copies, const at::Tensor &compact_queue, const at::Tensor &workspace, int64_t pages, int64_t page_size, int64_t limit,
                 const at::Tensor &lengths, const at::Tensor &block_table, const at::Tensor &free_pages, const at::Tensor &queue,
                 const std::optional<at::Tensor> &table_out, const std::optional<at::Tensor> &queue_out, py::handle stream) {
    const char *what = "page_compact";
    const int device = device_of(lengths, what);
    const Table table = table_of(block_table, device, what), to = table_out_of(table_out, table, device, what);
    const Workspace ws = workspace_of(workspace, device, what);
    const auto *lengths_at = ints(lengths, table.requests, device, what, "lengths");
    auto *ring = ints(free_pages, 1, device, what, "free_pages", true);
    const auto *queue_at = counters(queue, device, what, "queue");
    auto *copies_at = static_cast<int32_t *>(matrix(copies, at::kInt, copies.size(0), 3, device, what, "the plan's copies"));
    auto *queue_to = counters(queue_out.has_value() ? *queue_out : compact_queue, device, what, "queue_out");
    void *s = stream_of(stream, device);
    const OnDevice on(device);
    return c_page_compact(pages, limit, lengths_at, table.requests, table.p, table.ld, to.p, to.ld, table.width, page_size, ring, free_pages.size(0), queue_at,
                          copies_at, copies.size(0), queue_to, ws.p, ws.bytes, s);
}

int copy_pages(const std::vector<uintptr_t> &from, const std::vector<uintptr_t> &to, int device, const at::Tensor &copies, py::handle stream) {
    const char *what = "copy_pages";
    if (copies.dim() != 2) {
        refuse("copy_pages: copies must be int32 [n, 3], got ", described(copies));
    }
    const auto *copies_at = static_cast<const int32_t *>(matrix(copies, at::kInt, copies.size(0), 3, device, what, "copies"));
    std::vector<hm_kv_cache> source, target;
    for (const uintptr_t c : from) {
        source.push_back(*reinterpret_cast<const hm_kv_cache *>(c));
    }
    for (const uintptr_t c : to) {
        target.push_back(*reinterpret_cast<const hm_kv_cache *>(c));
    }
    void *s = stream_of(stream, device);
    const OnDevice on(device);
    return c_copy_pages(source.data(), target.empty() ? nullptr : target.data(), static_cast<int64_t>(source.size()), copies_at, copies.size(0), s);
}

int share_plan(const at::Tensor &shared, const at::Tensor &plan, int64_t page_size, int64_t q_heads, int64_t kv_heads, int64_t window, const at::Tensor &block_table,
               const at::Tensor &positions, const std::optional<at::Tensor> &requests, py::handle stream) {
    const char *what = "share_plan";
    const int device = device_of(block_table, what);
    const Table table = table_of(block_table, device, what);
    const int64_t rows = shared.numel();
    auto *shared_at = ints(shared, rows, device, what, "the plan's shared");
    const auto *pos = ints(positions, rows, device, what, "positions", true);
    const auto *req = requests.has_value() ? ints(*requests, rows, device, what, "requests", true) : nullptr;
    const Workspace ws = workspace_of(plan, device, what);
    void *s = stream_of(stream, device);
    const OnDevice on(device);
    return c_share_plan(table.p, table.ld, table.requests, table.width, page_size, pos, req, rows, q_heads, kv_heads, window, shared_at, ws.p, ws.bytes, s);
}

int shared_attention(const at::Tensor &out, const at::Tensor &q, uintptr_t cache, int device, const at::Tensor &block_table, const at::Tensor &positions,
                     const std::optional<at::Tensor> &requests, double scale, int64_t plan_rows, int64_t plan_q_heads, int64_t plan_kv_heads, int64_t page_size,
                     const at::Tensor &plan, const at::Tensor &workspace, py::handle stream) {
    const char *what = "shared_attention";
    const auto *c = reinterpret_cast<const hm_kv_cache *>(cache);
    const int64_t d = c->head_dim;
    if (q.dim() < 2) {
        refuse("shared_attention: q must be [rows, query heads, ", d, "], got ", described(q));
    }
    const int64_t rows = q.size(0), q_heads = q.dim() == 3 ? q.size(1) : q.size(-1) / d;
    if (rows != plan_rows || q_heads != plan_q_heads || c->kv_heads != plan_kv_heads || c->page_size != page_size) {
        refuse("shared_attention: the plan is of ", plan_rows, " rows, ", plan_q_heads, " / ", plan_kv_heads, " heads and pages of ", page_size, ", the call of ", rows,
               " rows, ", q_heads, " / ", c->kv_heads, " heads and pages of ", c->page_size);
    }
    const Rows in = row_array(q, rows, q_heads, d, type_of(c->dtype), device, what, "q"), to = row_array(out, rows, q_heads, d, type_of(c->dtype), device, what, "out");
    const Table table = table_of(block_table, device, what);
    const auto *pos = ints(positions, rows, device, what, "positions", true);
    const auto *req = requests.has_value() ? ints(*requests, rows, device, what, "requests", true) : nullptr;
    const Workspace made = workspace_of(plan, device, what), ws = workspace_of(workspace, device, what);
    void *s = stream_of(stream, device);
    const OnDevice on(device);
    return c_shared_attention(c, to.p, to.ld, in.p, in.ld, rows, q_heads, table.p, table.ld, table.requests, table.width, pos, req, static_cast<float>(scale), made.p,
                              made.bytes, ws.p, ws.bytes, s);
}

} // namespace

void hm_host::def_branches(py::module_ &m) {
    m.def("bind_branches", &bind_branches);
    m.def("beam_select", &beam_select);
    m.def("page_fork", &page_fork);
    m.def("page_compact", &page_compact);
    m.def("copy_pages", &copy_pages);
    m.def("share_plan", &share_plan);
    m.def("shared_attention", &shared_attention);
}
