// The Python calls' host side of the attention operators: argument checks on torch tensors and the C ABI calls, compiled. In Python
// the checks took 5 us of a call, more than a call of few rows takes now (page_plan of 64 requests 4.2 us, qk_norm_rope of a row 4.2).
// The C ABI's functions come from the library that the ctypes binding loaded (bind), so there is one of it. Host code only.
#include "hm_w4a16.h"

#include <torch/extension.h>

#include <hip/hip_runtime_api.h>

#include <optional>

namespace {

decltype(&hm_page_plan) c_page_plan = nullptr;
decltype(&hm_qk_norm_rope) c_qk_norm_rope = nullptr;
decltype(&hm_paged_attention) c_paged_attention = nullptr;
PyObject *current_stream = nullptr; // of a device index: its handle
PyObject *handle_of = nullptr;      // of a stream argument that is not None: its handle

void bind(uintptr_t page_plan, uintptr_t qk_norm_rope, uintptr_t paged_attention, py::object current, py::object handle) {
    c_page_plan = reinterpret_cast<decltype(c_page_plan)>(page_plan);
    c_qk_norm_rope = reinterpret_cast<decltype(c_qk_norm_rope)>(qk_norm_rope);
    c_paged_attention = reinterpret_cast<decltype(c_paged_attention)>(paged_attention);
    // kept until the process ends
    current_stream = current.release().ptr();
    handle_of = handle.release().ptr();
}

template <class... Parts> [[noreturn]] void refuse(const Parts &...parts) {
    std::ostringstream s;
    (s << ... << parts);
    throw py::value_error(s.str());
}

std::string described(const at::Tensor &t) {
    std::ostringstream s;
    s << t.scalar_type() << " " << t.sizes() << " with strides " << t.strides() << " on " << t.device();
    return s.str();
}

int device_of(const at::Tensor &t, const char *what) {
    if (!t.is_cuda()) {
        refuse(what, ": needs device tensors, got one on ", t.device());
    }
    return t.get_device();
}

// Address of a contiguous vector of n elements (or more).
void *vector(const at::Tensor &t, at::ScalarType type, int64_t n, int device, const char *what, const char *name, bool more = false) {
    if (t.scalar_type() != type || t.dim() != 1 || !t.is_contiguous() || (more ? t.size(0) < n : t.size(0) != n) || !t.is_cuda() || t.get_device() != device) {
        refuse(what, ": ", name, " must be a contiguous ", type, " vector of ", n, more ? " or more" : "", " elements on cuda:", device, ", got ", described(t));
    }
    return t.data_ptr();
}

void *vector(const std::optional<at::Tensor> &t, at::ScalarType type, int64_t n, int device, const char *what, const char *name, bool more = false) {
    return t.has_value() ? vector(*t, type, n, device, what, name, more) : nullptr;
}

struct Rows {
    void *p;
    int64_t ld;
};

// [rows, heads * d] or [rows, heads, d] with packed heads.
Rows row_array(const at::Tensor &t, int64_t rows, int64_t heads, int64_t d, at::ScalarType type, int device, const char *what, const char *name) {
    bool ok = t.scalar_type() == type && t.is_cuda() && t.get_device() == device;
    if (ok && t.dim() == 3) {
        ok = t.size(0) == rows && t.size(1) == heads && t.size(2) == d && t.stride(2) == 1 && (heads == 1 || t.stride(1) == d);
    } else if (ok) {
        ok = t.dim() == 2 && t.size(0) == rows && t.size(1) == heads * d && t.stride(1) == 1;
    }
    if (!ok) {
        refuse(what, ": ", name, " must be ", type, " [", rows, ", ", heads, " x ", d, "] with contiguous rows on cuda:", device, ", got ", described(t));
    }
    return {t.data_ptr(), rows > 1 ? t.stride(0) : heads * d}; // a single row's stride may be anything
}

struct Table {
    int32_t *p;
    int64_t ld, requests, width;
};

Table table_of(const at::Tensor &t, int device, const char *what) {
    if (t.scalar_type() != at::kInt || t.dim() != 2 || (t.size(1) > 1 && t.stride(1) != 1) || !t.is_cuda() || t.get_device() != device) {
        refuse(what, ": block_table must be int32 [requests, pages of a request] with contiguous rows on cuda:", device, ", got ", described(t));
    }
    return {static_cast<int32_t *>(t.data_ptr()), t.size(0) > 1 ? t.stride(0) : t.size(1), t.size(0), t.size(1)};
}

void *stream_of(py::handle stream, int device) {
    PyObject *h = nullptr;
    if (stream.is_none()) {
        const auto index = py::reinterpret_steal<py::object>(PyLong_FromLong(device));
        h = PyObject_CallOneArg(current_stream, index.ptr());
    } else {
        h = PyObject_CallOneArg(handle_of, stream.ptr());
    }
    if (h == nullptr) {
        throw py::error_already_set();
    }
    const auto owned = py::reinterpret_steal<py::object>(h);
    void *p = PyLong_AsVoidPtr(h);
    if (p == nullptr && PyErr_Occurred()) {
        throw py::error_already_set();
    }
    return p;
}

// A launch goes to the current device: the tensors' one, for as long as this lives.
class OnDevice {
  public:
    explicit OnDevice(int device) {
        if (hipGetDevice(&before_) != hipSuccess || before_ == device || hipSetDevice(device) != hipSuccess) {
            before_ = -1;
        }
    }
    ~OnDevice() {
        if (before_ >= 0) {
            (void)hipSetDevice(before_);
        }
    }
    OnDevice(const OnDevice &) = delete;
    OnDevice &operator=(const OnDevice &) = delete;

  private:
    int before_ = -1;
};

at::ScalarType type_of(int32_t dtype) { return dtype == HM_FP16 ? at::kHalf : at::kBFloat16; }

int page_plan(const at::Tensor &slots, const at::Tensor &positions, const at::Tensor &requests, const at::Tensor &starts, const at::Tensor &plan_lengths,
              const at::Tensor &plan_queue, int64_t page_size, const at::Tensor &lengths, const at::Tensor &added, const at::Tensor &block_table,
              const at::Tensor &free_pages, const at::Tensor &queue, const std::optional<at::Tensor> &lengths_out,
              const std::optional<at::Tensor> &queue_out, py::handle stream) {
    const char *what = "page_plan";
    const int device = device_of(lengths, what);
    const Table table = table_of(block_table, device, what);
    const int64_t n = table.requests, rows = slots.numel();
    if (starts.numel() != n + 1) {
        refuse("page_plan: the plan is of ", starts.numel() - 1, " requests, the table of ", n);
    }
    const at::Tensor &n_out = lengths_out.has_value() ? *lengths_out : plan_lengths, &q_out = queue_out.has_value() ? *queue_out : plan_queue;
    const auto i32 = [&](const at::Tensor &t, int64_t count, const char *name) { return static_cast<int32_t *>(vector(t, at::kInt, count, device, what, name)); };
    const auto i64 = [&](const at::Tensor &t, int64_t count, const char *name) { return static_cast<int64_t *>(vector(t, at::kLong, count, device, what, name)); };
    int32_t *ring = static_cast<int32_t *>(vector(free_pages, at::kInt, 1, device, what, "free_pages", true));
    void *s = stream_of(stream, device);
    const OnDevice on(device);
    return c_page_plan(i32(lengths, n, "lengths"), i32(added, n, "added"), n, table.p, table.ld, table.width, page_size, ring, free_pages.size(0),
                       i64(queue, 4, "queue"), i64(slots, rows, "the plan's slots"), i32(positions, rows, "the plan's positions"),
                       i32(requests, rows, "the plan's requests"), rows, i32(starts, n + 1, "the plan's starts"), i32(n_out, n, "lengths_out"),
                       i64(q_out, 4, "queue_out"), s);
}

int qk_norm_rope(const at::Tensor &q_out, const at::Tensor &qkv, const at::Tensor &frequencies, const at::Tensor &positions, uintptr_t cache,
                 int cache_device, const std::optional<at::Tensor> &slots, const std::optional<at::Tensor> &k_out, int64_t kv_heads, int64_t head_dim,
                 const std::optional<at::Tensor> &q_weight, const std::optional<at::Tensor> &k_weight, const std::optional<at::Tensor> &bias, double eps,
                 bool interleaved, py::handle stream) {
    const char *what = "qk_norm_rope";
    const int device = device_of(qkv, what);
    const at::ScalarType type = qkv.scalar_type();
    if (type != at::kHalf && type != at::kBFloat16) {
        refuse("qk_norm_rope: qkv must be bfloat16 or float16, got ", type);
    }
    const auto *c = reinterpret_cast<const hm_kv_cache *>(cache);
    if (c != nullptr) {
        if (k_out.has_value() || !slots.has_value()) {
            refuse("qk_norm_rope: a cache takes slots and no k_out");
        }
        if (type_of(c->dtype) != type || cache_device != device) {
            refuse("qk_norm_rope: the cache must be ", type, " on cuda:", device);
        }
        kv_heads = c->kv_heads, head_dim = c->head_dim;
    } else if (!k_out.has_value() || slots.has_value() || kv_heads <= 0 || head_dim <= 0) {
        refuse("qk_norm_rope: without a cache, needs k_out, kv_heads and head_dim and no slots");
    }
    if (qkv.dim() != 2 || head_dim > INT32_MAX || kv_heads > INT32_MAX || qkv.size(1) % head_dim != 0 || qkv.size(1) / head_dim <= 2 * kv_heads ||
        qkv.size(1) > INT32_MAX) {
        refuse("qk_norm_rope: qkv must be [rows, (q_heads + 2 x ", kv_heads, ") x ", head_dim, "], got ", described(qkv));
    }
    const int64_t rows = qkv.size(0), heads = qkv.size(1) / head_dim, q_heads = heads - 2 * kv_heads, pairs = frequencies.numel();
    if (pairs > head_dim / 2) {
        refuse("qk_norm_rope: ", pairs, " frequencies for heads of ", head_dim);
    }
    hm_qk_norm_rope_args a{};
    const Rows x = row_array(qkv, rows, heads, head_dim, type, device, what, "qkv"), q = row_array(q_out, rows, q_heads, head_dim, type, device, what, "q_out");
    a.qkv = x.p, a.ldqkv = x.ld, a.q = q.p, a.ldq = q.ld;
    if (c == nullptr) {
        const Rows k = row_array(*k_out, rows, kv_heads, head_dim, type, device, what, "k_out");
        a.k = k.p, a.ldk = k.ld;
    } else {
        a.slots = static_cast<const int64_t *>(vector(*slots, at::kLong, rows, device, what, "slots", true));
    }
    a.bias = vector(bias, type, heads * head_dim, device, what, "bias");
    a.q_weight = vector(q_weight, type, head_dim, device, what, "q_weight");
    a.k_weight = vector(k_weight, type, head_dim, device, what, "k_weight");
    a.frequencies = static_cast<const double *>(vector(frequencies, at::kDouble, pairs, device, what, "frequencies"));
    a.positions = static_cast<const int32_t *>(vector(positions, at::kInt, rows, device, what, "positions", true));
    a.rows = rows;
    a.q_heads = static_cast<int32_t>(q_heads), a.kv_heads = static_cast<int32_t>(kv_heads), a.head_dim = static_cast<int32_t>(head_dim);
    a.rotary_dim = static_cast<int32_t>(2 * pairs);
    a.eps = static_cast<float>(eps);
    a.interleaved = interleaved;
    a.dtype = type == at::kHalf ? HM_FP16 : HM_BF16;
    void *s = stream_of(stream, device);
    const OnDevice on(device);
    return c_qk_norm_rope(&a, c, s);
}

int paged_attention(const at::Tensor &out, const at::Tensor &q, uintptr_t cache, int device, const at::Tensor &block_table, const at::Tensor &positions,
                    const std::optional<at::Tensor> &requests, double scale, int64_t window, const std::optional<at::Tensor> &workspace,
                    py::handle stream) {
    const char *what = "paged_attention";
    const auto *c = reinterpret_cast<const hm_kv_cache *>(cache);
    const int64_t d = c->head_dim;
    if (q.dim() < 2) {
        refuse("paged_attention: q must be [rows, query heads, ", d, "], got ", described(q));
    }
    const int64_t rows = q.size(0), q_heads = q.dim() == 3 ? q.size(1) : q.size(-1) / d;
    const Rows in = row_array(q, rows, q_heads, d, type_of(c->dtype), device, what, "q"), to = row_array(out, rows, q_heads, d, type_of(c->dtype), device, what, "out");
    const Table table = table_of(block_table, device, what);
    const auto *pos = static_cast<const int32_t *>(vector(positions, at::kInt, rows, device, what, "positions", true));
    const auto *req = static_cast<const int32_t *>(vector(requests, at::kInt, rows, device, what, "requests", true));
    uintptr_t aligned = 0; // without a workspace the call itself refuses
    size_t bytes = 0;
    if (workspace.has_value()) {
        if (!workspace->is_cuda() || workspace->get_device() != device || !workspace->is_contiguous()) {
            refuse("paged_attention: the workspace must be a contiguous tensor on cuda:", device, ", got ", described(*workspace));
        }
        const uintptr_t base = reinterpret_cast<uintptr_t>(workspace->data_ptr());
        aligned = (base + 255) / 256 * 256;
        bytes = workspace->nbytes() > aligned - base ? workspace->nbytes() - (aligned - base) : 0;
    }
    void *s = stream_of(stream, device);
    const OnDevice on(device);
    return c_paged_attention(c, to.p, to.ld, in.p, in.ld, rows, q_heads, table.p, table.ld, table.requests, table.width, pos, req, static_cast<float>(scale), window,
                             reinterpret_cast<void *>(aligned), bytes, s);
}

} // namespace

PYBIND11_MODULE(TORCH_EXTENSION_NAME, m) {
    m.doc() = "Checks and calls of the attention operators over a paged cache (heteromega_amd/attention.py)";
    m.def("bind", &bind);
    m.def("page_plan", &page_plan);
    m.def("qk_norm_rope", &qk_norm_rope);
    m.def("paged_attention", &paged_attention);
}
