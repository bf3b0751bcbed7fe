// Checks of torch tensors that the compiled host side of the Python calls shares (hm_attention_host.cpp, hm_branch_host.cpp). Host code only.
#pragma once

#include "hm_w4a16.h"

#include <torch/extension.h>

#include <hip/hip_runtime_api.h>

#include <optional>

namespace hm_host {

inline PyObject *current_stream = nullptr; // of a device index: its handle
inline PyObject *handle_of = nullptr;      // of a stream argument that is not None: its handle

template <class... Parts> [[noreturn]] void refuse(const Parts &...parts) {
    std::ostringstream s;
    (s << ... << parts);
    throw py::value_error(s.str());
}

inline std::string described(const at::Tensor &t) {
    std::ostringstream s;
    s << t.scalar_type() << " " << t.sizes() << " with strides " << t.strides() << " on " << t.device();
    return s.str();
}

inline int device_of(const at::Tensor &t, const char *what) {
    if (!t.is_cuda()) {
        refuse(what, ": needs device tensors, got one on ", t.device());
    }
    return t.get_device();
}

// Address of a contiguous vector of n elements (or more).
inline void *vector(const at::Tensor &t, at::ScalarType type, int64_t n, int device, const char *what, const char *name, bool more = false) {
    if (t.scalar_type() != type || t.dim() != 1 || !t.is_contiguous() || (more ? t.size(0) < n : t.size(0) != n) || !t.is_cuda() || t.get_device() != device) {
        refuse(what, ": ", name, " must be a contiguous ", type, " vector of ", n, more ? " or more" : "", " elements on cuda:", device, ", got ", described(t));
    }
    return t.data_ptr();
}

inline void *vector(const std::optional<at::Tensor> &t, at::ScalarType type, int64_t n, int device, const char *what, const char *name, bool more = false) {
    return t.has_value() ? vector(*t, type, n, device, what, name, more) : nullptr;
}

struct Rows {
    void *p;
    int64_t ld;
};

// [rows, heads * d] or [rows, heads, d] with packed heads.
inline Rows row_array(const at::Tensor &t, int64_t rows, int64_t heads, int64_t d, at::ScalarType type, int device, const char *what, const char *name) {
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

inline Table table_of(const at::Tensor &t, int device, const char *what) {
    if (t.scalar_type() != at::kInt || t.dim() != 2 || (t.size(1) > 1 && t.stride(1) != 1) || !t.is_cuda() || t.get_device() != device) {
        refuse(what, ": block_table must be int32 [requests, pages of a request] with contiguous rows on cuda:", device, ", got ", described(t));
    }
    return {static_cast<int32_t *>(t.data_ptr()), t.size(0) > 1 ? t.stride(0) : t.size(1), t.size(0), t.size(1)};
}

inline void *stream_of(py::handle stream, int device) {
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

inline at::ScalarType type_of(int32_t dtype) { return dtype == HM_FP16 ? at::kHalf : at::kBFloat16; }

// What a call may use of a workspace tensor, from its first 256-byte boundary on.
struct Workspace {
    void *p;
    size_t bytes;
};

inline Workspace workspace_of(const at::Tensor &t, int device, const char *what) {
    if (!t.is_cuda() || t.get_device() != device || !t.is_contiguous()) {
        refuse(what, ": the workspace must be a contiguous tensor on cuda:", device, ", got ", described(t));
    }
    const uintptr_t base = reinterpret_cast<uintptr_t>(t.data_ptr()), aligned = (base + 255) / 256 * 256;
    return {reinterpret_cast<void *>(aligned), t.nbytes() > aligned - base ? t.nbytes() - (aligned - base) : 0};
}

void def_branches(py::module_ &m); // hm_branch_host.cpp

} // namespace hm_host
