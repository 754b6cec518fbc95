// Parts of the native host path that its sources share: errors, column-major tensors, the context of a call.
#pragma once
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/utils/pybind.h>
#include <torch/csrc/autograd/custom_function.h>
#include <ATen/ATen.h>
#include <ATen/core/grad_mode.h>
#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>
#include <nvtx3/nvToolsExt.h>

#include <cmath>
#include <mutex>
#include <optional>
#include <vector>

#include "../../include/circatt_b200.h"

namespace py = pybind11;
using at::Tensor;
using torch::autograd::AutogradContext;
using torch::autograd::Function;
using torch::autograd::variable_list;

namespace circatt {

typedef c10::SmallVector<int64_t, 6> Shape;

// ---------------------------------------------------------------- errors
inline PyObject* g_error_class = nullptr;          // CircAttError
inline bool g_nvtx = false;

// Raises `cls` with `msg` on any thread (the autograd engine hands a python_error back to the caller).
[[noreturn]] inline void raise(PyObject* cls, const std::string& msg) {
    py::gil_scoped_acquire gil;
    PyErr_SetString(cls, msg.c_str());
    python_error e;
    e.persist();
    throw e;
}

inline void check(int rc) {
    if (rc == CA_OK) return;
    raise(g_error_class, "circatt_b200 status " + std::to_string(rc) + ": " + ca_last_error());
}

inline void require_cuda(const Tensor& t) {
    if (!t.is_cuda())
        raise(PyExc_RuntimeError, "CirculantAttention is only CUDA compatible (no CPU path): got a tensor on " + t.device().str());
}

// ---------------------------------------------------------------- column-major tensors
inline bool is_colmajor(const Tensor& t) {
    int64_t expect = 1;
    const auto sz = t.sizes(), st = t.strides();
    for (size_t i = 0; i < sz.size(); ++i) {
        if (sz[i] != 1 && st[i] != expect) return false;
        expect *= sz[i];
    }
    return true;
}

inline Shape colmajor_strides(c10::IntArrayRef shape) {
    Shape st;
    int64_t acc = 1;
    for (int64_t n : shape) { st.push_back(acc); acc *= n; }
    return st;
}

inline Tensor empty_cm(c10::IntArrayRef shape, const Tensor& like, at::ScalarType dtype) {
    return at::empty_strided(shape, colmajor_strides(shape), like.options().dtype(dtype));
}

inline Tensor colmajor(const Tensor& t) {
    if (is_colmajor(t)) return t;
    Tensor out = empty_cm(t.sizes(), t, t.scalar_type());
    out.copy_(t);
    return out;
}

inline Tensor dense(const Tensor& t) {
    const auto d = t.scalar_type();
    if (d != at::kFloat && d != at::kComplexFloat && d != at::kBFloat16)
        raise(PyExc_TypeError, std::string("only Float32, ComplexF32 and (fused attention) BFloat16 are supported, got ") + c10::toString(d));
    return colmajor(t);
}

inline Tensor view_cm(const Tensor& t, c10::IntArrayRef shape) { return t.as_strided(shape, colmajor_strides(shape), t.storage_offset()); }

inline int64_t prod(c10::IntArrayRef v) {
    int64_t n = 1;
    for (int64_t x : v) n *= x;
    return n;
}

// ---------------------------------------------------------------- call context
// Device of the call, its current stream, and (per host thread) the device word in which kernels flag a wait that
// ran out.
struct StatusWords {
    std::mutex m;
    Tensor word[64];
};
inline StatusWords& status_words() {
    static StatusWords* w = new StatusWords;     // never destroyed: outlives the CUDA context at exit
    return *w;
}
inline thread_local int t_status_device = -1;

inline Tensor status_word(int device) {
    TORCH_CHECK(device >= 0 && device < 64, "device index out of range");
    StatusWords& s = status_words();
    Tensor w;
    {
        std::lock_guard<std::mutex> lock(s.m);
        if (!s.word[device].defined())
            s.word[device] = at::zeros({1}, at::TensorOptions().dtype(at::kInt).device(at::kCUDA, device));
        w = s.word[device];
    }
    if (t_status_device != device) {
        check(ca_status_word(w.data_ptr<int32_t>()));
        t_status_device = device;
    }
    return w;
}

struct Call {
    c10::cuda::CUDAGuard guard;
    void* stream;
    bool range;
    explicit Call(const Tensor& t, const char* name = nullptr)
        : guard(t.device()), stream(c10::cuda::getCurrentCUDAStream(t.device().index()).stream()), range(name && g_nvtx) {
        if (name) status_word(t.device().index());
        if (range) nvtxRangePushA(name);
    }
    ~Call() { if (range) nvtxRangePop(); }
};

inline Tensor scratch(size_t bytes, const Tensor& like) {
    if (!bytes) return Tensor();
    return at::empty({(int64_t)bytes}, like.options().dtype(at::kByte));
}
inline void* ptr(const Tensor& t) { return t.defined() ? t.data_ptr() : nullptr; }
inline float* fptr(const Tensor& t) { return t.defined() ? static_cast<float*>(t.data_ptr()) : nullptr; }

inline bool tracked(std::initializer_list<const Tensor*> ts) {
    if (!at::GradMode::is_enabled()) return false;
    for (const Tensor* t : ts)
        if (t->defined() && t->requires_grad()) return true;
    return false;
}

}  // namespace circatt
