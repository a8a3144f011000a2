// What the CPython modules over libf8mi's C ABI share on the way from torch tensors to its entry points.  Host code only, and one translation unit a module:
// everything here is that module's own.
#pragma once
#include <dlfcn.h>

#include <algorithm>
#include <optional>
#include <utility>

#include <ATen/ATen.h>
#include <ATen/PythonTorchFunctionTLS.h>
#include <ATen/TracerMode.h>
#include <c10/core/DeviceGuard.h>
#include <c10/core/impl/LocalDispatchKeySet.h>
#include <c10/core/impl/TorchDispatchModeTLS.h>
#include <c10/hip/HIPFunctions.h>
#include <c10/hip/HIPStream.h>
#include <torch/csrc/Dtype.h>
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/PyInterpreter.h>
#include <torch/csrc/autograd/custom_function.h>
#include <torch/csrc/autograd/python_variable.h>
#include <torch/csrc/autograd/variable.h>
#include <torch/csrc/utils/object_ptr.h>

#include "../../include/f8mi.h"

namespace {

using torch::autograd::AutogradContext;
using torch::autograd::variable_list;

decltype(&f8mi_last_error) last_error = nullptr;  // null until the module has been loaded
PyObject* native_error = nullptr;  // float8_experimental_amd._native.Float8NativeError

struct NativeFailure : std::runtime_error {
    using std::runtime_error::runtime_error;
};
void check(int rc, const char* what) {
    if (rc != 0) throw NativeFailure(std::string(what) + " failed with code " + std::to_string(rc) + ": " + last_error());
}

int dtype_code(at::ScalarType t) {
    return t == at::kBFloat16 ? F8MI_BF16 : t == at::kHalf ? F8MI_FP16 : t == at::kFloat ? F8MI_FP32 : -1;
}
void* stream_of(const at::Tensor& t) { return c10::hip::getCurrentHIPStream(t.get_device()).stream(); }
void* ptr(const at::Tensor& t) { return t.defined() ? t.data_ptr() : nullptr; }

// Whether somebody has to see operators: a dispatch or function mode, a trace (what a functional transform follows shows in the tensors).  A kernel's launch is none, and
// a trace would hold the allocation of its output alone.  torch.set_default_device is a function mode that asks for nothing.
PyObject* device_context = nullptr;  // torch.utils._device.DeviceContext
bool watched() {
    if (c10::impl::TorchDispatchModeTLS::any_modes_set() || at::tracer::impl::is_dispatch_enabled()) return true;
    if (at::impl::torch_function_mode_enabled())
        for (int64_t i = 0; i < at::impl::PythonTorchFunctionTLS::stack_len(); i++)
            if ((PyObject*)Py_TYPE(at::impl::PythonTorchFunctionTLS::get_stack_at(i)->ptr(getPyInterpreter())) != device_context) return true;
    return false;
}

// Undefined: not taken.  A plain tensor (or Parameter) of a type that the kernels read, on `device`, whose memory holds its values, without a forward-mode
// derivative (which would be dropped)
at::Tensor plain(PyObject* o, int device) {
    if (!THPVariable_CheckExact(o)) return {};
    const at::Tensor& t = THPVariable_Unpack(o);
    using K = c10::DispatchKey;
    constexpr c10::DispatchKeySet others({K::Python, K::FuncTorchBatched, K::FuncTorchGradWrapper, K::Batched, K::Functionalize, K::Negative, K::ZeroTensor});
    return t.defined() && t.is_cuda() && t.layout() == at::kStrided && !t.key_set().has_any(others) && t.get_device() == device && dtype_code(t.scalar_type()) >= 0 && !t._fw_grad(0).defined() ? t : at::Tensor();
}

// What hooks on saved tensors hand back (they hand back what they like) is what was saved, or the kernels would read other memory
bool as_saved(const at::Tensor& t, const c10::Device& device, at::ScalarType type, at::IntArrayRef sizes) {
    using K = c10::DispatchKey;
    constexpr c10::DispatchKeySet others({K::Python, K::FuncTorchBatched, K::FuncTorchGradWrapper, K::Batched, K::Functionalize, K::ZeroTensor});
    return t.defined() && t.device() == device && t.layout() == at::kStrided && t.scalar_type() == type && t.sizes() == sizes && !t.key_set().has_any(others);
}

// Below autograd, and below functional transforms: what is plain is a constant to them (what they follow is not taken), but what is allocated inside one
// would be a tensor of it, without memory.
struct Below {
    const at::AutoDispatchBelowADInplaceOrView autograd;
    const c10::impl::ExcludeDispatchKeyGuard transforms{c10::DispatchKeySet({c10::DispatchKey::FuncTorchDynamicLayerFrontMode, c10::DispatchKey::FuncTorchDynamicLayerBackMode})};
};

// A matrix as the kernels read it: unit column stride, `ld` from row to row (0: the same row throughout); copied where its layout needs it.
struct Rows {
    at::Tensor t;
    int64_t rows, cols, ld;
    Rows(const at::Tensor& x, int64_t cols_) : cols(cols_) {
        rows = cols ? x.numel() / cols : 0;
        t = x.is_neg() ? x.resolve_neg() : x;
        if (t.dim() == 2 && t.size(1) == cols && (t.stride(1) == 1 || cols == 1) && (t.stride(0) >= cols || rows == 1)) {
            ld = rows == 1 ? cols : t.stride(0);
            return;
        }
        if (t.dim() >= 2 && t.size(-1) == cols && t.stride(-1) == 1 && rows > 1) {
            bool one = true;  // expanded over all leading dimensions: what autograd hands to backward after a sum
            for (int64_t d = 0; d + 1 < t.dim(); d++) one &= t.stride(d) == 0 || t.size(d) == 1;
            if (one) {
                ld = 0;
                return;
            }
        }
        t = t.contiguous();
        ld = cols;
    }
    int dtype() const { return dtype_code(t.scalar_type()); }
};

struct Blocks {  // where a copy and its scales lie
    uint8_t *data = nullptr, *scales = nullptr;
};
// Parts of one allocation: a layer allocates what it keeps for backward and what it does not with one call each, not eight.
struct Parts {
    int64_t bytes = 0;
    int64_t take(int64_t n) {
        const int64_t at = bytes;
        bytes += (n + 255) / 256 * 256;
        return at;
    }
};
struct BlocksAt {  // offsets in such an allocation; -1: not there
    int64_t data = -1, scales = -1;
    BlocksAt() = default;
    BlocksAt(Parts& p, int64_t rows, int64_t k, bool with_data = true, bool with_scales = true) {
        const int64_t kp = (k + 127) / 128 * 128;
        if (with_data) data = p.take(kp * rows);
        if (with_scales) scales = p.take(kp / 128 * ((rows + 127) / 128 * 128));
    }
    Blocks in(const at::Tensor& t) const {
        uint8_t* base = (uint8_t*)t.data_ptr();
        return {data < 0 ? nullptr : base + data, scales < 0 ? nullptr : base + scales};
    }
};
at::Tensor bytes_on(const at::Tensor& like, const Parts& p) { return at::empty({p.bytes}, like.options().dtype(at::kByte).memory_format(at::MemoryFormat::Contiguous)); }

// [m, n] = a [m, k] times b [n, k]; transposed: b's data is the other copy of its tensor
template <typename Lib>
at::Tensor block_gemm(const Lib& L, const at::Tensor& like, const Blocks& a, const Blocks& b, bool transposed, int64_t m, int64_t n, int64_t k, at::ScalarType type, const at::Tensor& bias = {}) {
    const int64_t kp = (k + 127) / 128 * 128;
    at::Tensor c = at::empty({m, n}, like.options().dtype(type).memory_format(at::MemoryFormat::Contiguous));
    const int64_t bytes = L.block_gemm_workspace_bytes(m, n, kp);
    const at::Tensor ws = bytes ? at::empty({bytes / 4}, like.options().dtype(at::kFloat)) : at::Tensor();
    check(L.block_gemm(a.data, a.scales, b.data, b.scales, transposed, m, n, kp, c.data_ptr(), dtype_code(type), n, ptr(bias), ptr(ws), bytes, stream_of(c)), "f8mi_block_gemm");
    return c;
}

// An argument that may be absent: autograd gives it an edge only where it is there.
using MaybeTensor = std::optional<at::Tensor>;
MaybeTensor maybe(const at::Tensor& t) { return t.defined() ? MaybeTensor(t) : MaybeTensor(); }

// ---- Python

PyObject* wrap(const at::Tensor& t) {
    if (!t.defined()) Py_RETURN_NONE;
    return THPVariable_Wrap(t);
}
struct WithoutGil {
    PyThreadState* state = PyEval_SaveThread();
    ~WithoutGil() { PyEval_RestoreThread(state); }
};
template <typename F>
PyObject* guarded(F body) {
    HANDLE_TH_ERRORS
    try {
        return body();
    } catch (const NativeFailure& f) {
        PyErr_SetString(native_error, f.what());
        return nullptr;
    }
    END_HANDLE_TH_ERRORS
}
bool expect(Py_ssize_t got, Py_ssize_t want, const char* name) {
    if (!last_error) PyErr_SetString(PyExc_RuntimeError, "load() has not been called");
    else if (got != want) PyErr_Format(PyExc_TypeError, "%s takes %zd arguments, got %zd", name, want, got);
    else return true;
    return false;
}
// false: not taken; None leaves t undefined
bool optional(PyObject* o, int device, at::Tensor& t) {
    if (o == Py_None) return true;
    t = plain(o, device);
    return t.defined();
}
bool wants_grad(const at::Tensor& t) { return t.defined() && t.requires_grad() && at::GradMode::is_enabled(); }

// The device whose tensors a call takes: the current one as torch has it for this thread, without a call into Python.  -1, which no tensor is on, where
// nothing is taken.
int device_taken() {
    static const bool any = c10::hip::device_count() > 0;
    return any && !watched() ? (int)c10::hip::current_device() : -1;
}

// The entry points of libf8mi: get(pointer, name) for each, between open() and done().
struct Loader {
    void* handle = nullptr;
    const char *path = nullptr, *missing = nullptr;
    PyObject* error = nullptr;
    bool open(PyObject* args) {  // (path of libf8mi.so, error class)
        if (!PyArg_ParseTuple(args, "sO", &path, &error)) return false;
        handle = dlopen(path, RTLD_NOW | RTLD_LOCAL);
        if (!handle) PyErr_Format(PyExc_ImportError, "%s", dlerror());
        return handle != nullptr;
    }
    template <typename F>
    void get(F& f, const char* name) {
        f = reinterpret_cast<F>(dlsym(handle, name));
        if (!f) missing = name;
    }
    PyObject* done() {
        get(last_error, "f8mi_last_error");
        if (missing) {
            last_error = nullptr;
            return PyErr_Format(PyExc_ImportError, "%s does not export %s", path, missing);
        }
        THPObjectPtr module(PyImport_ImportModule("torch.utils._device"));
        device_context = module ? PyObject_GetAttrString(module.get(), "DeviceContext") : nullptr;
        if (!device_context) {
            last_error = nullptr;
            return nullptr;
        }
        Py_INCREF(error);
        native_error = error;
        Py_RETURN_NONE;
    }
};

template <typename F>
PyCFunction fast(F f) { return (PyCFunction)(void (*)(void))f; }

}  // namespace
