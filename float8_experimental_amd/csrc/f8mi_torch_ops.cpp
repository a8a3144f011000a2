// The host path of the blockwise scaled linear, layer norm and gradient clipping over libf8mi's C ABI, as a CPython module on torch
// tensors: one call allocates what the kernels write and queues all launches, and the backward passes are nodes that run without the
// interpreter.  Host code only.
//
// Every function returns None, without having queued or allocated anything, for tensors that it does not take (subclasses, other devices or
// types) and while somebody has to see operators (modes, traces): the caller then goes through the registered operators, or raises.  Workspaces are temporaries of torch's caching allocator, which
// hands their memory out again in stream order: calls on any number of threads, streams and captures share nothing.
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

struct Lib {
    decltype(&f8mi_block_scale_bytes) block_scale_bytes;
    decltype(&f8mi_block_cast) block_cast;
    decltype(&f8mi_block_gemm) block_gemm;
    decltype(&f8mi_block_gemm_workspace_bytes) block_gemm_workspace_bytes;
    decltype(&f8mi_block_linear_few_rows) block_linear_few_rows;
    decltype(&f8mi_column_sum_finish) column_sum_finish;
    decltype(&f8mi_layer_norm) layer_norm;
    decltype(&f8mi_layer_norm_backward) layer_norm_backward;
    decltype(&f8mi_layer_norm_workspace_bytes) layer_norm_workspace_bytes;
    decltype(&f8mi_grad_clip) grad_clip;
    decltype(&f8mi_grad_clip_workspace_bytes) grad_clip_workspace_bytes;
    decltype(&f8mi_last_error) last_error;
} L;
PyObject* native_error = nullptr;  // float8_experimental_amd._native.Float8NativeError

struct NativeFailure : std::runtime_error {
    using std::runtime_error::runtime_error;
};
void check(int rc, const char* what) {
    if (rc != 0) throw NativeFailure(std::string(what) + " failed with code " + std::to_string(rc) + ": " + L.last_error());
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

// ---- blockwise scaled linear

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

f8mi_block_cast_job job_of(const Rows& x, bool square, const Blocks& a, const Blocks& t, float* sums = nullptr) {
    return {x.t.data_ptr(), x.rows, x.cols, x.ld, x.dtype(), square, a.data, a.data ? a.scales : nullptr, t.data, t.scales, sums};
}
// [m, n] = a [m, k] times b [n, k]; transposed: b's data is the other copy of its tensor
at::Tensor block_gemm(const at::Tensor& like, const Blocks& a, const Blocks& b, bool transposed, int64_t m, int64_t n, int64_t k, at::ScalarType type, const at::Tensor& bias = {}) {
    const int64_t kp = (k + 127) / 128 * 128;
    at::Tensor c = at::empty({m, n}, like.options().dtype(type).memory_format(at::MemoryFormat::Contiguous));
    const int64_t bytes = L.block_gemm_workspace_bytes(m, n, kp);
    const at::Tensor ws = bytes ? at::empty({bytes / 4}, like.options().dtype(at::kFloat)) : at::Tensor();
    check(L.block_gemm(a.data, a.scales, b.data, b.scales, transposed, m, n, kp, c.data_ptr(), dtype_code(type), n, ptr(bias), ptr(ws), bytes, stream_of(c)), "f8mi_block_gemm");
    return c;
}

// The weight needs one copy if the backward product can read it transposed
bool one_weight_copy(int64_t k, int64_t n) { return k % 128 == 0 && n % 128 == 0; }

// What a layer keeps for backward, in one allocation: x transposed and its scales for the gradient of the weight; the weight, transposed or as it is,
// and the scales of its transpose for the gradient of x.
struct Kept {
    Parts parts;
    BlocksAt xt, w, wt;
    Kept(int64_t m, int64_t k, int64_t n, bool need_dx, bool need_dw) {
        if (need_dw) xt = BlocksAt(parts, k, m);
        if (need_dx) {
            const bool one = one_weight_copy(k, n);
            if (one) w = BlocksAt(parts, n, k, true, false);
            wt = BlocksAt(parts, k, n, !one);
        }
    }
};

// An argument that may be absent: autograd gives it an edge only where it is there.
using MaybeTensor = std::optional<at::Tensor>;
MaybeTensor maybe(const at::Tensor& t) { return t.defined() ? MaybeTensor(t) : MaybeTensor(); }

struct BlockwiseLinear : torch::autograd::Function<BlockwiseLinear> {
    // kept: see Kept; null: nothing is
    static at::Tensor compute(const at::Tensor& x, const at::Tensor& weight, const at::Tensor& bias, bool need_dx, bool need_dw, at::Tensor* kept) {
        const c10::DeviceGuard guard(x.device());
        const Below below;
        const int64_t k = weight.size(1), n = weight.size(0);
        const Rows xr(x, k), wr(weight, k);
        const int64_t m = xr.rows;
        std::vector<int64_t> y_shape(x.sizes().begin(), x.sizes().end());
        y_shape.back() = n;
        if (m == 0) return at::empty(y_shape, x.options());
        const Kept k_at(m, k, n, need_dx, need_dw);
        Parts parts;
        const BlocksAt x8_at(parts, m, k), w8_at(parts, n, k, k_at.w.data < 0);
        const at::Tensor mem = bytes_on(x, parts);
        Blocks xt, wt, w8 = w8_at.in(mem);
        const Blocks x8 = x8_at.in(mem);
        if (k_at.parts.bytes) {
            *kept = bytes_on(x, k_at.parts);
            xt = k_at.xt.in(*kept);
            wt = k_at.wt.in(*kept);
            if (k_at.w.data >= 0) w8.data = k_at.w.in(*kept).data;
        }
        const f8mi_block_cast_job jobs[2] = {job_of(xr, false, x8, xt), job_of(wr, true, w8, wt)};
        check(L.block_cast(jobs, 2, stream_of(x)), "f8mi_block_cast");
        const at::Tensor b = bias.defined() ? bias.to(x.scalar_type()).contiguous() : at::Tensor();
        at::Tensor y = block_gemm(x, x8, w8, false, m, n, k, x.scalar_type(), b);
        return x.dim() == 2 ? y : at::_unsafe_view(y, y_shape);
    }
    static at::Tensor forward(AutogradContext* ctx, const at::Tensor& x, const at::Tensor& weight, const MaybeTensor& bias_, bool need_dx, bool need_dw) {
        const at::Tensor bias = bias_.value_or(at::Tensor());
        at::Tensor kept;
        at::Tensor y = compute(x, weight, bias, need_dx, need_dw, &kept);
        ctx->saved_data["x_shape"] = x.sizes().vec();
        ctx->saved_data["types"] = (int64_t)x.scalar_type() | (int64_t)weight.scalar_type() << 8 | (bias.defined() ? (int64_t)bias.scalar_type() + 1 : 0) << 16 | (int64_t)need_dx << 24 | (int64_t)need_dw << 25;
        ctx->saved_data["n"] = weight.size(0);
        ctx->save_for_backward({kept});
        return y;
    }
    static variable_list backward(AutogradContext* ctx, const variable_list& grads) {
        TORCH_CHECK(!at::GradMode::is_enabled(), "blockwise_linear has no second derivative (create_graph=True)");
        const auto saved = ctx->get_saved_variables();
        const auto x_shape = ctx->saved_data["x_shape"].toIntVector();
        const int64_t k = x_shape.back(), n = ctx->saved_data["n"].toInt(), types = ctx->saved_data["types"].toInt();
        const at::ScalarType xt = (at::ScalarType)(types & 255), wt = (at::ScalarType)(types >> 8 & 255), bt = (at::ScalarType)((types >> 16 & 255) - 1);
        const bool kept_dx = types >> 24 & 1, kept_dw = types >> 25 & 1;
        const bool need_dx = ctx->needs_input_grad(0), need_dw = ctx->needs_input_grad(1);
        const bool need_db = (types >> 16 & 255) && ctx->needs_input_grad(2);
        at::Tensor dx, dw, db;
        if (!grads[0].defined()) return {dx, dw, db, at::Tensor(), at::Tensor()};
        const c10::DeviceGuard guard(grads[0].device());
        const Below below;
        const Rows dy(grads[0].scalar_type() == xt ? grads[0] : grads[0].to(xt), n);
        const int64_t m = dy.rows;
        if (m == 0) {
            if (need_dx) dx = at::empty(x_shape, dy.t.options());
            if (need_dw) dw = at::zeros({n, k}, dy.t.options().dtype(wt));
            if (need_db) db = at::zeros({n}, dy.t.options().dtype(bt));
            return {dx, dw, db, at::Tensor(), at::Tensor()};
        }
        if (!(need_dx || need_dw || need_db)) return {dx, dw, db, at::Tensor(), at::Tensor()};
        TORCH_CHECK((!need_dx || kept_dx) && (!need_dw || kept_dw), "blockwise_linear: a gradient is asked for that the forward pass was not told of");
        const Kept k_at(m, k, n, kept_dx, kept_dw);
        const at::Tensor& kept = saved[0];
        if (need_dx || need_dw)
            TORCH_CHECK(as_saved(kept, grads[0].device(), at::kByte, {k_at.parts.bytes}) && kept.is_contiguous(), "blockwise_linear: what was saved for backward is not what came back");
        Parts parts;
        const BlocksAt g8_at = need_dx ? BlocksAt(parts, m, n) : BlocksAt(), gt_at = need_dw ? BlocksAt(parts, n, m) : BlocksAt();
        const int64_t sum_rows = (m + 127) / 128, sums_at = need_db ? parts.take(sum_rows * n * 4) : 0;
        const at::Tensor mem = bytes_on(dy.t, parts);
        const Blocks g8 = g8_at.in(mem), gt = gt_at.in(mem);
        float* sums = need_db ? (float*)((uint8_t*)mem.data_ptr() + sums_at) : nullptr;
        const f8mi_block_cast_job job = job_of(dy, false, g8, gt, sums);
        check(L.block_cast(&job, 1, stream_of(dy.t)), "f8mi_block_cast");
        if (need_dx) {
            const bool one = one_weight_copy(k, n);
            const Blocks w{one ? k_at.w.in(kept).data : k_at.wt.in(kept).data, k_at.wt.in(kept).scales};
            dx = block_gemm(dy.t, g8, w, one, m, k, n, xt);
            if (x_shape.size() != 2) dx = dx.view(x_shape);
        }
        if (need_dw) dw = block_gemm(dy.t, gt, k_at.xt.in(kept), false, n, k, m, wt);
        if (need_db) {
            db = at::empty({n}, dy.t.options().dtype(bt));
            check(L.column_sum_finish(sums, sum_rows, n, F8MI_FP32, db.data_ptr(), dtype_code(bt), stream_of(dy.t)), "f8mi_column_sum_finish");
        }
        return {dx, dw, db, at::Tensor(), at::Tensor()};
    }
};

// ---- layer norm

struct LayerNorm : torch::autograd::Function<LayerNorm> {
    static at::Tensor compute(const at::Tensor& x, const at::Tensor& weight, const at::Tensor& bias, int64_t cols, double eps, at::Tensor* stats_out) {
        const c10::DeviceGuard guard(x.device());
        const Below below;
        const Rows r(x, cols);
        const int pt = weight.defined() ? dtype_code(weight.scalar_type()) : bias.defined() ? dtype_code(bias.scalar_type()) : r.dtype();
        const at::Tensor w = weight.defined() ? weight.contiguous() : weight, b = bias.defined() ? bias.contiguous() : bias;
        const at::Tensor y = at::empty(x.sizes(), x.options()), stats = stats_out ? at::empty({r.rows, 2}, x.options().dtype(at::kFloat)) : at::Tensor();
        if (r.rows) check(L.layer_norm(r.t.data_ptr(), r.rows, cols, r.ld, r.dtype(), ptr(w), ptr(b), pt, (float)eps, y.data_ptr(), (float*)ptr(stats), stream_of(x)), "f8mi_layer_norm");
        if (stats_out) *stats_out = stats;
        return y;
    }
    static at::Tensor forward(AutogradContext* ctx, const at::Tensor& x, const MaybeTensor& weight_, const MaybeTensor& bias_, int64_t cols, double eps) {
        const at::Tensor weight = weight_.value_or(at::Tensor()), bias = bias_.value_or(at::Tensor());
        at::Tensor stats;
        at::Tensor y = compute(x, weight, bias, cols, eps, &stats);
        ctx->save_for_backward({x, weight, stats});
        ctx->saved_data["x_shape"] = x.sizes().vec();
        ctx->saved_data["x_type"] = (int64_t)x.scalar_type();
        ctx->saved_data["cols"] = cols;
        ctx->saved_data["has_weight"] = weight.defined();
        ctx->saved_data["has_bias"] = bias.defined();
        ctx->saved_data["w_shape"] = weight.defined() ? weight.sizes().vec() : std::vector<int64_t>();
        ctx->saved_data["b_shape"] = bias.defined() ? bias.sizes().vec() : std::vector<int64_t>();
        ctx->saved_data["p_type"] = (int64_t)(weight.defined() ? weight.scalar_type() : bias.defined() ? bias.scalar_type() : x.scalar_type());
        return y;
    }
    static variable_list backward(AutogradContext* ctx, const variable_list& grads) {
        TORCH_CHECK(!at::GradMode::is_enabled(), "layer_norm has no second derivative (create_graph=True)");
        const bool has_weight = ctx->saved_data["has_weight"].toBool(), has_bias = ctx->saved_data["has_bias"].toBool();
        const bool need_dx = ctx->needs_input_grad(0), need_dw = has_weight && ctx->needs_input_grad(1), need_db = has_bias && ctx->needs_input_grad(has_weight ? 2 : 1);
        at::Tensor dx, dw, db;
        if (!grads[0].defined() || !(need_dx || need_dw || need_db)) return {dx, dw, db, at::Tensor(), at::Tensor()};
        const auto saved = ctx->get_saved_variables();
        const at::Tensor &x = saved[0], &stats = saved[2];
        const c10::DeviceGuard guard(grads[0].device());
        const Below below;
        const int64_t cols = ctx->saved_data["cols"].toInt();
        const at::ScalarType pt = (at::ScalarType)ctx->saved_data["p_type"].toInt();
        TORCH_CHECK(as_saved(x, grads[0].device(), (at::ScalarType)ctx->saved_data["x_type"].toInt(), ctx->saved_data["x_shape"].toIntVector()) &&
                        as_saved(stats, grads[0].device(), at::kFloat, {x.numel() / cols, 2}) && stats.is_contiguous() && !stats.is_neg() && saved[1].defined() == has_weight &&
                        (!has_weight || as_saved(saved[1], grads[0].device(), pt, ctx->saved_data["w_shape"].toIntVector())),
                    "layer_norm: what was saved for backward is not what came back");
        const Rows r(x, cols), dy(grads[0].scalar_type() == x.scalar_type() ? grads[0] : grads[0].to(x.scalar_type()), cols);
        const at::Tensor w = has_weight ? saved[1].resolve_neg().contiguous() : saved[1];
        if (need_dx) dx = at::empty(x.sizes(), x.options().memory_format(at::MemoryFormat::Contiguous));
        if (need_dw) dw = at::empty(ctx->saved_data["w_shape"].toIntVector(), x.options().dtype(pt));
        if (need_db) db = at::empty(ctx->saved_data["b_shape"].toIntVector(), x.options().dtype(pt));
        const int64_t bytes = need_dw || need_db ? L.layer_norm_workspace_bytes(r.rows, cols, r.dtype()) : 0;
        const at::Tensor ws = bytes ? at::empty({bytes / 4}, x.options().dtype(at::kFloat)) : at::Tensor();
        check(L.layer_norm_backward(ptr(dy.t), dy.ld, ptr(r.t), r.ld, r.rows, cols, r.dtype(), ptr(w), dtype_code(pt), (const float*)ptr(stats), ptr(dx), ptr(dw), ptr(db), ptr(ws),
                                    bytes, stream_of(x)), "f8mi_layer_norm_backward");
        return {dx, dw, db, at::Tensor(), at::Tensor()};
    }
};

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
    if (!L.last_error) PyErr_SetString(PyExc_RuntimeError, "f8mi_torch_ops: load() has not been called");
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

// blockwise_linear(x [..., k], weight [n, k], bias or None) -> y, with its history, or None (also for shapes that do not fit: the caller says what is
// wrong with them).
PyObject* blockwise_linear(PyObject*, PyObject* const* a, Py_ssize_t n_args) {
    if (!expect(n_args, 3, "blockwise_linear")) return nullptr;
    return guarded([&]() -> PyObject* {
        const int device = device_taken();
        const at::Tensor x = plain(a[0], device), w = plain(a[1], device);
        at::Tensor bias;
        if (!x.defined() || !w.defined() || !optional(a[2], device, bias)) Py_RETURN_NONE;
        if (w.dim() != 2 || w.size(0) == 0 || w.size(1) == 0 || x.dim() == 0 || x.size(-1) != w.size(1) || (bias.defined() && (bias.dim() != 1 || bias.size(0) != w.size(0)))) Py_RETURN_NONE;
        at::Tensor y;
        {
            const WithoutGil no_gil;
            const bool gx = wants_grad(x), gw = wants_grad(w);
            if (gx || gw || wants_grad(bias)) y = BlockwiseLinear::apply(x, w, maybe(bias), gx, gw);
            else y = BlockwiseLinear::compute(x, w, bias, false, false, nullptr);
        }
        return wrap(y);
    });
}

// Cast and product of a few rows in one kernel: every workgroup converts all of the activations for itself, which costs more than the launch it saves
// once there are many of them and many rows.  The lines are those measured for the linears with one scale; for block scales they were not measured.
bool one_kernel_pays(int64_t m, int64_t n, int64_t kp, int dt) {
    if (m > 16 || m * kp > F8MI_FEW_ROWS_ELEMS) return false;
    return dt == F8MI_FP32 ? n <= 16384 || m * n <= 65536 : m * n <= 262144;
}

// blockwise_inference_linear(x [..., k], data, scales of the weight, n, k, bias or None) -> y or None
PyObject* blockwise_inference_linear(PyObject*, PyObject* const* a, Py_ssize_t n_args) {
    if (!expect(n_args, 6, "blockwise_inference_linear")) return nullptr;
    return guarded([&]() -> PyObject* {
        const int device = device_taken();
        const int64_t n = PyLong_AsLongLong(a[3]), k = PyLong_AsLongLong(a[4]);
        const at::Tensor x = plain(a[0], device);
        at::Tensor bias;
        if (!x.defined() || x.dim() < 1 || x.size(-1) != k || k <= 0 || wants_grad(x) || !THPVariable_Check(a[1]) || !THPVariable_Check(a[2]) || !optional(a[5], device, bias)) Py_RETURN_NONE;
        if (bias.defined() && (bias.dim() != 1 || bias.size(0) != n)) Py_RETURN_NONE;
        const at::Tensor data = THPVariable_Unpack(a[1]), scales = THPVariable_Unpack(a[2]);
        const int64_t kp = (k + 127) / 128 * 128;
        if (!data.is_cuda() || data.get_device() != device || data.scalar_type() != at::kFloat8_e4m3fn || !data.is_contiguous() || data.numel() != kp * n || !scales.is_cuda() ||
            scales.get_device() != device || scales.scalar_type() != at::kByte || !scales.is_contiguous() || scales.numel() != L.block_scale_bytes(n, k))
            Py_RETURN_NONE;
        at::Tensor y;
        {
            const WithoutGil no_gil;
            const c10::DeviceGuard guard(x.device());
            const Below below;
            std::vector<int64_t> y_shape(x.sizes().begin(), x.sizes().end());
            y_shape.back() = n;
            const Rows xr(x, k);
            const at::Tensor b = bias.defined() ? bias.to(x.scalar_type()).contiguous() : at::Tensor();
            if (xr.rows == 0) {
                y = at::empty(y_shape, x.options());
            } else if (one_kernel_pays(xr.rows, n, kp, xr.dtype())) {
                y = at::empty(y_shape, x.options());
                check(L.block_linear_few_rows(xr.t.data_ptr(), xr.ld, xr.dtype(), data.data_ptr(), scales.data_ptr(), xr.rows, n, k, y.data_ptr(), n, ptr(b), stream_of(x)),
                      "f8mi_block_linear_few_rows");
            } else {
                Parts parts;
                const BlocksAt x8_at(parts, xr.rows, k);
                const at::Tensor mem = bytes_on(x, parts);
                const Blocks x8 = x8_at.in(mem);
                const f8mi_block_cast_job job = job_of(xr, false, x8, Blocks());
                check(L.block_cast(&job, 1, stream_of(x)), "f8mi_block_cast");
                y = block_gemm(x, x8, {(uint8_t*)data.data_ptr(), (uint8_t*)scales.data_ptr()}, false, xr.rows, n, k, x.scalar_type(), b);
                if (x.dim() != 2) y = y.view(y_shape);
            }
        }
        return wrap(y);
    });
}

// layer_norm(x, normalized_shape (an int or a tuple), weight or None, bias or None, eps) -> y, with its history, or None (also for shapes and types that
// do not fit: the caller says what is wrong with them, or converts them).
PyObject* layer_norm(PyObject*, PyObject* const* a, Py_ssize_t n_args) {
    if (!expect(n_args, 5, "layer_norm")) return nullptr;
    return guarded([&]() -> PyObject* {
        const int device = device_taken();
        const at::Tensor x = plain(a[0], device);
        at::Tensor w, b;
        if (!x.defined() || !optional(a[2], device, w) || !optional(a[3], device, b)) Py_RETURN_NONE;
        std::vector<int64_t> shape;
        if (PyLong_Check(a[1])) shape.push_back(PyLong_AsLongLong(a[1]));
        else if (PyTuple_Check(a[1]))  // (torch.Size is one)
            for (Py_ssize_t i = 0; i < PyTuple_GET_SIZE(a[1]); i++) {
                if (!PyLong_Check(PyTuple_GET_ITEM(a[1], i))) Py_RETURN_NONE;
                shape.push_back(PyLong_AsLongLong(PyTuple_GET_ITEM(a[1], i)));
            }
        if (PyErr_Occurred()) {  // a number that no dimension has
            PyErr_Clear();
            Py_RETURN_NONE;
        }
        const int64_t d = (int64_t)shape.size();
        if (d == 0 || x.dim() < d || x.sizes().slice(x.dim() - d) != at::IntArrayRef(shape)) Py_RETURN_NONE;
        int64_t cols = 1;
        for (const int64_t s : shape) cols *= s;
        if (cols <= 0) Py_RETURN_NONE;
        for (const at::Tensor* p : {&w, &b})
            if (p->defined() && (p->sizes() != at::IntArrayRef(shape) || (p->scalar_type() != x.scalar_type() && p->scalar_type() != at::kFloat))) Py_RETURN_NONE;
        if (w.defined() && b.defined() && w.scalar_type() != b.scalar_type()) Py_RETURN_NONE;
        const double eps = PyFloat_AsDouble(a[4]);
        if (eps == -1.0 && PyErr_Occurred()) return nullptr;
        at::Tensor y;
        {
            const WithoutGil no_gil;
            if (wants_grad(x) || wants_grad(w) || wants_grad(b)) y = LayerNorm::apply(x, maybe(w), maybe(b), cols, eps);
            else y = LayerNorm::compute(x, w, b, cols, eps, nullptr);
        }
        return wrap(y);
    });
}

// Whether two of them share memory: one read while the other is written, in place, would be scaled or not as it happens.
bool overlapping(const std::vector<at::Tensor>& ts) {
    std::vector<std::pair<uintptr_t, uintptr_t>> at;
    at.reserve(ts.size());
    for (const at::Tensor& t : ts)
        if (t.numel()) at.emplace_back((uintptr_t)t.data_ptr(), (uintptr_t)t.data_ptr() + t.nbytes());
    std::sort(at.begin(), at.end());
    for (size_t i = 1; i < at.size(); i++)
        if (at[i].first < at[i - 1].second) return true;
    return false;
}

// grad_clip(list, what, kind, max_norm) -> (norm (fp32, 0-dim), list or None), or None: something in the list is not taken.
// what: "norm" of the tensors; "grads": the gradients of the tensors are clipped in place; None: clipped into new tensors of the tensors' own
// types; a dtype: of that type.
PyObject* grad_clip(PyObject*, PyObject* const* a, Py_ssize_t n_args) {
    if (!expect(n_args, 4, "grad_clip")) return nullptr;
    return guarded([&]() -> PyObject* {
        const int kind = (int)PyLong_AsLong(a[2]), device = device_taken();
        const double max_norm = PyFloat_AsDouble(a[3]);
        const bool of_params = PyUnicode_Check(a[1]) && PyUnicode_CompareWithASCIIString(a[1], "grads") == 0;
        const bool to_new = !PyUnicode_Check(a[1]);
        const bool typed = THPDtype_Check(a[1]);
        if (!PyList_Check(a[0]) || device < 0) Py_RETURN_NONE;
        std::vector<at::Tensor> xs, outs;
        xs.reserve((size_t)PyList_GET_SIZE(a[0]));
        for (Py_ssize_t i = 0; i < PyList_GET_SIZE(a[0]); i++) {
            PyObject* o = PyList_GET_ITEM(a[0], i);
            at::Tensor g;
            if (of_params) {
                if (!THPVariable_Check(o)) Py_RETURN_NONE;
                const at::Tensor grad = THPVariable_Unpack(o).grad();
                if (!grad.defined()) continue;
                THPObjectPtr wrapped(THPVariable_Wrap(grad));  // a subclass shows in its Python type only
                g = plain(wrapped.get(), device);
            } else {
                g = plain(o, device);
            }
            if (!g.defined() || !g.is_non_overlapping_and_dense()) Py_RETURN_NONE;
            xs.push_back(g);
        }
        if (of_params && overlapping(xs)) Py_RETURN_NONE;
        at::Tensor norm;
        {
            const WithoutGil no_gil;
            const Below below;
            const c10::DeviceGuard guard(c10::Device(c10::kCUDA, (c10::DeviceIndex)device));
            const auto options = at::TensorOptions().device(c10::Device(c10::kCUDA, (c10::DeviceIndex)device));
            std::vector<f8mi_grad> grads(xs.size());
            for (size_t i = 0; i < xs.size(); i++) {
                if (to_new) outs.push_back(at::empty_strided(xs[i].sizes(), xs[i].strides(), typed ? xs[i].options().dtype(((THPDtype*)a[1])->scalar_type) : xs[i].options()));
                const at::Tensor& out = to_new ? outs[i] : xs[i];
                grads[i] = {xs[i].data_ptr(), out.data_ptr(), xs[i].numel(), dtype_code(xs[i].scalar_type()), dtype_code(out.scalar_type())};
                if (of_params) torch::autograd::impl::bump_version(xs[i]);
            }
            norm = at::empty({}, options.dtype(at::kFloat));
            const int64_t count = (int64_t)xs.size(), bytes = L.grad_clip_workspace_bytes(count);
            const at::Tensor ws = at::empty({bytes / 8}, options.dtype(at::kDouble));
            check(L.grad_clip(grads.data(), count, kind, (float)max_norm, to_new || of_params, (float*)norm.data_ptr(), ws.data_ptr(), bytes, stream_of(norm)), "f8mi_grad_clip");
        }
        THPObjectPtr list(Py_None);
        Py_INCREF(Py_None);
        if (to_new) {
            list = THPObjectPtr(PyList_New((Py_ssize_t)outs.size()));
            if (!list) return nullptr;
            for (size_t i = 0; i < outs.size(); i++) PyList_SET_ITEM(list.get(), (Py_ssize_t)i, wrap(outs[i]));
        }
        THPObjectPtr n(wrap(norm));
        return PyTuple_Pack(2, n.get(), list.get());
    });
}

// load(path of libf8mi.so, error class): resolves the entry points
PyObject* load(PyObject*, PyObject* args) {
    const char* path;
    PyObject* error;
    if (!PyArg_ParseTuple(args, "sO", &path, &error)) return nullptr;
    void* h = dlopen(path, RTLD_NOW | RTLD_LOCAL);
    if (!h) return PyErr_Format(PyExc_ImportError, "%s", dlerror());
    const char* missing = nullptr;
    auto get = [&](auto& f, const char* name) {
        f = reinterpret_cast<std::decay_t<decltype(f)>>(dlsym(h, name));
        if (!f) missing = name;
    };
    get(L.block_scale_bytes, "f8mi_block_scale_bytes");
    get(L.block_cast, "f8mi_block_cast");
    get(L.block_gemm, "f8mi_block_gemm");
    get(L.block_gemm_workspace_bytes, "f8mi_block_gemm_workspace_bytes");
    get(L.block_linear_few_rows, "f8mi_block_linear_few_rows");
    get(L.column_sum_finish, "f8mi_column_sum_finish");
    get(L.layer_norm, "f8mi_layer_norm");
    get(L.layer_norm_backward, "f8mi_layer_norm_backward");
    get(L.layer_norm_workspace_bytes, "f8mi_layer_norm_workspace_bytes");
    get(L.grad_clip, "f8mi_grad_clip");
    get(L.grad_clip_workspace_bytes, "f8mi_grad_clip_workspace_bytes");
    get(L.last_error, "f8mi_last_error");
    if (missing) {
        L.last_error = nullptr;
        return PyErr_Format(PyExc_ImportError, "%s does not export %s", path, missing);
    }
    THPObjectPtr module(PyImport_ImportModule("torch.utils._device"));
    device_context = module ? PyObject_GetAttrString(module.get(), "DeviceContext") : nullptr;
    if (!device_context) {
        L.last_error = nullptr;
        return nullptr;
    }
    Py_INCREF(error);
    native_error = error;
    Py_RETURN_NONE;
}

template <typename F>
PyCFunction fast(F f) { return (PyCFunction)(void (*)(void))f; }
PyMethodDef methods[] = {
    {"load", load, METH_VARARGS, nullptr},
    {"blockwise_linear", fast(blockwise_linear), METH_FASTCALL, nullptr},
    {"blockwise_inference_linear", fast(blockwise_inference_linear), METH_FASTCALL, nullptr},
    {"layer_norm", fast(layer_norm), METH_FASTCALL, nullptr},
    {"grad_clip", fast(grad_clip), METH_FASTCALL, nullptr},
    {nullptr, nullptr, 0, nullptr},
};
PyModuleDef module = {PyModuleDef_HEAD_INIT, "_f8mi_torch_ops", nullptr, -1, methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__f8mi_torch_ops(void) { return PyModule_Create(&module); }
