// The host path of RMS norm, dropout, low-rank adapters and the served blockwise linear on activations that have been cast, over libf8mi's C ABI, as a
// CPython module on torch tensors: one call allocates what the kernels write and queues all launches, and the backward passes are nodes that
// run without the interpreter.
//
// Every function returns None, without having queued or allocated anything, for what it does not take (subclasses, other devices, types or shapes) and while
// somebody has to see operators (modes, traces): the caller then says what is wrong, or goes through the registered operators.  Workspaces are temporaries of
// torch's caching allocator, which hands their memory out again in stream order.
#include <c10/hip/HIPCachingAllocator.h>

#include "f8mi_torch_util.h"

namespace {

struct Lib {
    decltype(&f8mi_block_scale_bytes) block_scale_bytes;
    decltype(&f8mi_block_gemm) block_gemm;
    decltype(&f8mi_block_gemm_workspace_bytes) block_gemm_workspace_bytes;
    decltype(&f8mi_rms_norm) rms_norm;
    decltype(&f8mi_rms_norm_block) rms_norm_block;
    decltype(&f8mi_rms_norm_backward) rms_norm_backward;
    decltype(&f8mi_rms_norm_workspace_bytes) rms_norm_workspace_bytes;
    decltype(&f8mi_dropout) dropout;
    decltype(&f8mi_adapter_rows_words) adapter_rows_words;
    decltype(&f8mi_adapters) adapters;
    decltype(&f8mi_adapters_workspace_bytes) adapters_workspace_bytes;
    decltype(&f8mi_adapters_backward) adapters_backward;
    decltype(&f8mi_adapters_backward_workspace_bytes) adapters_backward_workspace_bytes;
} L;

// A dense tensor of `type` on the device that a call runs on, that nobody follows
bool dense(const at::Tensor& t, int device, at::ScalarType type) {
    using K = c10::DispatchKey;
    constexpr c10::DispatchKeySet others({K::Python, K::FuncTorchBatched, K::FuncTorchGradWrapper, K::Batched, K::Functionalize, K::Negative, K::ZeroTensor});
    return t.defined() && t.is_cuda() && t.layout() == at::kStrided && !t.key_set().has_any(others) && t.get_device() == device && t.scalar_type() == type && t.is_contiguous();
}
at::Tensor empty_like_sizes(const at::Tensor& t, at::IntArrayRef sizes) { return at::empty(sizes, t.options().memory_format(at::MemoryFormat::Contiguous)); }
at::Tensor workspace(const at::Tensor& like, int64_t bytes) { return bytes ? at::empty({bytes}, like.options().dtype(at::kByte).memory_format(at::MemoryFormat::Contiguous)) : at::Tensor(); }
at::Tensor in_type(const at::Tensor& t, at::ScalarType type) { return t.scalar_type() == type ? t : t.to(type); }

// ---- RMS norm

struct RmsNorm : torch::autograd::Function<RmsNorm> {
    static at::Tensor compute(const at::Tensor& x, const at::Tensor& weight, const at::Tensor& residual, int64_t cols, double eps, at::Tensor* sum, at::Tensor* rstd) {
        const c10::DeviceGuard guard(x.device());
        const Below below;
        const Rows r(x, cols);
        const int pt = weight.defined() ? dtype_code(weight.scalar_type()) : r.dtype();
        const at::Tensor w = weight.defined() ? weight.contiguous() : weight;
        const at::Tensor y = empty_like_sizes(x, x.sizes());
        if (rstd) *rstd = at::empty({r.rows}, x.options().dtype(at::kFloat));
        std::optional<Rows> res;
        if (residual.defined()) {
            res.emplace(residual, cols);
            *sum = empty_like_sizes(x, x.sizes());
        }
        if (r.rows)
            check(L.rms_norm(r.t.data_ptr(), r.ld, res ? res->t.data_ptr() : nullptr, res ? res->ld : 0, r.rows, cols, r.dtype(), ptr(w), pt, (float)eps, y.data_ptr(), res ? sum->data_ptr() : nullptr,
                             rstd ? (float*)rstd->data_ptr() : nullptr, stream_of(x)), "f8mi_rms_norm");
        return y;
    }
    static variable_list forward(AutogradContext* ctx, const at::Tensor& x, const MaybeTensor& weight_, const MaybeTensor& residual_, int64_t cols, double eps) {
        const at::Tensor weight = weight_.value_or(at::Tensor()), residual = residual_.value_or(at::Tensor());
        at::Tensor sum, rstd;
        at::Tensor y = compute(x, weight, residual, cols, eps, &sum, &rstd);
        ctx->set_materialize_grads(false);
        ctx->save_for_backward({residual.defined() ? sum : x, weight, rstd});
        ctx->saved_data["x_shape"] = x.sizes().vec();
        ctx->saved_data["types"] = (int64_t)x.scalar_type() | (int64_t)(weight.defined() ? weight.scalar_type() : x.scalar_type()) << 8 | (int64_t)weight.defined() << 16 | (int64_t)residual.defined() << 17;
        ctx->saved_data["cols"] = cols;
        ctx->saved_data["w_shape"] = weight.defined() ? weight.sizes().vec() : std::vector<int64_t>();
        return residual.defined() ? variable_list{y, sum} : variable_list{y};
    }
    static variable_list backward(AutogradContext* ctx, const variable_list& grads) {
        TORCH_CHECK(!at::GradMode::is_enabled(), "rms_norm has no second derivative (create_graph=True)");
        const int64_t types = ctx->saved_data["types"].toInt(), cols = ctx->saved_data["cols"].toInt();
        const at::ScalarType xt = (at::ScalarType)(types & 255), pt = (at::ScalarType)(types >> 8 & 255);
        const bool has_weight = types >> 16 & 1, has_residual = types >> 17 & 1;
        const bool need_dx = ctx->needs_input_grad(0), need_dw = has_weight && ctx->needs_input_grad(1), need_dr = has_residual && ctx->needs_input_grad(has_weight ? 2 : 1);
        const auto shape = ctx->saved_data["x_shape"].toIntVector();
        at::Tensor dx, dw;
        const at::Tensor ds = has_residual ? grads[1] : at::Tensor();
        auto result = [&] { return variable_list{need_dx ? dx : at::Tensor(), dw, need_dr ? dx : at::Tensor(), at::Tensor(), at::Tensor()}; };
        if (!grads[0].defined()) {  // y is not used: what comes is the gradient of the sum
            if (ds.defined()) dx = in_type(ds, xt);
            return result();
        }
        if (!(need_dx || need_dw || need_dr)) return result();
        const auto saved = ctx->get_saved_variables();
        const at::Tensor &s = saved[0], &rstd = saved[2];
        const at::Device device = grads[0].device();
        const c10::DeviceGuard guard(device);
        const Below below;
        TORCH_CHECK(as_saved(s, device, xt, shape) && as_saved(rstd, device, at::kFloat, {s.numel() / cols}) && rstd.is_contiguous() && !rstd.is_neg() && saved[1].defined() == has_weight &&
                        (!has_weight || as_saved(saved[1], device, pt, ctx->saved_data["w_shape"].toIntVector())),
                    "rms_norm: what was saved for backward is not what came back");
        const Rows r(s, cols), dy(in_type(grads[0], xt), cols);
        std::optional<Rows> d;
        if (ds.defined()) d.emplace(in_type(ds, xt), cols);
        const at::Tensor w = has_weight ? saved[1].resolve_neg().contiguous() : saved[1];
        if (need_dx || need_dr) dx = empty_like_sizes(s, shape);
        if (need_dw) dw = at::empty(ctx->saved_data["w_shape"].toIntVector(), s.options().dtype(pt).memory_format(at::MemoryFormat::Contiguous));
        const int64_t bytes = need_dw ? L.rms_norm_workspace_bytes(r.rows, cols, r.dtype(), dtype_code(pt)) : 0;
        const at::Tensor ws = workspace(s, bytes);
        check(L.rms_norm_backward(ptr(dy.t), dy.ld, ptr(r.t), r.ld, d ? ptr(d->t) : nullptr, d ? d->ld : 0, r.rows, cols, r.dtype(), ptr(w), dtype_code(pt), (const float*)ptr(rstd), ptr(dx), ptr(dw),
                                  ptr(ws), bytes, stream_of(s)), "f8mi_rms_norm_backward");
        return result();
    }
};

// ---- dropout

struct Dropout : torch::autograd::Function<Dropout> {
    // x and the residual as n dense values
    static at::Tensor compute(const at::Tensor& x, const at::Tensor& residual, const at::Tensor& seed, double p) {
        const c10::DeviceGuard guard(x.device());
        const Below below;
        const at::Tensor xc = (x.is_neg() ? x.resolve_neg() : x).contiguous(), rc = residual.defined() ? (residual.is_neg() ? residual.resolve_neg() : residual).contiguous() : residual;
        const at::Tensor out = empty_like_sizes(x, x.sizes());
        if (x.numel()) check(L.dropout(xc.data_ptr(), ptr(rc), x.numel(), dtype_code(x.scalar_type()), p, (const int64_t*)seed.data_ptr(), out.data_ptr(), stream_of(x)), "f8mi_dropout");
        return out;
    }
    static at::Tensor forward(AutogradContext* ctx, const at::Tensor& x, const MaybeTensor& residual, const at::Tensor& seed, double p) {
        ctx->save_for_backward({seed});
        ctx->saved_data["p"] = p;
        ctx->saved_data["type"] = (int64_t)x.scalar_type();
        ctx->saved_data["residual"] = residual.has_value();
        return compute(x, residual.value_or(at::Tensor()), seed, p);
    }
    static variable_list backward(AutogradContext* ctx, const variable_list& grads) {
        TORCH_CHECK(!at::GradMode::is_enabled(), "dropout has no second derivative (create_graph=True)");
        at::Tensor dx;
        if (!grads[0].defined()) return {dx, dx, dx, dx};
        const at::Tensor g = in_type(grads[0], (at::ScalarType)ctx->saved_data["type"].toInt());
        if (ctx->needs_input_grad(0)) {
            const auto saved = ctx->get_saved_variables();
            TORCH_CHECK(as_saved(saved[0], g.device(), at::kLong, saved[0].sizes()) && saved[0].numel() == 1 && !saved[0].is_neg(), "dropout: what was saved for backward is not what came back");
            dx = compute(g, {}, saved[0], ctx->saved_data["p"].toDouble());
        }
        return {dx, ctx->saved_data["residual"].toBool() && ctx->needs_input_grad(1) ? g : at::Tensor(), at::Tensor(), at::Tensor()};
    }
};

// ---- low-rank adapters

struct Adapters : torch::autograd::Function<Adapters> {
    static at::Tensor compute(const at::Tensor& x, const at::Tensor& a, const at::Tensor& b, const at::Tensor& y, const at::Tensor& table, const at::Tensor& scale, double factor, at::Tensor* h) {
        const c10::DeviceGuard guard(x.device());
        const Below below;
        // A batch's table belongs to the stream that it was made on, and the next batch's takes its place (select_adapters): the allocator has to know that another stream still reads it.  (Nothing
        // where it is the same stream.)
        c10::hip::HIPCachingAllocator::recordStream(table.storage().data_ptr(), c10::hip::getCurrentHIPStream(x.get_device()));
        const int64_t count = a.size(0), rank = a.size(1), k = a.size(2), n = b.size(1);
        const Rows xr(x, k);
        std::optional<Rows> yr;
        if (y.defined()) yr.emplace(y, n);
        const at::Tensor ac = in_type(a, x.scalar_type()).contiguous(), bc = in_type(b, x.scalar_type()).contiguous();
        std::vector<int64_t> shape(x.sizes().begin(), x.sizes().end());
        shape.back() = n;
        const at::Tensor out = empty_like_sizes(x, shape);
        if (h) *h = at::empty({xr.rows, (rank + 15) / 16 * 16}, x.options().dtype(at::kFloat).memory_format(at::MemoryFormat::Contiguous));
        if (xr.rows == 0) return out;
        const int64_t bytes = L.adapters_workspace_bytes(xr.rows, k, n, rank, count, xr.dtype());
        const at::Tensor ws = workspace(x, bytes);
        check(L.adapters(xr.t.data_ptr(), xr.ld, ac.data_ptr(), bc.data_ptr(), (const float*)ptr(scale), (float)factor, table.data_ptr(), xr.rows, k, n, rank, count, xr.dtype(),
                         yr ? yr->t.data_ptr() : nullptr, yr ? yr->ld : 0, out.data_ptr(), h ? (float*)h->data_ptr() : nullptr, ptr(ws), bytes, stream_of(x)), "f8mi_adapters");
        return out;
    }
    static at::Tensor forward(AutogradContext* ctx, const at::Tensor& x, const at::Tensor& a, const at::Tensor& b, const MaybeTensor& y, const at::Tensor& table, const MaybeTensor& scale, double factor,
                              bool need_da, bool need_db) {
        at::Tensor h;
        at::Tensor out = compute(x, a, b, y.value_or(at::Tensor()), table, scale.value_or(at::Tensor()), factor, need_db ? &h : nullptr);
        ctx->save_for_backward({need_da ? x : at::Tensor(), a, b, table, scale.value_or(at::Tensor()), h});
        ctx->saved_data["x_shape"] = x.sizes().vec();
        ctx->saved_data["a_shape"] = a.sizes().vec();
        ctx->saved_data["n"] = b.size(1);
        ctx->saved_data["types"] = (int64_t)x.scalar_type() | (int64_t)a.scalar_type() << 8 | (int64_t)y.has_value() << 16 | (int64_t)scale.has_value() << 17 | (int64_t)need_db << 18 | (int64_t)need_da << 19;
        ctx->saved_data["factor"] = factor;
        return out;
    }
    static variable_list backward(AutogradContext* ctx, const variable_list& grads) {
        TORCH_CHECK(!at::GradMode::is_enabled(), "low_rank_adapters has no second derivative (create_graph=True)");
        const int64_t types = ctx->saved_data["types"].toInt();
        const at::ScalarType xt = (at::ScalarType)(types & 255), pt = (at::ScalarType)(types >> 8 & 255);
        const bool has_y = types >> 16 & 1, has_scale = types >> 17 & 1, kept_h = types >> 18 & 1, kept_x = types >> 19 & 1;
        const bool need_dx = ctx->needs_input_grad(0), need_da = ctx->needs_input_grad(1), need_db = ctx->needs_input_grad(2), need_dy = has_y && ctx->needs_input_grad(3);
        at::Tensor dx, da, db, none;
        if (!grads[0].defined()) return {none, none, none, none, none, none, none, none, none};
        const at::Tensor g = in_type(grads[0], xt);
        auto result = [&] { return variable_list{dx, da, db, need_dy ? g : none, none, none, none, none, none}; };
        if (!(need_dx || need_da || need_db)) return result();
        const auto x_shape = ctx->saved_data["x_shape"].toIntVector(), a_shape = ctx->saved_data["a_shape"].toIntVector();
        const int64_t count = a_shape[0], rank = a_shape[1], k = a_shape[2], n = ctx->saved_data["n"].toInt();
        const c10::Device device = g.device();
        const c10::DeviceGuard guard(device);
        const auto saved = ctx->get_saved_variables();
        const at::Tensor &x = saved[0], &a = saved[1], &b = saved[2], &table = saved[3], &scale = saved[4], &h = saved[5];
        const Below below;
        const Rows gr(g, n);
        TORCH_CHECK((!need_da || (kept_x && as_saved(x, device, xt, x_shape))) && as_saved(a, device, pt, a_shape) && as_saved(b, device, pt, {count, n, rank}) &&
                        as_saved(table, device, at::kInt, {L.adapter_rows_words(gr.rows, count)}) && table.is_contiguous() && !table.is_neg() && scale.defined() == has_scale &&
                        (!has_scale || (as_saved(scale, device, at::kFloat, {count}) && scale.is_contiguous() && !scale.is_neg())) && (!need_db || kept_h) &&
                        (!need_db || (as_saved(h, device, at::kFloat, {gr.rows, (rank + 15) / 16 * 16}) && h.is_contiguous() && !h.is_neg())),
                    "low_rank_adapters: what was saved for backward is not what came back");
        std::optional<Rows> xr;
        if (need_da) xr.emplace(x, k);
        const at::Tensor ac = in_type(a, xt).resolve_neg().contiguous(), bc = in_type(b, xt).resolve_neg().contiguous();
        if (need_dx) dx = empty_like_sizes(g, x_shape);
        const auto p_options = g.options().dtype(pt).memory_format(at::MemoryFormat::Contiguous);
        if (gr.rows == 0) {
            if (need_da) da = at::zeros(a_shape, p_options);
            if (need_db) db = at::zeros({count, n, rank}, p_options);
            return result();
        }
        if (need_da) da = at::empty(a_shape, p_options);
        if (need_db) db = at::empty({count, n, rank}, p_options);
        const int64_t bytes = L.adapters_backward_workspace_bytes(gr.rows, k, n, rank, count, gr.dtype(), need_dx, need_da, need_db);
        const at::Tensor ws = workspace(g, bytes);
        check(L.adapters_backward(ptr(gr.t), gr.ld, xr ? ptr(xr->t) : nullptr, xr ? xr->ld : 0, ptr(ac), ptr(bc), (const float*)ptr(scale), (float)ctx->saved_data["factor"].toDouble(), ptr(table), (const float*)ptr(h), gr.rows, k, n,
                                  rank, count, gr.dtype(), ptr(dx), ptr(da), ptr(db), dtype_code(pt), ptr(ws), bytes, stream_of(g)), "f8mi_adapters_backward");
        return result();
    }
};

// ---- Python

// A shape that x ends in (an int or a tuple): its number of values, and of dimensions; 0: it is none
int64_t trailing(PyObject* o, const at::Tensor& x, int64_t& d) {
    std::vector<int64_t> shape;
    if (PyLong_Check(o)) shape.push_back(PyLong_AsLongLong(o));
    else if (PyTuple_Check(o))  // (torch.Size is one)
        for (Py_ssize_t i = 0; i < PyTuple_GET_SIZE(o); i++) {
            if (!PyLong_Check(PyTuple_GET_ITEM(o, i))) return 0;
            shape.push_back(PyLong_AsLongLong(PyTuple_GET_ITEM(o, i)));
        }
    if (PyErr_Occurred()) {  // a number that no dimension has
        PyErr_Clear();
        return 0;
    }
    d = (int64_t)shape.size();
    if (d == 0 || x.dim() < d || x.sizes().slice(x.dim() - d) != at::IntArrayRef(shape)) return 0;
    int64_t cols = 1;
    for (const int64_t s : shape) cols *= s;
    return std::max<int64_t>(cols, 0);
}

struct RmsCall {  // the arguments that both forms of the norm take: x, normalized_shape, weight or None, eps, residual or None
    at::Tensor x, weight, residual;
    int64_t cols = 0;
    double eps = 0;
    bool taken(PyObject* const* a) {
        const int device = device_taken();
        x = plain(a[0], device);
        if (!x.defined() || !optional(a[2], device, weight) || !optional(a[4], device, residual)) return false;
        int64_t dims = 0;
        cols = trailing(a[1], x, dims);
        if (cols == 0 || (residual.defined() && (residual.sizes() != x.sizes() || residual.scalar_type() != x.scalar_type()))) return false;
        if (weight.defined() && (weight.sizes() != x.sizes().slice(x.dim() - dims) || (weight.scalar_type() != x.scalar_type() && weight.scalar_type() != at::kFloat))) return false;
        eps = PyFloat_AsDouble(a[3]);
        return true;
    }
};

// rms_norm(x, normalized_shape, weight or None, eps, residual or None) -> y, or (y, sum) with a residual, with their history, or None
PyObject* rms_norm(PyObject*, PyObject* const* a, Py_ssize_t n_args) {
    if (!expect(n_args, 5, "rms_norm")) return nullptr;
    return guarded([&]() -> PyObject* {
        RmsCall c;
        if (!c.taken(a)) Py_RETURN_NONE;
        if (c.eps == -1.0 && PyErr_Occurred()) return nullptr;
        at::Tensor y, sum;
        {
            const WithoutGil no_gil;
            if (wants_grad(c.x) || wants_grad(c.weight) || wants_grad(c.residual)) {
                const variable_list out = RmsNorm::apply(c.x, maybe(c.weight), maybe(c.residual), c.cols, c.eps);
                y = out[0];
                if (out.size() > 1) sum = out[1];
            } else {
                y = RmsNorm::compute(c.x, c.weight, c.residual, c.cols, c.eps, &sum, nullptr);
            }
        }
        if (!c.residual.defined()) return wrap(y);
        THPObjectPtr first(wrap(y)), second(wrap(sum));
        return PyTuple_Pack(2, first.get(), second.get());
    });
}

// rms_norm_blockwise(x, normalized_shape, weight or None, eps, residual or None) -> (data, scales, sum or None), or None
PyObject* rms_norm_blockwise(PyObject*, PyObject* const* a, Py_ssize_t n_args) {
    if (!expect(n_args, 5, "rms_norm_blockwise")) return nullptr;
    return guarded([&]() -> PyObject* {
        RmsCall c;
        if (!c.taken(a)) Py_RETURN_NONE;
        if (c.eps == -1.0 && PyErr_Occurred()) return nullptr;
        if (c.cols != c.x.size(-1) || wants_grad(c.x) || wants_grad(c.weight) || wants_grad(c.residual)) Py_RETURN_NONE;
        at::Tensor data, scales, sum;
        {
            const WithoutGil no_gil;
            const c10::DeviceGuard guard(c.x.device());
            const Below below;
            const Rows r(c.x, c.cols);
            std::optional<Rows> res;
            if (c.residual.defined()) {
                res.emplace(c.residual, c.cols);
                sum = empty_like_sizes(c.x, c.x.sizes());
            }
            const int64_t kp = (c.cols + 127) / 128 * 128;
            const at::Tensor w = c.weight.defined() ? c.weight.contiguous() : c.weight;
            data = at::empty({kp / 64, r.rows, 64}, c.x.options().dtype(at::kFloat8_e4m3fn).memory_format(at::MemoryFormat::Contiguous));
            scales = at::empty({kp / 128, (r.rows + 127) / 128 * 128}, c.x.options().dtype(at::kByte).memory_format(at::MemoryFormat::Contiguous));
            if (r.rows)
                check(L.rms_norm_block(r.t.data_ptr(), r.ld, res ? res->t.data_ptr() : nullptr, res ? res->ld : 0, r.rows, c.cols, r.dtype(), ptr(w), w.defined() ? dtype_code(w.scalar_type()) : r.dtype(),
                                       (float)c.eps, data.data_ptr(), scales.data_ptr(), res ? sum.data_ptr() : nullptr, stream_of(c.x)), "f8mi_rms_norm_block");
        }
        THPObjectPtr d(wrap(data)), s(wrap(scales)), t(wrap(sum));
        return PyTuple_Pack(3, d.get(), s.get(), t.get());
    });
}

// blockwise_inference_linear_cast(data, scales of the activations, rows, dtype of the result, data, scales of the weight, n, k, bias or None) -> y [rows, n] or None
PyObject* blockwise_inference_linear_cast(PyObject*, PyObject* const* a, Py_ssize_t n_args) {
    if (!expect(n_args, 9, "blockwise_inference_linear_cast")) return nullptr;
    return guarded([&]() -> PyObject* {
        const int device = device_taken();
        const int64_t rows = PyLong_AsLongLong(a[2]), n = PyLong_AsLongLong(a[6]), k = PyLong_AsLongLong(a[7]), kp = (k + 127) / 128 * 128;
        at::Tensor bias;
        for (const int i : {0, 1, 4, 5})
            if (!THPVariable_CheckExact(a[i])) Py_RETURN_NONE;
        if (!THPDtype_Check(a[3]) || !optional(a[8], device, bias) || rows < 0 || n <= 0 || k <= 0 || (bias.defined() && (bias.dim() != 1 || bias.size(0) != n))) Py_RETURN_NONE;
        const at::ScalarType type = ((THPDtype*)a[3])->scalar_type;
        const at::Tensor x8 = THPVariable_Unpack(a[0]), xs = THPVariable_Unpack(a[1]), w8 = THPVariable_Unpack(a[4]), ws = THPVariable_Unpack(a[5]);
        if (dtype_code(type) < 0 || !dense(x8, device, at::kFloat8_e4m3fn) || x8.numel() != kp * rows || !dense(xs, device, at::kByte) || xs.numel() != L.block_scale_bytes(rows, k) ||
            !dense(w8, device, at::kFloat8_e4m3fn) || w8.numel() != kp * n || !dense(ws, device, at::kByte) || ws.numel() != L.block_scale_bytes(n, k))
            Py_RETURN_NONE;
        at::Tensor y;
        {
            const WithoutGil no_gil;
            const c10::DeviceGuard guard(x8.device());
            const Below below;
            const at::Tensor b = bias.defined() ? bias.to(type).contiguous() : at::Tensor();
            if (rows == 0) y = at::empty({0, n}, x8.options().dtype(type));
            else y = block_gemm(L, x8, {(uint8_t*)x8.data_ptr(), (uint8_t*)xs.data_ptr()}, {(uint8_t*)w8.data_ptr(), (uint8_t*)ws.data_ptr()}, false, rows, n, k, type, b);
        }
        return wrap(y);
    });
}

// dropout(x, p, seed, residual or None) -> out, with its history, or None
PyObject* dropout(PyObject*, PyObject* const* a, Py_ssize_t n_args) {
    if (!expect(n_args, 4, "dropout")) return nullptr;
    return guarded([&]() -> PyObject* {
        const int device = device_taken();
        const at::Tensor x = plain(a[0], device);
        at::Tensor residual;
        if (!x.defined() || !optional(a[3], device, residual) || !THPVariable_CheckExact(a[2])) Py_RETURN_NONE;
        const at::Tensor seed = THPVariable_Unpack(a[2]);
        if (!dense(seed, device, at::kLong) || seed.numel() != 1 || (residual.defined() && (residual.sizes() != x.sizes() || residual.scalar_type() != x.scalar_type()))) Py_RETURN_NONE;
        const double p = PyFloat_AsDouble(a[1]);
        if (p == -1.0 && PyErr_Occurred()) return nullptr;
        if (!(p >= 0.0 && p < 1.0)) Py_RETURN_NONE;
        at::Tensor out;
        {
            const WithoutGil no_gil;
            if (wants_grad(x) || wants_grad(residual)) out = Dropout::apply(x, maybe(residual), seed, p);
            else out = Dropout::compute(x, residual, seed, p);
        }
        return wrap(out);
    });
}

// low_rank_adapters(x [..., k], a [count, r, k], b [count, n, r], a batch's table, its rows and its count of adapters, y [..., n] or None, scale [count] (fp32) or None, factor) -> out, with its history, or None
PyObject* low_rank_adapters(PyObject*, PyObject* const* args, Py_ssize_t n_args) {
    if (!expect(n_args, 9, "low_rank_adapters")) return nullptr;
    return guarded([&]() -> PyObject* {
        const int device = device_taken();
        const at::Tensor x = plain(args[0], device), a = plain(args[1], device), b = plain(args[2], device);
        at::Tensor y, scale;
        if (!x.defined() || !a.defined() || !b.defined() || !THPVariable_CheckExact(args[3]) || !optional(args[6], device, y) || !optional(args[7], device, scale)) Py_RETURN_NONE;
        const at::Tensor table = THPVariable_Unpack(args[3]);
        if (a.dim() != 3 || b.dim() != 3 || a.numel() == 0 || b.numel() == 0 || a.size(0) != b.size(0) || a.size(1) != b.size(2) || a.scalar_type() != b.scalar_type() || x.dim() == 0 ||
            x.size(-1) != a.size(2) || a.size(1) > F8MI_ADAPTER_MAX_RANK)
            Py_RETURN_NONE;
        const int64_t count = a.size(0), rows = x.numel() / a.size(2);
        if (PyLong_AsLongLong(args[4]) != rows || PyLong_AsLongLong(args[5]) != count) Py_RETURN_NONE;
        if (!dense(table, device, at::kInt) || table.dim() != 1 || table.numel() != L.adapter_rows_words(rows, count)) Py_RETURN_NONE;
        if (scale.defined() && (scale.scalar_type() != at::kFloat || scale.dim() != 1 || scale.size(0) != count || !scale.is_contiguous() || wants_grad(scale))) Py_RETURN_NONE;
        if (y.defined() && (y.scalar_type() != x.scalar_type() || y.dim() != x.dim() || y.size(-1) != b.size(1) || y.sizes().slice(0, y.dim() - 1) != x.sizes().slice(0, x.dim() - 1))) Py_RETURN_NONE;
        const double factor = PyFloat_AsDouble(args[8]);
        if (factor == -1.0 && PyErr_Occurred()) return nullptr;
        at::Tensor out;
        {
            const WithoutGil no_gil;
            if (wants_grad(x) || wants_grad(a) || wants_grad(b) || wants_grad(y)) out = Adapters::apply(x, a, b, maybe(y), table, maybe(scale), factor, wants_grad(a), wants_grad(b));
            else out = Adapters::compute(x, a, b, y, table, scale, factor, nullptr);
        }
        return wrap(out);
    });
}

// load(path of libf8mi.so, error class): resolves the entry points
PyObject* load(PyObject*, PyObject* args) {
    Loader lib;
    if (!lib.open(args)) return nullptr;
    lib.get(L.block_scale_bytes, "f8mi_block_scale_bytes");
    lib.get(L.block_gemm, "f8mi_block_gemm");
    lib.get(L.block_gemm_workspace_bytes, "f8mi_block_gemm_workspace_bytes");
    lib.get(L.rms_norm, "f8mi_rms_norm");
    lib.get(L.rms_norm_block, "f8mi_rms_norm_block");
    lib.get(L.rms_norm_backward, "f8mi_rms_norm_backward");
    lib.get(L.rms_norm_workspace_bytes, "f8mi_rms_norm_workspace_bytes");
    lib.get(L.dropout, "f8mi_dropout");
    lib.get(L.adapter_rows_words, "f8mi_adapter_rows_words");
    lib.get(L.adapters, "f8mi_adapters");
    lib.get(L.adapters_workspace_bytes, "f8mi_adapters_workspace_bytes");
    lib.get(L.adapters_backward, "f8mi_adapters_backward");
    lib.get(L.adapters_backward_workspace_bytes, "f8mi_adapters_backward_workspace_bytes");
    return lib.done();
}

PyMethodDef methods[] = {
    {"load", load, METH_VARARGS, nullptr},
    {"rms_norm", fast(rms_norm), METH_FASTCALL, nullptr},
    {"rms_norm_blockwise", fast(rms_norm_blockwise), METH_FASTCALL, nullptr},
    {"blockwise_inference_linear_cast", fast(blockwise_inference_linear_cast), METH_FASTCALL, nullptr},
    {"dropout", fast(dropout), METH_FASTCALL, nullptr},
    {"low_rank_adapters", fast(low_rank_adapters), METH_FASTCALL, nullptr},
    {nullptr, nullptr, 0, nullptr},
};
PyModuleDef module = {PyModuleDef_HEAD_INIT, "_f8mi_torch_model", nullptr, -1, methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__f8mi_torch_model(void) { return PyModule_Create(&module); }
