"""The blockwise scaled linear and layer norm as ``torch.library`` custom ops, for ``torch.compile`` and whoever else has to see operators: opaque
nodes with known shapes, one per direction, with the numbers of the eager path."""
import contextlib
from typing import Optional, Tuple

import torch

from . import _native

_e4m3 = torch.float8_e4m3fn
_KB, _BLOCK = _native.KB, _native.BLOCK
_HP_DTYPES = (torch.bfloat16, torch.float16, torch.float32)


def _data_shape(rows: int, k: int):
    return (_native.padded_k(k) // _KB, rows, _KB)


def _scales_shape(rows: int, k: int):
    return (_native.padded_k(k) // _BLOCK, -(-rows // _BLOCK) * _BLOCK)


def _one_weight_copy(k: int, n: int) -> bool:
    return k % _BLOCK == 0 and n % _BLOCK == 0


def _check_operands(what: str, x2: torch.Tensor, *operands) -> None:
    """Each operand (name, tensor or None, shape, types) is what the kernels read beside the matrix x2.  The entry points have checked their arguments, but not those that a trace is
    replayed with or that hooks on saved tensors hand back: without this their memory would be read past its end."""
    if x2.dim() != 2 or x2.dtype not in _HP_DTYPES:
        raise _native.Float8NativeError(f"{what}: {tuple(x2.shape)} ({x2.dtype}) is no matrix of bfloat16, float16 or float32")
    for name, t, shape, dtypes in operands:
        if t is not None and (tuple(t.shape) != tuple(shape) or t.dtype not in dtypes or t.device != x2.device):
            raise _native.Float8NativeError(f"{what}: {name} {tuple(t.shape)} ({t.dtype}) on {t.device} beside {tuple(x2.shape)} ({x2.dtype}) on {x2.device}; {tuple(shape)} is needed")


@torch.library.custom_op("f8mi::blockwise_linear_fwd", mutates_args=())
def blockwise_linear_fwd(x2: torch.Tensor, weight: torch.Tensor, bias: Optional[torch.Tensor], need_dx: bool, need_dw: bool) -> Tuple[
        torch.Tensor, torch.Tensor, torch.Tensor, torch.Tensor, torch.Tensor]:
    """(y, x transposed: data, scales; weight for the gradient of x: data, scales); what backward will not need is empty."""
    (m, k), n = x2.shape, weight.shape[0]
    one = _one_weight_copy(k, n)
    empty = lambda dt: torch.empty(0, dtype=dt, device=x2.device)
    if m == 0:  # nothing is read in backward, but the shapes are those of any number of tokens
        return _blockwise_linear_shapes(x2, weight, need_dx, need_dw)
    with _native.transient_workspaces():
        (x8, x8t), (w8, w8t) = _native.block_cast([(x2, False, True, need_dw), (weight, True, True, need_dx and ("scales" if one else True))])
        y = _native.block_gemm(x8, w8, x2.dtype, None if bias is None else bias.to(x2.dtype).contiguous())
    return (y, x8t.data if need_dw else empty(_e4m3), x8t.scales if need_dw else empty(torch.uint8),
            (w8.data if one else w8t.data) if need_dx else empty(_e4m3), w8t.scales if need_dx else empty(torch.uint8))


def _blockwise_linear_shapes(x2, weight, need_dx, need_dw):
    (m, k), n = x2.shape, weight.shape[0]
    make = lambda shape, dt, wanted: torch.empty(shape if wanted else (0,), dtype=dt, device=x2.device)
    w_shape = _data_shape(n, k) if _one_weight_copy(k, n) else _data_shape(k, n)
    return (torch.empty((m, n), dtype=x2.dtype, device=x2.device), make(_data_shape(k, m), _e4m3, need_dw), make(_scales_shape(k, m), torch.uint8, need_dw),
            make(w_shape, _e4m3, need_dx), make(_scales_shape(k, n), torch.uint8, need_dx))


@blockwise_linear_fwd.register_fake
def _(x2, weight, bias, need_dx, need_dw):
    return _blockwise_linear_shapes(x2, weight, need_dx, need_dw)


@torch.library.custom_op("f8mi::blockwise_linear_bwd", mutates_args=())
def blockwise_linear_bwd(dy2: torch.Tensor, xt: torch.Tensor, xt_scales: torch.Tensor, w: torch.Tensor, w_scales: torch.Tensor, k: int, w_dtype: torch.dtype,
                         b_dtype: Optional[torch.dtype], need_dx: bool, need_dw: bool) -> Tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
    """(dx, dw, dbias); an unneeded gradient (``b_dtype`` None: of the bias) is empty."""
    m, n = dy2.shape
    empty = lambda dt: torch.empty(0, dtype=dt, device=dy2.device)
    if m == 0:
        return (dy2.new_empty((0, k)) if need_dx else empty(dy2.dtype), dy2.new_zeros((n, k), dtype=w_dtype) if need_dw else empty(w_dtype),
                dy2.new_zeros(n, dtype=b_dtype) if b_dtype is not None else empty(dy2.dtype))
    w_shape = _data_shape(n, k) if _one_weight_copy(k, n) else _data_shape(k, n)
    _check_operands("blockwise_linear, backward", dy2, ("x", xt if need_dw else None, _data_shape(k, m), (_e4m3,)), ("x's scales", xt_scales if need_dw else None, _scales_shape(k, m), (torch.uint8,)),
                    ("weight", w if need_dx else None, w_shape, (_e4m3,)), ("the weight's scales", w_scales if need_dx else None, _scales_shape(k, n), (torch.uint8,)))
    xt, xt_scales, w, w_scales = (t.contiguous() for t in (xt, xt_scales, w, w_scales))
    with _native.transient_workspaces():
        ((g8, g8t, *db),) = _native.block_cast([(dy2, False, need_dx, need_dw, *([b_dtype] if b_dtype is not None else []))])
        dx, dw = empty(dy2.dtype), empty(w_dtype)
        if need_dx:
            one = _one_weight_copy(k, n)
            dx = _native.block_gemm(g8, _native.Blocks(None if one else w, w_scales, k, n), dy2.dtype, transposed=_native.Blocks(w, None, n, k) if one else None)
        if need_dw:
            dw = _native.block_gemm(g8t, _native.Blocks(xt, xt_scales, k, m), w_dtype)
    return dx, dw, db[0] if db else empty(dy2.dtype)


@blockwise_linear_bwd.register_fake
def _(dy2, xt, xt_scales, w, w_scales, k, w_dtype, b_dtype, need_dx, need_dw):
    m, n = dy2.shape
    return (torch.empty((m, k) if need_dx else (0,), dtype=dy2.dtype, device=dy2.device), torch.empty((n, k) if need_dw else (0,), dtype=w_dtype, device=dy2.device),
            torch.empty(0 if b_dtype is None else n, dtype=b_dtype or dy2.dtype, device=dy2.device))


class _BlockwiseLinearFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x2, weight, bias):
        y, *saved = blockwise_linear_fwd(x2, weight, bias, ctx.needs_input_grad[0], ctx.needs_input_grad[1])
        ctx.k, ctx.w_dtype, ctx.b_dtype = x2.shape[1], weight.dtype, None if bias is None else bias.dtype
        ctx.save_for_backward(*saved)
        return y

    @staticmethod
    def backward(ctx, gy):
        need_dx, need_dw, need_db = ctx.needs_input_grad
        dx, dw, db = blockwise_linear_bwd(gy, *ctx.saved_tensors, ctx.k, ctx.w_dtype, ctx.b_dtype if need_db else None, need_dx, need_dw)
        return dx if need_dx else None, dw if need_dw else None, db if need_db else None


# What a trace holds: one operator with its history, the same with gradients and without, that can be saved (an autograd function cannot).
_traced = torch.library.Library("f8mi", "FRAGMENT")
_traced.define("blockwise_linear(Tensor x2, Tensor weight, Tensor? bias) -> Tensor")
_traced.define("layer_norm(Tensor x2, Tensor? weight, Tensor? bias, float eps) -> Tensor")


@contextlib.contextmanager
def _untraced():
    """What an operator does is not in the trace that holds the operator."""
    state = torch._C._get_tracing_state()
    torch._C._set_tracing_state(None)
    try:
        yield
    finally:
        torch._C._set_tracing_state(state)


def _records(*tensors: Optional[torch.Tensor]) -> bool:
    return torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in tensors)


@torch.library.impl(_traced, "blockwise_linear", "CompositeImplicitAutograd")
def _traced_blockwise_linear(x2, weight, bias):
    with _untraced():
        y = _native.ops().blockwise_linear(x2, weight, bias)
        return _blockwise_linear(x2, weight, bias) if y is None else y


def _blockwise_linear(x2: torch.Tensor, weight: torch.Tensor, bias: Optional[torch.Tensor]) -> torch.Tensor:
    return _BlockwiseLinearFn.apply(x2, weight, bias) if _records(x2, weight, bias) else blockwise_linear_fwd(x2, weight, bias, False, False)[0]


def blockwise_linear(x: torch.Tensor, weight: torch.Tensor, bias: Optional[torch.Tensor]) -> torch.Tensor:
    y = (torch.ops.f8mi.blockwise_linear if torch.jit.is_tracing() else _blockwise_linear)(x.reshape(-1, x.shape[-1]), weight, bias)
    return y.reshape(*x.shape[:-1], weight.shape[0])


@torch.library.custom_op("f8mi::blockwise_inference_linear", mutates_args=())
def _blockwise_inference_linear(x2: torch.Tensor, data: torch.Tensor, scales: torch.Tensor, bias: Optional[torch.Tensor]) -> torch.Tensor:
    n = data.shape[1]
    if x2.shape[0] == 0:
        return x2.new_empty((0, n))
    k = x2.shape[1]
    y = _native.ops().blockwise_inference_linear(x2.detach(), data, scales, n, k, bias)
    if y is not None:
        return y
    if data.dtype is not _e4m3 or data.shape != _data_shape(n, k) or scales.dtype is not torch.uint8 or scales.shape != _scales_shape(n, k) or not (
            x2.device == data.device == scales.device and data.is_contiguous() and scales.is_contiguous()):
        raise _native.Float8NativeError(f"blockwise_inference_linear: {k} in_features on {x2.device} for a weight {tuple(data.shape)} ({data.dtype}) on {data.device} with scales "
                                        f"{tuple(scales.shape)} ({scales.dtype}) on {scales.device}")
    # a mode that is still on inside the operator
    ((x8, _),) = _native.block_cast([(x2.detach(), False, True, False)])
    return _native.block_gemm(x8, _native.Blocks(data, scales, n, k), x2.dtype, None if bias is None else bias.to(x2.dtype).contiguous())


@_blockwise_inference_linear.register_fake
def _(x2, data, scales, bias):
    return torch.empty((x2.shape[0], data.shape[1]), dtype=x2.dtype, device=x2.device)


def blockwise_inference_linear(x: torch.Tensor, data: torch.Tensor, scales: torch.Tensor, bias: Optional[torch.Tensor]) -> torch.Tensor:
    return _blockwise_inference_linear(x.reshape(-1, x.shape[-1]), data, scales, bias).reshape(*x.shape[:-1], data.shape[1])


# ---- layer norm


@torch.library.custom_op("f8mi::layer_norm_fwd", mutates_args=())
def layer_norm_fwd(x2: torch.Tensor, weight: Optional[torch.Tensor], bias: Optional[torch.Tensor], eps: float) -> Tuple[torch.Tensor, torch.Tensor]:
    """(y, (mean, rstd) of each row)"""
    p_dtypes = (x2.dtype, torch.float32) if weight is None or bias is None else (weight.dtype,) if weight.dtype in (x2.dtype, torch.float32) else ()
    _check_operands("layer_norm", x2, ("weight", weight, x2.shape[1:], p_dtypes), ("bias", bias, x2.shape[1:], p_dtypes))
    return _native.layer_norm(x2, weight, bias, eps)


@layer_norm_fwd.register_fake
def _(x2, weight, bias, eps):
    return torch.empty(x2.shape, dtype=x2.dtype, device=x2.device), torch.empty((x2.shape[0], 2), dtype=torch.float32, device=x2.device)


@torch.library.custom_op("f8mi::layer_norm_bwd", mutates_args=())
def layer_norm_bwd(dy2: torch.Tensor, x2: torch.Tensor, weight: Optional[torch.Tensor], p_dtype: torch.dtype, stats: torch.Tensor, need_dx: bool, need_dw: bool,
                   need_db: bool) -> Tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
    """(dx, dweight, dbias); an unneeded gradient is empty."""
    _check_operands("layer_norm, backward", x2, ("the gradient", dy2, x2.shape, (x2.dtype,)), ("weight", weight, x2.shape[1:], (p_dtype,)), ("statistics", stats, (x2.shape[0], 2), (torch.float32,)))
    stats = stats.contiguous()
    grads = _native.layer_norm_backward(dy2, x2, weight, p_dtype, stats, need_dx, need_dw, need_db)
    return tuple(torch.empty(0, dtype=dt, device=x2.device) if g is None else g for g, dt in zip(grads, (x2.dtype, p_dtype, p_dtype)))


@layer_norm_bwd.register_fake
def _(dy2, x2, weight, p_dtype, stats, need_dx, need_dw, need_db):
    p = lambda need: torch.empty(x2.shape[1] if need else 0, dtype=p_dtype, device=x2.device)
    return torch.empty(x2.shape if need_dx else (0,), dtype=x2.dtype, device=x2.device), p(need_dw), p(need_db)


class _LayerNormFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x2, weight, bias, eps):
        y, stats = layer_norm_fwd(x2, weight, bias, eps)
        ctx.p_dtype = next((p.dtype for p in (weight, bias) if p is not None), x2.dtype)
        ctx.has_weight = weight is not None
        ctx.save_for_backward(x2, stats, *([weight] if weight is not None else []))
        return y

    @staticmethod
    def backward(ctx, gy):
        x2, stats, *weight = ctx.saved_tensors
        needs = ctx.needs_input_grad[:3]
        grads = layer_norm_bwd(gy, x2, weight[0] if ctx.has_weight else None, ctx.p_dtype, stats, *needs)
        return tuple(g if need else None for g, need in zip(grads, needs)) + (None,)


@torch.library.impl(_traced, "layer_norm", "CompositeImplicitAutograd")
def _traced_layer_norm(x2, weight, bias, eps):
    with _untraced():
        y = _native.ops().layer_norm(x2, x2.shape[1], weight, bias, eps)
        return _layer_norm(x2, weight, bias, eps) if y is None else y


def _layer_norm(x2: torch.Tensor, weight: Optional[torch.Tensor], bias: Optional[torch.Tensor], eps: float) -> torch.Tensor:
    return _LayerNormFn.apply(x2, weight, bias, eps) if _records(x2, weight, bias) else layer_norm_fwd(x2, weight, bias, eps)[0]


def layer_norm(x: torch.Tensor, weight: Optional[torch.Tensor], bias: Optional[torch.Tensor], cols: int, eps: float) -> torch.Tensor:
    flat = lambda p: None if p is None else p.reshape(-1)
    y = (torch.ops.f8mi.layer_norm if torch.jit.is_tracing() else _layer_norm)(x.reshape(-1, cols), flat(weight), flat(bias), eps)
    return y.reshape(x.shape)
