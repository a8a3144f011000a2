"""RMS norm, dropout, low-rank adapters and the served blockwise linear on activations that have been cast as ``torch.library`` custom ops, for ``torch.compile`` and
whoever else has to see operators: opaque nodes with known shapes, one per direction, with the numbers of the eager path."""
from typing import Optional, Tuple

import torch

from . import _native
from ._custom_ops_norm_blockwise import _HP_DTYPES, _check_operands, _data_shape, _records, _scales_shape, _untraced

_e4m3 = torch.float8_e4m3fn


def _empty(like: torch.Tensor, shape, dtype: Optional[torch.dtype] = None) -> torch.Tensor:
    return torch.empty(shape, dtype=dtype or like.dtype, device=like.device)


# What a trace holds: one operator with its history, the same with gradients and without, that can be saved (an autograd function cannot).
_traced = torch.library.Library("f8mi", "FRAGMENT")
_traced.define("rms_norm(Tensor x2, Tensor? weight, float eps) -> Tensor")
_traced.define("rms_norm_add(Tensor x2, Tensor? weight, Tensor residual2, float eps) -> (Tensor, Tensor)")
_traced.define("dropout(Tensor x, Tensor? residual, Tensor seed, float p) -> Tensor")
_traced.define("low_rank_adapters(Tensor x2, Tensor a, Tensor b, Tensor table, Tensor rows, int count, Tensor? y2, Tensor? scale, float factor) -> Tensor")


# ---- RMS norm


@torch.library.custom_op("f8mi::rms_norm_fwd", mutates_args=())
def rms_norm_fwd(x2: torch.Tensor, weight: Optional[torch.Tensor], residual2: Optional[torch.Tensor], eps: float) -> Tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
    """(y, x + residual (empty without one), rstd of each row)"""
    _check_operands("rms_norm", x2, ("weight", weight, x2.shape[1:], (x2.dtype, torch.float32)), ("residual", residual2, x2.shape, (x2.dtype,)))
    y, total, rstd = _native.rms_norm(x2, weight, residual2, eps)
    return y, _empty(x2, 0) if total is None else total, rstd


@rms_norm_fwd.register_fake
def _(x2, weight, residual2, eps):
    return _empty(x2, x2.shape), _empty(x2, 0 if residual2 is None else x2.shape), _empty(x2, x2.shape[0], torch.float32)


@torch.library.custom_op("f8mi::rms_norm_bwd", mutates_args=())
def rms_norm_bwd(dy2: torch.Tensor, s2: torch.Tensor, ds2: Optional[torch.Tensor], weight: Optional[torch.Tensor], rstd: torch.Tensor, need_dx: bool, need_dw: bool) -> Tuple[
        torch.Tensor, torch.Tensor]:
    """(dx, dweight); an unneeded gradient is empty."""
    _check_operands("rms_norm, backward", s2, ("the gradient", dy2, s2.shape, (s2.dtype,)), ("the sum's gradient", ds2, s2.shape, (s2.dtype,)),
                    ("weight", weight, s2.shape[1:], (s2.dtype, torch.float32)), ("rstd", rstd, s2.shape[:1], (torch.float32,)))
    dx, dw = _native.rms_norm_backward(dy2, s2, ds2, weight, rstd.contiguous(), need_dx, need_dw)
    return _empty(s2, 0) if dx is None else dx, _empty(s2, 0, s2.dtype if weight is None else weight.dtype) if dw is None else dw


@rms_norm_bwd.register_fake
def _(dy2, s2, ds2, weight, rstd, need_dx, need_dw):
    return _empty(s2, s2.shape if need_dx else 0), _empty(s2, s2.shape[1] if need_dw else 0, s2.dtype if weight is None else weight.dtype)


class _RmsNormFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x2, weight, residual2, eps):
        y, total, rstd = rms_norm_fwd(x2, weight, residual2, eps)
        ctx.has_weight, ctx.has_residual = weight is not None, residual2 is not None
        ctx.save_for_backward(total if ctx.has_residual else x2, rstd, *([weight] if ctx.has_weight else []))
        return (y, total) if ctx.has_residual else y

    @staticmethod
    def backward(ctx, gy, *gs):
        s2, rstd, *weight = ctx.saved_tensors
        need_dx, need_dw = ctx.needs_input_grad[0] or ctx.needs_input_grad[2], ctx.needs_input_grad[1]
        dx, dw = rms_norm_bwd(gy, s2, gs[0] if ctx.has_residual else None, weight[0] if ctx.has_weight else None, rstd, need_dx, need_dw)
        return dx if ctx.needs_input_grad[0] else None, dw if need_dw else None, dx if ctx.needs_input_grad[2] else None, None


def _rms_norm(x2, weight, residual2, eps):
    if _records(x2, weight, residual2):
        return _RmsNormFn.apply(x2, weight, residual2, eps)
    y, total, _ = rms_norm_fwd(x2, weight, residual2, eps)
    return y if residual2 is None else (y, total)


@torch.library.impl(_traced, "rms_norm", "CompositeImplicitAutograd")
def _traced_rms_norm(x2, weight, eps):
    with _untraced():
        y = _native.model_ops().rms_norm(x2, x2.shape[1], weight, eps, None)
        return _rms_norm(x2, weight, None, eps) if y is None else y


@torch.library.impl(_traced, "rms_norm_add", "CompositeImplicitAutograd")
def _traced_rms_norm_add(x2, weight, residual2, eps):
    with _untraced():
        out = _native.model_ops().rms_norm(x2, x2.shape[1], weight, eps, residual2)
        return _rms_norm(x2, weight, residual2, eps) if out is None else out


def rms_norm(x: torch.Tensor, weight: Optional[torch.Tensor], residual: Optional[torch.Tensor], cols: int, eps: float):
    x2, weight = x.reshape(-1, cols), None if weight is None else weight.reshape(-1)
    residual2 = None if residual is None else residual.reshape(-1, cols)
    if not torch.jit.is_tracing():
        out = _rms_norm(x2, weight, residual2, eps)
    else:
        out = torch.ops.f8mi.rms_norm(x2, weight, eps) if residual is None else torch.ops.f8mi.rms_norm_add(x2, weight, residual2, eps)
    return out.reshape(x.shape) if residual is None else tuple(t.reshape(x.shape) for t in out)


@torch.library.custom_op("f8mi::rms_norm_blockwise", mutates_args=())
def rms_norm_blockwise(x2: torch.Tensor, weight: Optional[torch.Tensor], residual2: Optional[torch.Tensor], eps: float) -> Tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
    """(data, scales, x + residual (empty without one))"""
    _check_operands("rms_norm_blockwise", x2, ("weight", weight, x2.shape[1:], (x2.dtype, torch.float32)), ("residual", residual2, x2.shape, (x2.dtype,)))
    out, total = _native.rms_norm_block(x2, weight, residual2, eps)
    return out.data, out.scales, _empty(x2, 0) if total is None else total


@rms_norm_blockwise.register_fake
def _(x2, weight, residual2, eps):
    rows, k = x2.shape
    return _empty(x2, _data_shape(rows, k), _e4m3), _empty(x2, _scales_shape(rows, k), torch.uint8), _empty(x2, 0 if residual2 is None else x2.shape)


@torch.library.custom_op("f8mi::blockwise_inference_linear_cast", mutates_args=())
def blockwise_inference_linear_cast(x_data: torch.Tensor, x_scales: torch.Tensor, data: torch.Tensor, scales: torch.Tensor, k: int, dtype: torch.dtype,
                                    bias: Optional[torch.Tensor]) -> torch.Tensor:
    m, n = x_data.shape[1], data.shape[1]
    for what, t, s, rows in (("activations", x_data, x_scales, m), ("a weight", data, scales, n)):
        if t.dtype is not _e4m3 or t.shape != _data_shape(rows, k) or s.dtype is not torch.uint8 or s.shape != _scales_shape(rows, k) or not (
                t.device == s.device == x_data.device and t.is_contiguous() and s.is_contiguous()):
            raise _native.Float8NativeError(f"blockwise_inference_linear_cast: {what} {tuple(t.shape)} ({t.dtype}) on {t.device} with scales {tuple(s.shape)} ({s.dtype}) on {s.device} for {k} in_features")
    if m == 0:
        return _empty(data, (0, n), dtype)
    return _native.block_gemm(_native.Blocks(x_data, x_scales, m, k), _native.Blocks(data, scales, n, k), dtype, None if bias is None else bias.to(dtype).contiguous())


@blockwise_inference_linear_cast.register_fake
def _(x_data, x_scales, data, scales, k, dtype, bias):
    return _empty(data, (x_data.shape[1], data.shape[1]), dtype)


# ---- dropout


@torch.library.custom_op("f8mi::dropout_masked", mutates_args=())
def dropout_masked(x: torch.Tensor, residual: Optional[torch.Tensor], seed: torch.Tensor, p: float) -> torch.Tensor:
    """residual + x / (1 - p) where kept"""
    if seed.dtype is not torch.int64 or seed.numel() != 1 or seed.device != x.device or (residual is not None and (residual.shape, residual.dtype, residual.device) != (x.shape, x.dtype, x.device)):
        raise _native.Float8NativeError(f"dropout: a seed {tuple(seed.shape)} ({seed.dtype}) on {seed.device}" + (
            "" if residual is None else f" and a residual {tuple(residual.shape)} ({residual.dtype}) on {residual.device}") + f" for x {tuple(x.shape)} ({x.dtype}) on {x.device}")
    return _native.dropout(x, residual, seed, p)


@dropout_masked.register_fake
def _(x, residual, seed, p):
    return _empty(x, x.shape)


class _DropoutFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, residual, seed, p):
        ctx.save_for_backward(seed)
        ctx.p = p
        return dropout_masked(x, residual, seed, p)

    @staticmethod
    def backward(ctx, g):
        (seed,) = ctx.saved_tensors
        return dropout_masked(g, None, seed, ctx.p) if ctx.needs_input_grad[0] else None, g if ctx.needs_input_grad[1] else None, None, None


def _dropout(x, residual, seed, p):
    return _DropoutFn.apply(x, residual, seed, p) if _records(x, residual) else dropout_masked(x, residual, seed, p)


@torch.library.impl(_traced, "dropout", "CompositeImplicitAutograd")
def _traced_dropout(x, residual, seed, p):
    with _untraced():
        out = _native.model_ops().dropout(x, p, seed, residual)
        return _dropout(x, residual, seed, p) if out is None else out


def dropout(x: torch.Tensor, residual: Optional[torch.Tensor], seed: torch.Tensor, p: float) -> torch.Tensor:
    return (torch.ops.f8mi.dropout if torch.jit.is_tracing() else _dropout)(x, residual, seed, p)


# ---- low-rank adapters


@torch.library.custom_op("f8mi::adapter_rows", mutates_args=())
def adapter_rows(ids: torch.Tensor, count: int) -> torch.Tensor:
    if ids.dtype not in (torch.int64, torch.int32):
        raise _native.Float8NativeError(f"adapter_rows: ids of {ids.dtype}; int64 or int32 is needed")
    return _native.adapter_rows(ids, count)


@adapter_rows.register_fake
def _(ids, count):
    return _empty(ids, adapter_rows_words(ids.numel(), count), torch.int32)


def adapter_rows_words(m: int, count: int) -> int:
    """f8mi_adapter_rows_words, also of sizes that a compiler knows as symbols only."""
    up4 = lambda v: (v + 3) // 4 * 4
    groups, chunk = count + 1, 64
    while chunk < 512 and chunk * 32 < m:
        chunk *= 2
    tiles = sum(m // height + (groups if groups < m else m) for height in (16, 64, chunk))
    return up4(groups) + up4(groups + 1) + up4(m) + 4 * tiles


def _check_adapters(what: str, rows2: torch.Tensor, a: torch.Tensor, b: torch.Tensor, table: torch.Tensor, rows: Optional[int], count: Optional[int], scale: Optional[torch.Tensor],
                    *operands) -> None:
    """``rows`` and ``count``: what the table was made for.  Its length alone does not say so (tables of 5 and of 8 rows are equally long), and the rows that it lists are read and written."""
    if a.dim() != 3 or b.dim() != 3 or a.dtype not in _HP_DTYPES or a.dtype is not b.dtype or a.device != rows2.device or b.device != rows2.device or (a.shape[0], a.shape[1]) != (b.shape[0], b.shape[2]):
        raise _native.Float8NativeError(f"{what}: a {tuple(a.shape)} ({a.dtype}) on {a.device} and b {tuple(b.shape)} ({b.dtype}) on {b.device} for rows on {rows2.device}")
    if (rows2.shape[0] if rows is None else rows, a.shape[0] if count is None else count) != (rows2.shape[0], a.shape[0]):
        raise _native.Float8NativeError(f"{what}: a table of {rows} rows and {count} adapters for {rows2.shape[0]} rows and {a.shape[0]} adapters")
    _check_operands(what, rows2, ("a batch's table", table, (adapter_rows_words(rows2.shape[0], a.shape[0]),), (torch.int32,)), ("scale", scale, a.shape[:1], (torch.float32,)), *operands)


@torch.library.custom_op("f8mi::adapters_fwd", mutates_args=())
def adapters_fwd(x2: torch.Tensor, a: torch.Tensor, b: torch.Tensor, table: torch.Tensor, y2: Optional[torch.Tensor], scale: Optional[torch.Tensor], factor: float, need_h: bool,
                 rows: Optional[int] = None, count: Optional[int] = None) -> Tuple[torch.Tensor, torch.Tensor]:
    """(out, h (empty unless needed)); ``rows`` and ``count``: of the table"""
    _check_adapters("low_rank_adapters", x2, a, b, table, rows, count, scale, ("x", x2, (x2.shape[0], a.shape[-1]), (x2.dtype,)), ("y", y2, (x2.shape[0], b.shape[1]), (x2.dtype,)))
    out, h = _native.adapters(x2, a, b, table.contiguous(), y2, None if scale is None else scale.contiguous(), factor, need_h)
    return out, _empty(x2, 0, torch.float32) if h is None else h


@adapters_fwd.register_fake
def _(x2, a, b, table, y2, scale, factor, need_h, rows=None, count=None):
    return _empty(x2, (x2.shape[0], b.shape[1])), _empty(x2, (x2.shape[0], (a.shape[1] + 15) // 16 * 16) if need_h else 0, torch.float32)


@torch.library.custom_op("f8mi::adapters_bwd", mutates_args=())
def adapters_bwd(dout2: torch.Tensor, x2: Optional[torch.Tensor], a: torch.Tensor, b: torch.Tensor, table: torch.Tensor, scale: Optional[torch.Tensor], factor: float, h: torch.Tensor, need_dx: bool,
                 need_da: bool, need_db: bool, rows: Optional[int] = None, count: Optional[int] = None) -> Tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
    """(dx, da, db); an unneeded gradient is empty."""
    if dout2.shape[0] == 0:
        return _empty(dout2, (0, a.shape[2]) if need_dx else 0), torch.zeros_like(a) if need_da else _empty(a, 0), torch.zeros_like(b) if need_db else _empty(b, 0)
    m, rank = dout2.shape[0], a.shape[1]
    _check_adapters("low_rank_adapters, backward", dout2, a, b, table, rows, count, scale, ("the gradient", dout2, (m, b.shape[1]), (dout2.dtype,)),
                    ("x", x2 if need_da else None, (m, a.shape[-1]), (dout2.dtype,)), ("h", h if need_db else None, (m, (rank + 15) // 16 * 16), (torch.float32,)))
    grads = _native.adapters_backward(dout2, x2, a, b, table.contiguous(), None if scale is None else scale.contiguous(), factor, h.contiguous(), need_dx, need_da, need_db)
    return tuple(_empty(t, 0) if g is None else g for g, t in zip(grads, (dout2, a, b)))


@adapters_bwd.register_fake
def _(dout2, x2, a, b, table, scale, factor, h, need_dx, need_da, need_db, rows=None, count=None):
    return _empty(dout2, (dout2.shape[0], a.shape[2]) if need_dx else 0), _empty(a, a.shape if need_da else 0), _empty(b, b.shape if need_db else 0)


class _AdaptersFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x2, a, b, table, rows, count, y2, scale, factor):
        out, h = adapters_fwd(x2, a, b, table, y2, scale, factor, ctx.needs_input_grad[2], rows, count)
        ctx.rows, ctx.count = rows, count
        ctx.factor, ctx.has_scale, ctx.has_x = factor, scale is not None, ctx.needs_input_grad[1]
        ctx.save_for_backward(a, b, table, h, *([x2] if ctx.has_x else []), *([scale] if ctx.has_scale else []))
        return out

    @staticmethod
    def backward(ctx, g):
        a, b, table, h, *rest = ctx.saved_tensors
        x2, scale = rest[0] if ctx.has_x else None, rest[-1] if ctx.has_scale else None
        needs = ctx.needs_input_grad[:3]
        grads = adapters_bwd(g, x2, a, b, table, scale, ctx.factor, h, *needs, ctx.rows, ctx.count) if any(needs) else (None,) * 3
        return tuple(d if need else None for d, need in zip(grads, needs)) + (None, None, None, g if ctx.needs_input_grad[6] else None, None, None)


def _low_rank_adapters(x2, a, b, table, rows, count, y2, scale, factor):
    if _records(x2, a, b, y2):
        return _AdaptersFn.apply(x2, a, b, table, rows, count, y2, scale, factor)
    return adapters_fwd(x2, a, b, table, y2, scale, factor, False, rows, count)[0]


@torch.library.impl(_traced, "low_rank_adapters", "CompositeImplicitAutograd")
def _traced_low_rank_adapters(x2, a, b, table, rows, count, y2, scale, factor):
    with _untraced():
        rows = int(rows)
        out = _native.model_ops().low_rank_adapters(x2, a, b, table, rows, count, y2, scale, factor)
        return _low_rank_adapters(x2, a, b, table, rows, count, y2, scale, factor) if out is None else out


def low_rank_adapters(x: torch.Tensor, a: torch.Tensor, b: torch.Tensor, table: torch.Tensor, rows: int, count: int, y: Optional[torch.Tensor], scale: Optional[torch.Tensor], factor: float) -> torch.Tensor:
    """``rows``, ``count``: of the table.  A trace has the rows as a number on the host: a constant where the table is one, else the rows of the numbers that the table is made of in the trace."""
    call = _low_rank_adapters
    if torch.jit.is_tracing():
        call, rows = torch.ops.f8mi.low_rank_adapters, torch.as_tensor(rows, device="cpu")
    return call(x.reshape(-1, x.shape[-1]), a, b, table, rows, count, None if y is None else y.reshape(-1, y.shape[-1]), scale, factor).reshape(*x.shape[:-1], b.shape[1])
