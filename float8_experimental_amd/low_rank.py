"""Low-rank adapters beside a projection, a different one for each row of the batch (csrc/f8mi_adapters.hip).

    out_i = y_i + scale_e * B_e (A_e x_i),   e = the adapter of row i

``y`` comes from the projection that all rows share: any of this package's linears, whose weight stays as it is.  ``AdapterRows`` sorts a batch's rows by adapter,
once for all layers; ``low_rank_adapters`` is the operator; ``AdaptedLinear`` a linear with its adapters, ``adapt_linears`` puts one around every linear of
a model and ``select_adapters`` tells all of them whose rows the next batch holds.
"""
import math
from typing import Callable, Optional, Union

import torch
import torch.nn as nn

from . import _custom_ops_model as _compiled
from . import _native
from .float8_blockwise import BlockwiseActivations, Float8BlockwiseInferenceLinear
from .residual_dropout import dropout as _dropout

_HP_DTYPES = (torch.bfloat16, torch.float16, torch.float32)
_INTEGERS = (torch.int64, torch.int32, torch.int16, torch.int8, torch.uint8)
MAX_RANK, MAX_COUNT, MAX_ROWS = 256, 32768, 1 << 24  # F8MI_ADAPTER_MAX_*


class AdapterRows:
    """The rows of a batch by adapter: ``adapters`` has one whole number for each row (``x.numel() / k`` of them, in their order), that of its adapter among ``count``; any other
    number, -1 for instance, means none.  Made once for a batch and used by all its layers, on any stream that waits for the one it is made on; it keeps what the numbers were then.

    A captured graph reads the table that it was captured with: it has to outlive the graph, or is made inside the capture, from numbers that are written between replays."""

    def __init__(self, adapters: torch.Tensor, count: int):
        _native._require_gpu(adapters, "adapters")
        if adapters.dtype not in _INTEGERS:
            raise TypeError(f"AdapterRows: adapters are {adapters.dtype}; whole numbers are needed")
        if not 1 <= count <= MAX_COUNT:
            raise ValueError(f"AdapterRows: {count} adapters; 1 to {MAX_COUNT} are possible")
        if adapters.numel() > MAX_ROWS:
            raise ValueError(f"AdapterRows: {adapters.numel()} rows; at most {MAX_ROWS} are possible")
        if adapters.dtype not in (torch.int64, torch.int32):
            adapters = adapters.long()
        self.count, self.rows = int(count), adapters.numel()
        self.table = _compiled.adapter_rows(adapters.detach(), self.count)

    def __repr__(self):
        return f"AdapterRows({self.rows} rows, {self.count} adapters, {self.table.device})"


def low_rank_adapters(x: torch.Tensor, a: torch.Tensor, b: torch.Tensor, adapters: Union[AdapterRows, torch.Tensor], y: Optional[torch.Tensor] = None,
                      scale: Union[float, torch.Tensor] = 1.0) -> torch.Tensor:
    """``y_i + scale_e * b[e] @ (a[e] @ x_i)`` for each row i of ``x`` with its adapter e; y_i for a row without one.

    ``x`` [..., k], ``a`` [count, rank, k], ``b`` [count, n, rank] with a rank of at most 256, ``y`` [..., n] of x's type (None: zeros), ``scale`` a number or one for each adapter
    (no gradient).  ``adapters``: an ``AdapterRows`` of this batch, or the numbers themselves, which are then sorted in this call.

    x in bfloat16, float16 or float32; a and b may have another of these types, they are rounded to x's for the products and their gradients have their own, rounded once; a row's
    ``a[e] @ x_i`` is kept in 32 bits, to 2^-16 of itself in the second product of 16-bit types (float16: or to 2^-39 of the row's largest).  Sums are fp32, in a fixed order; an
    infinity in 16-bit x, a, b or the gradient of the result may come out as NaN.  Under autocast x and y take the autocast type first."""
    if torch.is_autocast_enabled():
        dtype = torch.get_autocast_dtype("cuda")
        x, y = x.to(dtype), None if y is None else y.to(dtype)
    if not isinstance(adapters, AdapterRows):
        adapters = AdapterRows(adapters, a.shape[0])
    factor, per_adapter = (1.0, scale) if isinstance(scale, torch.Tensor) else (scale, None)
    if not torch.compiler.is_compiling():
        out = _native.model_ops().low_rank_adapters(x, a, b, adapters.table, adapters.rows, adapters.count, y, per_adapter, factor)
        if out is not None:
            return out
        _native.refuse_tangents("low_rank_adapters", x, a, b, y)
    for name, t in (("x", x), ("a", a), ("b", b), ("y", y), ("scale", per_adapter)):
        if t is None:
            continue
        _native._require_gpu(t, name)
        if t.dtype not in _HP_DTYPES:
            raise TypeError(f"low_rank_adapters: {name} is {t.dtype}; bfloat16, float16 or float32 is needed")
    if a.dim() != 3 or b.dim() != 3 or a.shape[0] != b.shape[0] or a.shape[1] != b.shape[2] or 0 in a.shape or 0 in b.shape:
        raise ValueError(f"low_rank_adapters: a of shape {tuple(a.shape)} and b of shape {tuple(b.shape)} are not [count, rank, k] and [count, n, rank]")
    (count, rank, k), n = a.shape, b.shape[1]
    if rank > MAX_RANK:
        raise ValueError(f"low_rank_adapters: rank {rank}; at most {MAX_RANK} is possible")
    if x.dim() == 0 or x.shape[-1] != k:
        raise ValueError(f"low_rank_adapters: x of shape {tuple(x.shape)} does not end in the {k} features of a")
    if y is not None and (y.shape != (*x.shape[:-1], n) or y.dtype != x.dtype):
        raise ValueError(f"low_rank_adapters: y of shape {tuple(y.shape)} ({y.dtype}) for x of shape {tuple(x.shape)} ({x.dtype}) and {n} features of b")
    if adapters.count != count or adapters.rows != x.numel() // k:
        raise ValueError(f"low_rank_adapters: {adapters} for {x.numel() // k} rows and {count} adapters")
    _native._require_gpu(adapters.table, "adapters")
    if per_adapter is not None:
        if per_adapter.shape != (count,):
            raise ValueError(f"low_rank_adapters: scale of shape {tuple(per_adapter.shape)} for {count} adapters")
        if torch.is_grad_enabled() and per_adapter.requires_grad:
            raise NotImplementedError("low_rank_adapters has no gradient of scale")
        per_adapter = per_adapter.float().contiguous()
    if a.dtype != b.dtype:
        a, b = a.float(), b.float()
    if not torch.compiler.is_compiling():
        out = _native.model_ops().low_rank_adapters(x, a, b, adapters.table, adapters.rows, adapters.count, y, per_adapter, factor)  # with adapters and a scale of types that it takes
        if out is not None:
            return out
    return _compiled.low_rank_adapters(x, a, b, adapters.table, adapters.rows, adapters.count, y, per_adapter, float(factor))


class AdaptedLinear(nn.Module):
    """A linear of any kind that this package has, with ``count`` low-rank adapters beside it.

    ``linear`` (its parameters no longer ask for gradients), ``adapter_a`` [count, rank, in_features] as ``nn.Linear`` initialises a weight and ``adapter_b`` [count,
    out_features, rank] of zeros, in ``dtype`` (None: that of the linear's weight, bfloat16 where that is float8).  ``alpha / rank`` (alpha None: rank) scales
    what they add, ``dropout`` of their input is dropped in training.  ``rows`` says which adapter each row of the batch has (``select_adapters``); None: no row has one.

    It is called as a linear is, and has no ``weight`` and no ``bias``: who multiplied by those would leave the adapters out."""

    def __init__(self, linear: nn.Module, count: int, rank: int, alpha: Optional[float] = None, dropout: float = 0.0, dtype: Optional[torch.dtype] = None):
        super().__init__()
        if not 1 <= rank <= MAX_RANK or not 1 <= count <= MAX_COUNT:
            raise ValueError(f"AdaptedLinear: {count} adapters of rank {rank}; 1 to {MAX_COUNT} of rank 1 to {MAX_RANK} are possible")
        if not 0.0 <= dropout <= 1.0:
            raise ValueError(f"AdaptedLinear: dropout={dropout} is not a probability")
        weight = linear.weight_data if isinstance(linear, Float8BlockwiseInferenceLinear) else linear.weight
        if dtype is None:
            dtype = weight.dtype if weight.dtype in _HP_DTYPES and not isinstance(linear, Float8BlockwiseInferenceLinear) else torch.bfloat16
        self.linear = linear.requires_grad_(False)
        self.in_features, self.out_features = linear.in_features, linear.out_features
        self.count, self.rank, self.dropout = count, rank, dropout
        self.scaling = (rank if alpha is None else alpha) / rank
        self.adapter_a = nn.Parameter(torch.empty(count, rank, self.in_features, dtype=dtype, device=weight.device))
        self.adapter_b = nn.Parameter(torch.empty(count, self.out_features, rank, dtype=dtype, device=weight.device))
        self.rows: Optional[AdapterRows] = None
        self.reset_adapters()

    def reset_adapters(self) -> None:
        with torch.no_grad():
            bound = 1 / math.sqrt(self.in_features)
            self.adapter_a.uniform_(-bound, bound)
            self.adapter_b.zero_()

    def forward(self, input: torch.Tensor) -> torch.Tensor:
        y = self.linear(input)
        if self.rows is None:
            return y
        if isinstance(input, BlockwiseActivations):
            raise TypeError("AdaptedLinear: the adapters need the activations in bfloat16, float16 or float32, not BlockwiseActivations")
        x = _dropout(input, self.dropout) if self.training and self.dropout > 0.0 else input
        return low_rank_adapters(x, self.adapter_a, self.adapter_b, self.rows, y, self.scaling)

    def extra_repr(self) -> str:
        return f"count={self.count}, rank={self.rank}, scaling={self.scaling}, dropout={self.dropout}"


# Linears whose module reads their weight, always or in evaluation, instead of calling them: what stands around them there is not asked
_READ_BY_THEIR_MODULE = ((nn.MultiheadAttention, ("out_proj",)), (nn.TransformerEncoderLayer, ("linear1", "linear2")))


def adapt_linears(module: nn.Module, count: int, rank: int, *, alpha: Optional[float] = None, dropout: float = 0.0, dtype: Optional[torch.dtype] = None,
                  module_filter_fn: Optional[Callable[[nn.Module, str], bool]] = None) -> nn.Module:
    """Puts an ``AdaptedLinear`` around every linear of ``module`` that passes ``module_filter_fn(linear, fqn)``; no parameter of ``module`` but its adapters asks for
    gradients any more.  A root-level linear is returned adapted; linears that have adapters already keep those, and one that is held under several names or by several modules has one set of them.

    ``nn.MultiheadAttention`` does not call its ``out_proj`` and ``nn.TransformerEncoderLayer`` not always its ``linear1`` and ``linear2``: they take the weights and multiply by themselves.  These
    linears have no adapters, and a filter that asks for one of them raises."""
    def wanted(m: nn.Module, fqn: str, parent: Optional[nn.Module] = None, name: str = "") -> bool:
        if not isinstance(m, (nn.Linear, Float8BlockwiseInferenceLinear)) or not (module_filter_fn is None or module_filter_fn(m, fqn)):
            return False
        read = any(isinstance(parent, kind) and name in names for kind, names in _READ_BY_THEIR_MODULE)
        if read and module_filter_fn is not None:
            raise ValueError(f"adapt_linears: {type(parent).__name__} reads the weight of {fqn!r} instead of calling it, so that adapters around it would do nothing; module_filter_fn has to leave it out")
        return not read

    found = []  # (module, name, linear): nothing is changed before all of them are known

    def visit(mod: nn.Module, prefix: str) -> None:
        for name, child in mod._modules.items():  # (named_children() has each module under one of its names)
            fqn = f"{prefix}.{name}" if prefix else name
            if child is None or isinstance(child, AdaptedLinear):
                continue
            if wanted(child, fqn, mod, name):
                found.append((mod, name, child))
            else:
                visit(child, fqn)

    root = wanted(module, "")
    if not root and not isinstance(module, AdaptedLinear):
        visit(module, "")
    kept = {id(p) for m in module.modules() if isinstance(m, AdaptedLinear) for p in (m.adapter_a, m.adapter_b)}
    for p in module.parameters():
        if id(p) not in kept:
            p.requires_grad_(False)
    around = lambda m: AdaptedLinear(m, count, rank, alpha, dropout, dtype).train(m.training)
    if root:
        return around(module)
    made = {}
    for mod, name, linear in found:
        if linear not in made:
            made[linear] = around(linear)
        setattr(mod, name, made[linear])
    return module


def select_adapters(module: nn.Module, adapters: Union[AdapterRows, torch.Tensor, None]) -> Optional[AdapterRows]:
    """The adapter of each row of the next batches, for every ``AdaptedLinear`` of ``module``: an ``AdapterRows``, the numbers themselves, or None for none.  Returns the ``AdapterRows``."""
    layers = [m for m in module.modules() if isinstance(m, AdaptedLinear)]
    if adapters is not None and not isinstance(adapters, AdapterRows):
        if not layers:
            raise ValueError("select_adapters: the module has no AdaptedLinear")
        adapters = AdapterRows(adapters, layers[0].count)
    if adapters is not None and any(layer.count != adapters.count for layer in layers):
        raise ValueError(f"select_adapters: {adapters} for layers of {sorted({layer.count for layer in layers})} adapters")
    for layer in layers:
        layer.rows = adapters
    return adapters
