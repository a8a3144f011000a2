"""Layer norm and RMS norm whose forward and backward passes read and write each tensor once (csrc/f8mi_layer_norm.hip, csrc/f8mi_rms_norm.hip)."""
import math
from typing import Optional, Sequence, Tuple, Union

import torch
import torch.nn as nn

from . import _custom_ops_model as _compiled_model
from . import _custom_ops_norm_blockwise as _compiled
from . import _native
from .float8_blockwise import BlockwiseActivations
from .module_swap import swap_modules

_HP_DTYPES = (torch.bfloat16, torch.float16, torch.float32)


def layer_norm(x: torch.Tensor, normalized_shape: Union[int, Sequence[int]], weight: Optional[torch.Tensor] = None,
               bias: Optional[torch.Tensor] = None, eps: float = 1e-5) -> torch.Tensor:
    """``torch.nn.functional.layer_norm``: ``(x - mean) / sqrt(var + eps) * weight + bias`` over the trailing ``normalized_shape``.

    ``x`` in bfloat16, float16 or float32, the result in its type (also under autocast); weight and bias in that type or in float32, their
    gradients in their own.  Statistics and sums are fp32; the sums of the parameters' gradients have a fixed order."""
    if not torch.compiler.is_compiling():
        y = _native.ops().layer_norm(x, normalized_shape, weight, bias, eps)
        if y is not None:
            return y
        _native.refuse_tangents("layer_norm", x, weight, bias)
    shape = (normalized_shape,) if isinstance(normalized_shape, int) else tuple(normalized_shape)
    _native._require_gpu(x, "x")
    if x.dtype not in _HP_DTYPES:
        raise TypeError(f"layer_norm: x is {x.dtype}; bfloat16, float16 or float32 is needed")
    if not shape or math.prod(shape) == 0 or tuple(x.shape[x.dim() - len(shape):]) != shape or x.dim() < len(shape):
        raise ValueError(f"layer_norm: x of shape {tuple(x.shape)} does not end in normalized_shape {shape}")
    for name, p in (("weight", weight), ("bias", bias)):
        if p is None:
            continue
        _native._require_gpu(p, name)
        if tuple(p.shape) != shape or p.dtype not in _HP_DTYPES:
            raise ValueError(f"layer_norm: {name} of shape {tuple(p.shape)} ({p.dtype}) for normalized_shape {shape}")
    # the kernels take both parameters in x's type or both in fp32
    if any(p is not None and p.dtype not in (x.dtype, torch.float32) for p in (weight, bias)) or (
            weight is not None and bias is not None and weight.dtype != bias.dtype):
        weight, bias = (None if p is None else p.float() for p in (weight, bias))
    if not torch.compiler.is_compiling():
        y = _native.ops().layer_norm(x, shape, weight, bias, float(eps))  # with parameters of the types it takes
        if y is not None:
            return y
    return _compiled.layer_norm(x, weight, bias, math.prod(shape), float(eps))


class LayerNorm(nn.LayerNorm):
    """``nn.LayerNorm`` on this package's kernels."""

    def forward(self, input: torch.Tensor) -> torch.Tensor:
        return layer_norm(input, self.normalized_shape, self.weight, self.bias, self.eps)

    @classmethod
    def from_float(cls, mod: nn.LayerNorm) -> "LayerNorm":
        """A layer sharing ``mod``'s parameters."""
        with torch.device("meta"):
            new_mod = cls(mod.normalized_shape, eps=mod.eps, elementwise_affine=mod.elementwise_affine, bias=mod.bias is not None)
        new_mod.weight, new_mod.bias = mod.weight, mod.bias
        new_mod.train(mod.training)
        return new_mod


def convert_layer_norms(module: nn.Module) -> nn.Module:
    """Swaps every ``nn.LayerNorm`` of ``module`` for a ``LayerNorm`` that shares its parameters; a root-level one is returned converted."""
    return swap_modules(module, nn.LayerNorm, LayerNorm.from_float)


def _rms_arguments(what: str, x, normalized_shape, weight, eps, residual):
    """(normalized_shape as a tuple, the weight in a type that the kernels take, eps), or an exception that says what does not fit."""
    shape = (normalized_shape,) if isinstance(normalized_shape, int) else tuple(normalized_shape)
    _native._require_gpu(x, "x")
    if x.dtype not in _HP_DTYPES:
        raise TypeError(f"{what}: x is {x.dtype}; bfloat16, float16 or float32 is needed")
    if not shape or math.prod(shape) == 0 or tuple(x.shape[x.dim() - len(shape):]) != shape or x.dim() < len(shape):
        raise ValueError(f"{what}: x of shape {tuple(x.shape)} does not end in normalized_shape {shape}")
    if weight is not None:
        _native._require_gpu(weight, "weight")
        if tuple(weight.shape) != shape or weight.dtype not in _HP_DTYPES:
            raise ValueError(f"{what}: weight of shape {tuple(weight.shape)} ({weight.dtype}) for normalized_shape {shape}")
        if weight.dtype not in (x.dtype, torch.float32):
            weight = weight.float()
    if residual is not None:
        _native._require_gpu(residual, "residual")
        if residual.shape != x.shape or residual.dtype != x.dtype:
            raise ValueError(f"{what}: residual of shape {tuple(residual.shape)} ({residual.dtype}) for x of shape {tuple(x.shape)} ({x.dtype})")
    return shape, weight, float(eps)


def rms_norm(x: torch.Tensor, normalized_shape: Union[int, Sequence[int]], weight: Optional[torch.Tensor] = None, eps: Optional[float] = None,
             residual: Optional[torch.Tensor] = None) -> Union[torch.Tensor, Tuple[torch.Tensor, torch.Tensor]]:
    """``torch.nn.functional.rms_norm``: ``x / sqrt(mean(x^2) + eps) * weight`` over the trailing ``normalized_shape`` (eps None: that of float32).

    With a ``residual`` of x's shape and type: ``(the norm of s, s)`` with ``s = x + residual`` rounded to their type, which the next residual addition
    goes on from; the gradient of both comes through both results.

    ``x`` in bfloat16, float16 or float32, the results in its type (also under autocast); the weight in that type or in float32, its gradient in its own.
    Statistics and sums are fp32 (squares whose mean float32 does not hold give zeros); the sums of the weight's gradient have a fixed order."""
    eps = torch.finfo(torch.float32).eps if eps is None else eps
    if not torch.compiler.is_compiling():
        out = _native.model_ops().rms_norm(x, normalized_shape, weight, eps, residual)
        if out is not None:
            return out
        _native.refuse_tangents("rms_norm", x, weight, residual)
    shape, weight, eps = _rms_arguments("rms_norm", x, normalized_shape, weight, eps, residual)
    if not torch.compiler.is_compiling():
        out = _native.model_ops().rms_norm(x, shape, weight, eps, residual)  # with a weight of a type that it takes
        if out is not None:
            return out
    return _compiled_model.rms_norm(x, weight, residual, math.prod(shape), eps)


def rms_norm_blockwise(x: torch.Tensor, normalized_shape: Union[int, Sequence[int]], weight: Optional[torch.Tensor] = None, eps: Optional[float] = None,
                       residual: Optional[torch.Tensor] = None) -> Union[BlockwiseActivations, Tuple[BlockwiseActivations, torch.Tensor]]:
    """``rms_norm`` over the last dimension into ``BlockwiseActivations``: e4m3 with a scale for each 128 values of a row, which any number of
    ``Float8BlockwiseInferenceLinear`` take without a cast of their own.  The normed values are rounded once, to e4m3.  No backward pass."""
    eps = torch.finfo(torch.float32).eps if eps is None else eps
    out = None if torch.compiler.is_compiling() else _native.model_ops().rms_norm_blockwise(x, normalized_shape, weight, eps, residual)
    if out is None:
        if not torch.compiler.is_compiling():
            _native.refuse_tangents("rms_norm_blockwise", x, weight, residual)
        shape, weight, eps = _rms_arguments("rms_norm_blockwise", x, normalized_shape, weight, eps, residual)
        if len(shape) != 1:
            raise ValueError(f"rms_norm_blockwise: blocks lie along the last dimension; normalized_shape {shape} has more")
        if torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in (x, weight, residual)):
            raise RuntimeError("rms_norm_blockwise has no backward pass: call it under torch.no_grad() or torch.inference_mode()")
        flat = lambda t: None if t is None else t.detach().reshape(-1, shape[0])
        out = _compiled_model.rms_norm_blockwise(flat(x), None if weight is None else weight.detach(), flat(residual), eps)
    kept = BlockwiseActivations(out[0], out[1], tuple(x.shape), x.dtype)
    return kept if residual is None else (kept, out[2].reshape(x.shape))


class RMSNorm(nn.RMSNorm):
    """``nn.RMSNorm`` on this package's kernels; a residual may come with the input (``rms_norm``)."""

    def forward(self, input: torch.Tensor, residual: Optional[torch.Tensor] = None):
        return rms_norm(input, self.normalized_shape, self.weight, self.eps, residual)

    def blockwise(self, input: torch.Tensor, residual: Optional[torch.Tensor] = None):
        """The same for served linears with block scales (``rms_norm_blockwise``)."""
        return rms_norm_blockwise(input, self.normalized_shape, self.weight, self.eps, residual)

    @classmethod
    def from_float(cls, mod: nn.RMSNorm) -> "RMSNorm":
        """A layer sharing ``mod``'s weight."""
        with torch.device("meta"):
            new_mod = cls(mod.normalized_shape, eps=mod.eps, elementwise_affine=mod.elementwise_affine)
        new_mod.weight = mod.weight
        new_mod.train(mod.training)
        return new_mod


def convert_rms_norms(module: nn.Module) -> nn.Module:
    """Swaps every ``nn.RMSNorm`` of ``module`` for an ``RMSNorm`` that shares its weight; a root-level one is returned converted."""
    return swap_modules(module, nn.RMSNorm, RMSNorm.from_float)
