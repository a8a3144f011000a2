"""Layer norm whose forward and backward passes read and write each tensor once (csrc/f8mi_layer_norm.hip)."""
import math
from typing import Optional, Sequence, Union

import torch
import torch.nn as nn

from . import _custom_ops_norm_blockwise as _compiled
from . import _native

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
    if type(module) is nn.LayerNorm:
        return LayerNorm.from_float(module)
    for name, child in module.named_children():
        if type(child) is nn.LayerNorm:
            setattr(module, name, LayerNorm.from_float(child))
        else:
            convert_layer_norms(child)
    return module
