"""Linear layers whose operands are e4m3 with a power-of-two scale for each block of 128 values.

Finer than one scale for the tensor: activations and gradients of outputs have a scale for each 128 neighbouring values of a row along
the contraction, weights one for each 128 x 128, so that one outlier costs its block precision and not the whole tensor.  A block is
kept as e4m3 of value / 2^S with the smallest S for which nothing saturates; the exponents go to the matrix instruction, which applies them
itself.  No amax pass, no history and no state: the cast finds the scales while it has the block in registers, and a layer reads
each tensor once.

    y = q(x) q(w)^T + bias,   dx = q(dy) q(w),   dw = q'(dy)^T q'(x)

with q' in blocks along the tokens, which the backward's contraction runs over.  The matrix cores add products: the eight of neighbouring k
are cut to multiples of 2^-13 of the largest of them, the groups of eight are added in fp32 (about 1.3e-5 of a result's size altogether, as in
``torch._scaled_mm``), and the result is rounded once.

``convert_to_float8_training`` with ``ScalingType.BLOCKWISE`` for all three tensors swaps ``nn.Linear`` for ``Float8BlockwiseLinear``,
``quantize_to_float8`` with ``ActivationCasting.BLOCKWISE`` for ``Float8BlockwiseInferenceLinear``; ``blockwise_linear`` is the function
behind the former.
"""
from typing import NamedTuple, Optional, Tuple, Union

import torch
import torch.nn as nn

from . import _custom_ops_model as _compiled_model
from . import _custom_ops_norm_blockwise as _compiled
from . import _native

_HP_DTYPES = (torch.bfloat16, torch.float16, torch.float32)


def _checked(x: torch.Tensor, n: int, k: int, bias: Optional[torch.Tensor], what: str) -> None:
    _native._require_gpu(x, "x")
    if x.dtype not in _HP_DTYPES:
        raise TypeError(f"{what}: x is {x.dtype}; bfloat16, float16 or float32 is needed")
    if x.dim() == 0 or x.shape[-1] != k:
        raise ValueError(f"{what}: x of shape {tuple(x.shape)} does not end in the {k} in_features of the weight")
    if n == 0 or k == 0:
        raise ValueError(f"{what}: a weight of shape {(n, k)} has no values")
    if bias is not None:
        _native._require_gpu(bias, "bias")
        if bias.shape != (n,) or bias.dtype not in _HP_DTYPES:
            raise ValueError(f"{what}: bias of shape {tuple(bias.shape)} ({bias.dtype}) for {n} out_features")


def blockwise_linear(x: torch.Tensor, weight: torch.Tensor, bias: Optional[torch.Tensor] = None) -> torch.Tensor:
    """``x @ weight.t() + bias`` with every product of forward and backward on block-scaled e4m3 operands.

    ``x`` [..., k] and ``weight`` [n, k] in bfloat16, float16 or float32 (the weight may have another type than x), ``bias`` [n], which is rounded to x's
    type before it is added; the result and the gradient of x have x's type, those of weight and bias the parameters' own, to which their fp32 sums are
    rounded once.  Under autocast x takes the autocast type first."""
    if torch.is_autocast_enabled():
        x = x.to(torch.get_autocast_dtype("cuda"))
    if not torch.compiler.is_compiling():
        y = _native.ops().blockwise_linear(x, weight, bias)
        if y is not None:
            return y
        _native.refuse_tangents("blockwise_linear", x, weight, bias)
    if weight.dim() != 2:
        raise ValueError(f"blockwise_linear: weight of shape {tuple(weight.shape)} is no matrix")
    n, k = weight.shape
    _checked(x, n, k, bias, "blockwise_linear")
    _native._require_gpu(weight, "weight")
    if weight.dtype not in _HP_DTYPES:
        raise TypeError(f"blockwise_linear: weight is {weight.dtype}; bfloat16, float16 or float32 is needed")
    return _compiled.blockwise_linear(x, weight, bias)


class Float8BlockwiseLinear(nn.Linear):
    """``nn.Linear`` on block-scaled float8 operands.  Construct through ``from_float`` / ``convert_to_float8_training``."""

    def forward(self, input: torch.Tensor) -> torch.Tensor:
        return blockwise_linear(input, self.weight, self.bias)

    def extra_repr(self):
        return f'{super().extra_repr()}, scaling="i:blk,w:blk,go:blk"'

    @classmethod
    def from_float(cls, mod: nn.Linear, config=None) -> "Float8BlockwiseLinear":
        """A layer sharing ``mod``'s parameters."""
        if config is not None and config.emulate:
            raise NotImplementedError("blockwise scaling has no emulated products")
        if config is not None and config.enable_fsdp_float8_all_gather:
            raise NotImplementedError("blockwise scaling has no weight scales to compute ahead of the forward pass")
        with torch.device("meta"):
            new_mod = cls(mod.in_features, mod.out_features, bias=False)
        new_mod.weight, new_mod.bias = mod.weight, mod.bias
        new_mod.train(mod.training)
        return new_mod


class BlockwiseActivations(NamedTuple):
    """Activations [..., k] as ``Float8BlockwiseInferenceLinear`` multiplies them: e4m3 with a scale for each 128 values of a row, in the placement of its weight.  What
    ``rms_norm_blockwise`` gives."""

    data: torch.Tensor  # [padded k / 64, rows, 64]
    scales: torch.Tensor
    shape: Tuple[int, ...]
    dtype: torch.dtype  # of the activations before, and of a linear's result

    def dequantized(self) -> torch.Tensor:
        """The values that the activations stand for, in fp32."""
        return _native.Blocks(self.data, self.scales, self.data.shape[1], self.shape[-1]).dequant().float().reshape(self.shape)


class Float8BlockwiseInferenceLinear(nn.Module):
    """A linear whose weight is kept as block-scaled e4m3, one byte a value and one for each 128 x 128 of them (repeated for its rows); the activations
    are cast per call.  Construct through ``from_float`` / ``quantize_to_float8``.

    ``weight_data`` [padded in_features / 64, out_features, 64] and ``weight_scales`` are buffers in the placement that the products read
    (``f8mi_block_gemm`` of include/f8mi.h); ``dequantized_weight`` gives the values back."""

    def __init__(self, in_features: int, out_features: int, bias: Optional[torch.Tensor] = None, device=None):
        super().__init__()
        self.in_features, self.out_features = in_features, out_features
        blocks = _native._blocks_alloc(out_features, in_features, device)
        self.register_buffer("weight_data", blocks.data)
        self.register_buffer("weight_scales", blocks.scales)
        self.bias = None if bias is None else nn.Parameter(bias, requires_grad=False)

    def _apply(self, fn, recurse=True):
        # to(dtype), half() and the like convert buffers of floating types, e4m3 among them, and type() all of them: the weight moves, and stays what it is
        kept = {name: self._buffers[name] for name in ("weight_data", "weight_scales")}
        super()._apply(fn, recurse)
        for name, t in kept.items():
            if self._buffers[name].dtype is not t.dtype:
                self._buffers[name] = t.to(self._buffers[name].device)
        return self

    def forward(self, input: Union[torch.Tensor, BlockwiseActivations]) -> torch.Tensor:
        if isinstance(input, BlockwiseActivations):
            return self._forward_cast(input)
        if torch.is_autocast_enabled():
            input = input.to(torch.get_autocast_dtype("cuda"))
        if not torch.compiler.is_compiling():
            y = _native.ops().blockwise_inference_linear(input, self.weight_data, self.weight_scales, self.out_features, self.in_features, self.bias)
            if y is not None:
                return y
            _native.refuse_tangents("Float8BlockwiseInferenceLinear", input, self.bias)
        _checked(input, self.out_features, self.in_features, self.bias, "Float8BlockwiseInferenceLinear")
        if torch.is_grad_enabled() and input.requires_grad:
            raise RuntimeError("Float8BlockwiseInferenceLinear has no backward pass: call it under torch.no_grad() or torch.inference_mode()")
        return _compiled.blockwise_inference_linear(input, self.weight_data, self.weight_scales, self.bias)

    def _forward_cast(self, input: BlockwiseActivations) -> torch.Tensor:
        k, n = self.in_features, self.out_features
        if input.shape[-1] != k:
            raise ValueError(f"Float8BlockwiseInferenceLinear: activations of shape {input.shape} do not end in the {k} in_features of the weight")
        dtype = torch.get_autocast_dtype("cuda") if torch.is_autocast_enabled() else input.dtype
        y = None
        if not torch.compiler.is_compiling():
            y = _native.model_ops().blockwise_inference_linear_cast(input.data, input.scales, input.data.shape[1], dtype, self.weight_data, self.weight_scales, n, k, self.bias)
        if y is None:
            if not torch.compiler.is_compiling():
                _native.refuse_tangents("Float8BlockwiseInferenceLinear", self.bias)
            _native._require_gpu(input.data, "input")
            if self.bias is not None:
                _native._require_gpu(self.bias, "bias")
                if self.bias.shape != (n,) or self.bias.dtype not in _HP_DTYPES:
                    raise ValueError(f"Float8BlockwiseInferenceLinear: bias of shape {tuple(self.bias.shape)} ({self.bias.dtype}) for {n} out_features")
            y = _compiled_model.blockwise_inference_linear_cast(input.data, input.scales, self.weight_data, self.weight_scales, k, dtype, self.bias)
        return y.reshape(*input.shape[:-1], n)

    def dequantized_weight(self) -> torch.Tensor:
        """[out_features, in_features] in fp32: the values that the weight stands for."""
        return _native.Blocks(self.weight_data, self.weight_scales, self.out_features, self.in_features).dequant().float()

    def extra_repr(self):
        return f"in_features={self.in_features}, out_features={self.out_features}, bias={self.bias is not None}, scaling=blockwise"

    @classmethod
    def from_float(cls, mod: nn.Linear) -> "Float8BlockwiseInferenceLinear":
        """The weight of ``mod`` (any linear with plain parameters) cast once; its bias is shared."""
        weight = mod.weight.detach()
        _native._require_gpu(weight, "weight")
        if weight.dtype not in _HP_DTYPES or weight.numel() == 0:
            raise TypeError(f"a weight of shape {tuple(weight.shape)} ({weight.dtype}) cannot be quantized")
        new_mod = cls(mod.in_features, mod.out_features, None if mod.bias is None else mod.bias.detach(), device="meta")
        ((blocks, _),) = _native.block_cast([(weight, True, True, False)])
        new_mod.weight_data, new_mod.weight_scales = blocks.data, blocks.scales
        new_mod.train(mod.training)
        return new_mod
