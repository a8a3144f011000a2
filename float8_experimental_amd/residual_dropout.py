"""Dropout whose mask is never stored, with the addition to the residual stream behind it (csrc/f8mi_dropout.hip)."""
from typing import Optional

import torch
import torch.nn as nn

from . import _custom_ops_model as _compiled
from . import _native
from .module_swap import swap_modules

_HP_DTYPES = (torch.bfloat16, torch.float16, torch.float32)


def dropout(x: torch.Tensor, p: float = 0.5, seed: Optional[torch.Tensor] = None, residual: Optional[torch.Tensor] = None) -> torch.Tensor:
    """``residual + (x / (1 - p) where kept, else 0)``, each value kept with probability 1 - p.

    Which values are kept follows from ``seed`` alone (one int64 on x's device; None: drawn from torch's generator of that device): value i, counted in the order of a
    contiguous x, where word i % 4 of the block i / 4 of the generator Philox 4x32-7 with the seed's bits as its key is at least p * 2^32.  The backward pass finds them again from the seed,
    which must not be written in between.  A captured graph reads the seed, or draws it, anew at each replay.

    ``x`` in bfloat16, float16 or float32; the residual has x's shape and type; computed in fp32 and rounded once."""
    if not 0.0 <= p <= 1.0:
        raise ValueError(f"dropout: p={p} is not a probability")
    if seed is None:
        _native._require_gpu(x, "x")
        seed = torch.randint(2**63 - 1, (1,), device=x.device)
    if not torch.compiler.is_compiling():
        out = _native.model_ops().dropout(x, p, seed, residual)
        if out is not None:
            return out
        _native.refuse_tangents("dropout", x, residual)
    _native._require_gpu(x, "x")
    if x.dtype not in _HP_DTYPES:
        raise TypeError(f"dropout: x is {x.dtype}; bfloat16, float16 or float32 is needed")
    _native._require_gpu(seed, "seed")
    if seed.dtype != torch.int64 or seed.numel() != 1:
        raise ValueError(f"dropout: seed of shape {tuple(seed.shape)} ({seed.dtype}); one int64 is needed")
    if residual is not None:
        _native._require_gpu(residual, "residual")
        if residual.shape != x.shape or residual.dtype != x.dtype:
            raise ValueError(f"dropout: residual of shape {tuple(residual.shape)} ({residual.dtype}) for x of shape {tuple(x.shape)} ({x.dtype})")
    if p == 1.0:  # nothing is kept
        nothing = torch.zeros_like(x) if not (torch.is_grad_enabled() and x.requires_grad) else x.masked_fill(torch.ones((), dtype=torch.bool, device=x.device), 0.0)
        return nothing if residual is None else residual + nothing
    return _compiled.dropout(x, residual, seed, float(p))


class Dropout(nn.Dropout):
    """``nn.Dropout`` on this package's kernel; a residual to add to may come with the input."""

    def __init__(self, p: float = 0.5, inplace: bool = False):
        if inplace:
            raise NotImplementedError("dropout in place is not implemented")
        super().__init__(p)

    def forward(self, input: torch.Tensor, residual: Optional[torch.Tensor] = None) -> torch.Tensor:
        if self.training and self.p > 0.0:
            return dropout(input, self.p, residual=residual)
        return input if residual is None else residual + input

    @classmethod
    def from_float(cls, mod: nn.Dropout) -> "Dropout":
        new_mod = cls(mod.p, mod.inplace)
        new_mod.train(mod.training)
        return new_mod


def convert_dropouts(module: nn.Module) -> nn.Module:
    """Swaps every ``nn.Dropout`` of ``module`` for a ``Dropout``; a root-level one is returned converted."""
    return swap_modules(module, nn.Dropout, Dropout.from_float)
