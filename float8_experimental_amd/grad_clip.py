"""The global norm of many gradients and their clipping, in two launches for each 96 tensors (csrc/f8mi_grad_clip.hip)."""
import functools
import math
from typing import Iterable, List, Optional, Tuple, Union

import torch

from . import _native

_HP_DTYPES = (torch.bfloat16, torch.float16, torch.float32)
_KINDS = {2.0: 2, 1.0: 1, math.inf: 0}  # F8MI_NORM_*


def _kind(norm_type: float) -> int:
    kind = _KINDS.get(float(norm_type))
    if kind is None:
        raise ValueError(f"norm_type {norm_type} is not implemented: 2, 1 or inf")
    return kind


def _readable(tensors: Iterable[torch.Tensor]) -> List[torch.Tensor]:
    """The tensors, or copies of those whose memory cannot be read in one run as their values; raises for those that are not taken."""
    out = []
    for t in tensors:
        _native._require_gpu(t, "gradient")
        if type(t) not in (torch.Tensor, torch.nn.Parameter) or t.layout is not torch.strided:
            raise TypeError(f"gradient: a {type(t).__name__} of layout {t.layout}; a plain dense tensor is needed")
        if t.dtype not in _HP_DTYPES:
            raise TypeError(f"gradient is {t.dtype}; bfloat16, float16 or float32 is needed")
        t = t.detach().resolve_neg()
        out.append(t if torch.ops.aten.is_non_overlapping_and_dense(t) else t.contiguous())
    return out


@torch._dynamo.disable
def _call_outside_graph(tensors, what, kind, max_norm):
    return _native.ops().grad_clip(tensors, what, kind, max_norm)


def _call(tensors: List[torch.Tensor], what, kind: int, max_norm: float):
    """(norm, new tensors or None), or None: something has to be looked at one by one."""
    if torch.compiler.is_compiling():
        return _call_outside_graph(tensors, what, kind, max_norm)
    return _native.ops().grad_clip(tensors, what, kind, max_norm)


def _must(result):
    if result is None:
        raise _native.Float8NativeError("gradient clipping under a dispatch mode, a trace or a functional transform is not implemented")
    return result


def _shown_to_function_modes(fn):
    """A ``TorchFunctionMode`` sees a call of ``fn`` as one operation."""

    @functools.wraps(fn)
    def call(*args, **kwargs):
        if not torch.compiler.is_compiling() and torch._C._is_torch_function_mode_enabled() and _native._function_mode_active():
            return torch.overrides.handle_torch_function(call, (), *args, **kwargs)
        return fn(*args, **kwargs)

    return call


@_shown_to_function_modes
def grad_norm(grads: Iterable[torch.Tensor], norm_type: float = 2.0, error_if_nonfinite: bool = False) -> torch.Tensor:
    """The norm (2, 1 or inf) of all values of all tensors as if they were one vector: a 0-dim float32 tensor.  Sums are kept in 64 bits
    and have a fixed order."""
    grads, kind = list(grads), _kind(norm_type)
    norm, _ = _call(grads, "norm", kind, 0.0) or _must(_call(_readable(grads), "norm", kind, 0.0))
    if error_if_nonfinite and not math.isfinite(norm.item()):
        raise RuntimeError(f"the norm of the gradients is {norm.item()} (error_if_nonfinite=True)")
    return norm


@_shown_to_function_modes
def clip_grads(grads: Iterable[torch.Tensor], max_norm: float, norm_type: float = 2.0, error_if_nonfinite: bool = False,
               out_dtype: Optional[torch.dtype] = None) -> Tuple[torch.Tensor, List[torch.Tensor]]:
    """(norm, ``[g * min(1, max_norm / (norm + 1e-6)) for g in grads]``) in new tensors of ``out_dtype`` (default: each gradient's own), for
    optimizers that take gradients of another type than the parameters': no fp32 copy of the gradients comes between."""
    if out_dtype is not None and out_dtype not in _HP_DTYPES:
        raise TypeError(f"clip_grads: out_dtype {out_dtype}; bfloat16, float16 or float32 is needed")
    grads, kind = list(grads), _kind(norm_type)
    if error_if_nonfinite:
        grad_norm(grads, norm_type, True)
    return _call(grads, out_dtype, kind, float(max_norm)) or _must(_call(_readable(grads), out_dtype, kind, float(max_norm)))


@_shown_to_function_modes
def clip_grad_norm_(parameters: Union[torch.Tensor, Iterable[torch.Tensor]], max_norm: float, norm_type: float = 2.0,
                    error_if_nonfinite: bool = False, foreach: Optional[bool] = None) -> torch.Tensor:
    """``torch.nn.utils.clip_grad_norm_`` for the norms 2, 1 and inf (``foreach`` chooses nothing: there is one implementation): scales the
    gradients of ``parameters`` in place so that their norm as one vector is at most ``max_norm``, and returns the norm before (0-dim
    float32).  A gradient that is listed more than once counts in the norm as often and is scaled once.  Nothing is written where nothing is
    clipped, and nothing waits for the GPU unless ``error_if_nonfinite``, which raises before a gradient is changed."""
    parameters, kind = [parameters] if isinstance(parameters, torch.Tensor) else list(parameters), _kind(norm_type)
    if error_if_nonfinite:
        grad_norm([p.grad for p in parameters if p.grad is not None], norm_type, True)
    done = _call(parameters, "grads", kind, float(max_norm))
    if done is None:
        grads = [p.grad for p in parameters if p.grad is not None]
        done = _must(_call(_readable(grads), None, kind, float(max_norm)))
        with torch.no_grad():
            for g, clipped in zip(grads, done[1]):
                g.copy_(clipped)
    return done[0]
