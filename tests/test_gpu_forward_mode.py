"""Blockwise linears and layer norm have no forward-mode derivatives: a tangent raises, and a dual level without one changes nothing."""
import pytest
import torch
import torch.autograd.forward_ad as fwd
import torch.nn as nn

pytestmark = pytest.mark.gpu
BF16 = torch.bfloat16


@pytest.fixture(scope="module")
def f8():
    import float8_experimental_amd

    return float8_experimental_amd


def calls(f8):
    """name -> (call, its differentiable arguments)"""
    r = lambda *s: torch.randn(s, device="cuda", dtype=BF16)
    served = f8.Float8BlockwiseInferenceLinear.from_float(nn.Linear(256, 128, device="cuda", dtype=BF16))
    return {"linear": (f8.blockwise_linear, [r(40, 256), r(128, 256), r(128)]), "served": (served, [r(3, 256)]), "served, many": (served, [r(300, 256)]),
            "norm": (lambda x, w, b: f8.layer_norm(x, 256, w, b), [r(40, 256), r(256), r(256)])}


@pytest.mark.parametrize("name", ["linear", "served", "served, many", "norm"])
def test_tangents_raise(f8, name):
    call, args = calls(f8)[name]
    for i in range(len(args)):
        for context in (torch.no_grad, torch.enable_grad):
            with fwd.dual_level(), context():
                dual = [fwd.make_dual(t, torch.ones_like(t)) if j == i else t for j, t in enumerate(args)]
                with pytest.raises(NotImplementedError, match="forward-mode"):
                    call(*dual)
    with pytest.raises(NotImplementedError, match="forward-mode"):
        torch.func.jvp(call, tuple(args), tuple(torch.ones_like(t) for t in args))


@pytest.mark.parametrize("name", ["linear", "served", "served, many", "norm"])
def test_levels_without_tangents_change_nothing(f8, name):
    call, args = calls(f8)[name]
    with torch.no_grad():
        want = call(*args)
        with fwd.dual_level():
            assert torch.equal(call(*args), want)
