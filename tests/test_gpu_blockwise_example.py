"""The example that trains and serves a model on the blockwise linears, layer norm and gradient clipping together."""
import importlib.util
import os

import pytest
import torch
import torch.nn as nn

import float8_experimental_amd as f8

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def example():
    path = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "examples", "train_and_serve_blockwise.py")
    spec = importlib.util.spec_from_file_location("train_and_serve_blockwise", path)
    module = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(module)
    return module


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("dim,hidden", [(256, 640), (200, 333)])
def test_a_model_learns_and_answers_from_its_served_weights(example, dtype, dim, hidden):
    losses, norms, model, served = example.run(steps=40, dim=dim, hidden=hidden, tokens=500, dtype=dtype)
    assert torch.isfinite(losses).all() and torch.isfinite(norms).all() and (norms > 0).all()
    assert losses[-5:].mean() < 0.5 * losses[0]
    kinds = {type(m) for m in model.modules()}
    assert f8.Float8BlockwiseLinear in kinds and f8.LayerNorm in kinds and nn.Linear not in kinds and nn.LayerNorm not in kinds
    assert f8.Float8BlockwiseLinear not in {type(m) for m in served.modules()}
    with torch.no_grad():
        for rows in (1, 7, 300):
            x = torch.randn(rows, dim, device="cuda", dtype=dtype)
            # the same casts and products but for the order of the sums, which may move a value to the next e4m3 one further on
            y, got = model(x).float(), served(x).float()
            assert (y - got).abs().max() <= 0.05 * y.abs().max()


def test_a_step_clips_to_the_norm_and_updates_by_the_clipped_gradients(example):
    torch.manual_seed(1)
    model = example.make_model(128, 256, 1, torch.bfloat16)
    masters = [p.detach().float().requires_grad_() for p in model.parameters()]
    before = [m.detach().clone() for m in masters]
    x, target = torch.randn(2, 100, 128, device="cuda", dtype=torch.bfloat16)
    loss = nn.functional.mse_loss(model(x).float(), target.float())
    grads = [g.double() for g in torch.autograd.grad(loss, list(model.parameters()))]
    want = torch.stack([g.pow(2).sum() for g in grads]).sum().sqrt()
    factor = 0.5 * want / (want + 1e-6)
    _, norm = example.train_step(model, torch.optim.SGD(masters, lr=1.0), masters, x, target, 0.5 * want.item())
    assert (norm.double() - want).abs() <= 1e-6 * want
    for m, b, g, p in zip(masters, before, grads, model.parameters()):
        # two roundings of fp32: the scaled gradient's and the update's
        assert ((b.double() - factor * g) - m.double()).abs().max() <= 2.0 ** -22 * (b.abs().max() + g.abs().max())
        assert torch.equal(p, m.to(p.dtype))
