"""Tensors whose offsets pass 32 bits: the last rows have the values that they have by themselves."""
import pytest
import torch

import float8_experimental_amd as f8

pytestmark = pytest.mark.gpu
ROWS, COLS = 600_000, 4096  # 4.9 GB of bfloat16


@pytest.fixture(scope="module")
def big():
    torch.manual_seed(0)
    yield torch.randn(ROWS, COLS, device="cuda", dtype=torch.bfloat16)
    torch.cuda.empty_cache()


def test_linear(big):
    """Blocks of the forward pass and of the gradient of x lie in their row, sums have one order whatever the number of rows."""
    w = (torch.randn(4096, COLS, device="cuda") / 64).bfloat16().requires_grad_()
    tail = big[-8192:].clone().requires_grad_()
    y = f8.blockwise_linear(tail, w)
    (want,) = torch.autograd.grad(y, tail, tail.detach())
    x = big.detach().requires_grad_()
    z = f8.blockwise_linear(x, w)
    assert torch.equal(z[-8192:], y)
    (got,) = torch.autograd.grad(z, x, big)
    assert torch.equal(got[-8192:], want)


def test_gradient_of_the_weight(big):
    """One token far behind 2^32 bytes, all others zero: its products alone."""
    x = torch.zeros_like(big)
    w = torch.zeros(256, COLS, device="cuda", dtype=torch.bfloat16, requires_grad=True)
    x[-3] = 2.0
    dy = torch.zeros(ROWS, 256, device="cuda", dtype=torch.bfloat16)
    dy[-3] = torch.arange(256, device="cuda").bfloat16() % 8
    (dw,) = torch.autograd.grad(f8.blockwise_linear(x, w), w, dy)
    assert torch.equal(dw, (2.0 * dy[-3])[:, None].expand_as(dw))


def test_layer_norm(big):
    w, b = torch.randn(2, COLS, device="cuda").unbind(0)
    tail = big[-1000:].clone().requires_grad_()
    y = f8.layer_norm(tail, COLS, w, b)
    (want,) = torch.autograd.grad(y, tail, tail.detach())
    x = big.detach().requires_grad_()
    z = f8.layer_norm(x, COLS, w, b)
    assert torch.equal(z[-1000:], y)
    (got,) = torch.autograd.grad(z, x, big)
    assert torch.equal(got[-1000:], want)


def test_clipping(big):
    total = sum(chunk.double().pow(2).sum() for chunk in big.split(50_000)).sqrt()
    norm, (clipped,) = f8.clip_grads([big], 1.0)
    assert abs(norm.double() - total) <= 2.0**-23 * total
    _, (tail,) = f8.clip_grads([big[-1000:]], 1e30)
    assert torch.equal(tail, big[-1000:])
    # the scaled value in fp32 has two roundings at most (factor, product), then one to bfloat16
    want = big[-1000:].double() / (total + 1e-6)
    assert ((clipped[-1000:].double() - want).abs() <= want.abs() * (2.0**-8 + 2.0**-22)).all()
