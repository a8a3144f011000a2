"""Traces of RMS norm, dropout and the adapters, replayed with tensors of other sizes: the formula's values where they fit, an error where they do not."""
import pytest
import torch

pytestmark = [pytest.mark.gpu, pytest.mark.filterwarnings("ignore")]
BF16, FP32 = torch.bfloat16, torch.float32


@pytest.fixture(scope="module")
def f8():
    import float8_experimental_amd

    return float8_experimental_amd


def normal(*shape, dtype=BF16, seed=0):
    return torch.randn(shape, generator=torch.Generator().manual_seed(seed)).to(dtype).cuda()


@pytest.mark.parametrize("grad", [False, True])
def test_norms_and_dropout(f8, grad):
    make = lambda m, seed: tuple(t.requires_grad_(grad) for t in (normal(m, 200, seed=seed), normal(200, seed=seed + 1), normal(m, 200, seed=seed + 2)))
    seed = torch.full((1,), 7, dtype=torch.int64, device="cuda")
    norm, drop = lambda x, w, r: f8.rms_norm(x, 200, w, 1e-6, r), lambda x, w, r: f8.dropout(x, 0.25, seed, r)
    for call in (norm, drop):
        traced = torch.jit.trace(call, make(5, 0))
        for m in (5, 64, 1):
            args = make(m, m)
            got, want = traced(*args), call(*args)
            assert all(torch.equal(p, q) for p, q in zip(got, want)) if isinstance(want, tuple) else torch.equal(got, want)
        x, w, r = make(5, 0)
        with pytest.raises(RuntimeError):
            traced(x, w, r[:4])
        if call is norm:
            with pytest.raises(RuntimeError):
                traced(x, w[:199], r)


@pytest.mark.parametrize("grad", [False, True])
def test_adapters(f8, grad):
    a, b, rows = normal(3, 8, 256), normal(3, 64, 8, seed=1), f8.AdapterRows(torch.arange(8, device="cuda") % 3, 3)
    x, y = normal(8, 256, seed=2).requires_grad_(grad), normal(8, 64, seed=3)
    call = lambda x, a, b, y: f8.low_rank_adapters(x, a, b, rows, y)
    traced = torch.jit.trace(call, (x, a, b, y))
    assert torch.equal(traced(x, a, b, y), call(x, a, b, y))
    for args in ((x[:5], a, b, y[:5]), (x[:5], a, b, y), (x, a[:2], b[:2], y), (x, a, b, y[:7]), (x, a, b[:, :63], y)):
        with pytest.raises(RuntimeError):
            traced(*args)
    inside = lambda x, ids, y: f8.low_rank_adapters(x, a, b, f8.AdapterRows(ids, 3), y)
    traced = torch.jit.trace(inside, (x, torch.arange(8, device="cuda") % 3, y))
    for m in (8, 5, 100):
        args = normal(m, 256, seed=m).requires_grad_(grad), torch.arange(m, device="cuda") % 4 - 1, normal(m, 64, seed=m + 1)
        assert torch.equal(traced(*args), inside(*args))
    with pytest.raises(RuntimeError):
        traced(x, torch.zeros(5, dtype=torch.int64, device="cuda"), y)
