"""The norm of many gradients and their clipping: the norm against 64 bits, the clipped values to the bit."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu

BF16, FP16, FP32 = torch.bfloat16, torch.float16, torch.float32


@pytest.fixture(scope="module")
def f8():
    import float8_experimental_amd

    return float8_experimental_amd


def values(shape, dtype, seed=0, std=1.0):
    return (torch.randn(shape, generator=torch.Generator().manual_seed(seed)) * std).to(dtype).cuda()


def norm64(grads, kind=2.0):
    v = torch.cat([g.double().reshape(-1) for g in grads])
    return v.square().sum().sqrt().item() if kind == 2.0 else v.abs().sum().item() if kind == 1.0 else v.abs().max().item()


def clipped(grads, norm, max_norm, dtype=None):
    """fp32 arithmetic on the returned norm, one rounding"""
    factor = torch.clamp(torch.tensor(max_norm, dtype=FP32) / (norm.cpu() + torch.tensor(1e-6, dtype=FP32)), max=1.0).cuda()
    return [(g.float() * factor).to(dtype or g.dtype) for g in grads]


def params_of(grads):
    params = [torch.nn.Parameter(torch.empty_like(g)) for g in grads]
    for p, g in zip(params, grads):
        p.grad = g
    return params


SIZES = [1, 2, 7, 8, 9, 1000, 4096, 16383, 16384, 16385, 100003, 3 * 16384 * 5 + 11]


@pytest.mark.parametrize("kind", [2.0, 1.0, math.inf])
@pytest.mark.parametrize("dtype", [BF16, FP16, FP32])
def test_one_tensor_of_any_size(f8, dtype, kind):
    for n in SIZES:
        g = values((n,), dtype, n)
        norm, (out,) = f8.clip_grads([g], 0.7, norm_type=kind)
        assert abs(norm.item() - norm64([g], kind)) <= 2.0**-23 * norm64([g], kind) and norm.dtype == FP32 and norm.dim() == 0
        assert torch.equal(out, clipped([g], norm, 0.7)[0])
        assert torch.equal(f8.grad_norm([g], kind), norm)


@pytest.mark.parametrize("count", [2, 95, 96, 97, 300])
@pytest.mark.parametrize("out_dtype", [None, FP32, BF16, FP16])
def test_lists_of_mixed_types_and_sizes(f8, count, out_dtype):
    kinds = (BF16, FP32, FP16)
    grads = [values((1 + 37 * i * i % 5000,), kinds[i % 3], i) for i in range(count)]
    grads[1] = values((300, 700), FP32, 5)
    norm, out = f8.clip_grads(grads, 3.0, out_dtype=out_dtype)
    assert abs(norm.item() - norm64(grads)) <= 2.0**-23 * norm64(grads)
    want = clipped(grads, norm, 3.0, out_dtype)
    assert all(p.dtype == (out_dtype or g.dtype) and p.shape == g.shape and torch.equal(p, q) for p, q, g in zip(out, want, grads))
    params = params_of([g.clone() for g in grads])
    assert torch.equal(f8.clip_grad_norm_(params, 3.0), norm)
    assert all(torch.equal(p.grad, q) for p, q in zip(params, clipped(grads, norm, 3.0)))


def test_below_the_limit_nothing_changes(f8):
    grads = [values((1000,), BF16), values((5, 7), FP32, 1)]
    params = params_of([g.clone() for g in grads])
    norm = f8.clip_grad_norm_(params, 2 * norm64(grads))
    assert all(torch.equal(p.grad, g) for p, g in zip(params, grads)) and abs(norm.item() - norm64(grads)) <= 2.0**-23 * norm64(grads)
    _, out = f8.clip_grads(grads, 1e30)
    assert all(torch.equal(p, q) and p.data_ptr() != q.data_ptr() for p, q in zip(out, grads))


def test_as_torch_does(f8):
    grads = [values((500, 30), FP32), values((77,), FP32, 1)]
    ours, theirs = params_of([g.clone() for g in grads]), params_of([g.clone() for g in grads])
    torch.testing.assert_close(f8.clip_grad_norm_(ours, 1.0), torch.nn.utils.clip_grad_norm_(theirs, 1.0), rtol=1e-6, atol=0)
    for p, q in zip(ours, theirs):
        torch.testing.assert_close(p.grad, q.grad, rtol=1e-6, atol=0)


def test_views_orders_and_alignments(f8):
    """Dense tensors in any order of dimensions are read as they lie; others through a copy; in place the gradient itself changes."""
    base = values((60, 80, 3), BF16)
    grads = [base[:, :, 0], base.transpose(0, 2), base[1:, 1:, 1], values((1001,), FP32, 2)[1:], values((301,), BF16, 3)[1:], values((4, 1), FP32, 4).expand(4, 50)]
    norm, out = f8.clip_grads(grads, 2.0)
    assert abs(norm.item() - norm64(grads)) <= 2.0**-23 * norm64(grads)
    assert all(torch.equal(p, q) for p, q in zip(out, clipped(grads, norm, 2.0)))
    weights = [torch.nn.Parameter(torch.zeros(s, device="cuda")) for s in ((40, 30), (30, 40), (64, 64))]
    grads = [values((30, 40), FP32).t(), values((30, 80), FP32, 1)[:, ::2], values((64, 64), FP32, 2)]
    want = [g.clone() for g in grads]
    for p, g in zip(weights, grads):
        p.grad = g
    norm = f8.clip_grad_norm_(iter(weights), 1.0)
    assert all(p.grad is g and torch.equal(g, q) for p, g, q in zip(weights, grads, clipped(want, norm, 1.0)))


def test_nothing_to_clip(f8):
    p = torch.nn.Parameter(torch.zeros(3, device="cuda"))
    assert f8.clip_grad_norm_([p], 1.0).item() == 0.0 and f8.clip_grad_norm_([], 1.0).item() == 0.0 and p.grad is None
    empty = torch.zeros((0, 4), device="cuda")
    norm, out = f8.clip_grads([empty, empty], 1.0)
    assert norm.item() == 0.0 and out[0].shape == (0, 4)
    norm, out = f8.clip_grads([empty, torch.full((2,), 3.0, device="cuda"), empty], 1e9)
    assert abs(norm.item() - math.sqrt(18)) < 1e-6 and out[1].tolist() == [3.0, 3.0]
    assert f8.clip_grad_norm_(params_of([torch.zeros(10, device="cuda")])[0], 1.0).item() == 0.0


def test_sizes_that_squares_in_fp32_would_lose(f8):
    for std in (1e-30, 1e25):
        grads = [values((5000,), FP32, 0, std), values((300,), BF16, 1, std)]
        norm, out = f8.clip_grads(grads, std)
        want = norm64(grads)
        assert abs(norm.item() - want) <= 2.0**-22 * want
    assert f8.grad_norm([torch.full((1 << 20,), 1e-3, device="cuda")], 1.0).item() == pytest.approx((1 << 20) * float(torch.tensor(1e-3)), rel=1e-7)


@pytest.mark.parametrize("kind", [2.0, 1.0, math.inf])
@pytest.mark.parametrize("bad", [math.nan, math.inf, -math.inf])
def test_values_that_are_not_finite(f8, kind, bad):
    grads = [values((5000,), FP32), values((40000,), BF16, 1)]
    grads[1][39990] = bad
    norm, out = f8.clip_grads(grads, 1.0, norm_type=kind)
    assert math.isnan(norm.item()) if math.isnan(bad) else norm.item() == math.inf
    for p, q in zip(out, clipped(grads, norm, 1.0)):
        assert torch.equal(p.isnan(), q.isnan()) and torch.equal(p[~p.isnan()], q[~q.isnan()])
    params = params_of([g.clone() for g in grads])
    with pytest.raises(RuntimeError):
        f8.clip_grad_norm_(params, 1.0, kind, error_if_nonfinite=True)
    assert torch.equal(params[0].grad, grads[0])  # raised before anything changed


def test_stream_graph_and_version(f8):
    grads = [values((300, 300), BF16), values((70,), FP32, 1)]
    want = f8.clip_grads(grads, 2.0)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = f8.clip_grads(grads, 2.0)
        f8.clip_grads(grads, 2.0)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(got[0], want[0]) and all(torch.equal(p, q) for p, q in zip(got[1], want[1]))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = f8.clip_grads(grads, 2.0)
    for i in range(3):
        grads[0].copy_(values((300, 300), BF16, 20 + i))
        graph.replay()
        torch.cuda.synchronize()
        want = f8.clip_grads(grads, 2.0)
        assert torch.equal(got[0], want[0]) and all(torch.equal(p, q) for p, q in zip(got[1], want[1]))
    params = params_of(grads)
    before = grads[0]._version
    f8.clip_grad_norm_(params, 1.0)
    assert grads[0]._version > before  # autograd hears of the change


def test_refusals(f8):
    g = values((10,), FP32)
    for bad in (lambda: f8.clip_grads([g], 1.0, norm_type=3.0), lambda: f8.grad_norm([g], 0.5)):
        with pytest.raises(ValueError):
            bad()
    for bad in (lambda: f8.clip_grads([g.double()], 1.0), lambda: f8.clip_grads([g], 1.0, out_dtype=torch.float64), lambda: f8.grad_norm([g.to_sparse()])):
        with pytest.raises(TypeError):
            bad()
    with pytest.raises(RuntimeError):
        f8.grad_norm([g, g.cpu()])
