"""float16 adapters whose inner values differ by 2^20 within a row, where the second matrix takes the small ones alone: what is left of them is the result."""
import pytest
import torch

pytestmark = pytest.mark.gpu
FP16, FP = torch.float16, 2.0**-24


@pytest.fixture(scope="module")
def f8():
    import float8_experimental_amd

    return float8_experimental_amd


def made(m, k, n, r, count):
    """Both passes: the first quarter of the rank is 2^20 times as large as the rest in a (in b for the gradient's half), and zero in b (in a)."""
    g = torch.Generator().manual_seed(m + n)
    normal = lambda *s: torch.randn(s, generator=g)
    x, dout = normal(m, k), normal(m, n)
    first = torch.arange(r) < max(1, r // 4)
    a, b = normal(count, r, k), normal(count, n, r)
    return x, a, b, dout, first


def products(x, w, v, ids, first_product):
    """(second product, what it may be off by) of rows x with w [count, r, k] and v [count, n, r], in 64 bits"""
    out, off = torch.zeros(len(x), v.shape[1], dtype=torch.float64), torch.zeros(len(x), v.shape[1], dtype=torch.float64)
    for e in range(len(w)):
        at = (ids == e).nonzero().flatten()
        xe = x[at].double()
        h = xe @ w[e].double().t()
        # fp32 sums, then two fp16 parts: 2^-21 of themselves or 2^-38 of the row's largest
        h_off = (first_product + 40) * FP * (xe.abs() @ w[e].double().abs().t()) + 2.0**-21 * h.abs() + 2.0**-38 * h.abs().amax(1, keepdim=True)
        out[at] = h @ v[e].double().t()
        off[at] = (h_off + (2 * w.shape[1] + 16) * FP * h.abs()) @ v[e].double().abs().t()
    return out, off


def check(got, exact, off):
    tol = 2.0**-11 * exact.abs() + 1.001 * off + 2.0**-25
    worst = ((got.detach().cpu().double() - exact).abs() / tol).max().item()
    assert worst <= 1.0, worst


SHAPES = [  # one launch, two, tiles of 64 rows with their columns through LDS or not, ranks that end inside an instruction
    (1, 64, 128, 16, 1), (16, 64, 500, 5, 3), (20, 5000, 200, 16, 2), (20, 300, 200, 64, 2), (100, 64, 60, 16, 1), (200, 64, 300, 12, 2), (100, 200, 300, 64, 1), (130, 64, 256, 100, 1), (100, 96, 130, 256, 1),
]


@pytest.mark.parametrize("shape", SHAPES, ids=lambda s: "x".join(map(str, s)))
def test_small_inner_values_beside_large_ones(f8, shape):
    m, k, n, r, count = shape
    x, a, b, dout, first = made(*shape)
    ids = torch.arange(m) % count
    rows = f8.AdapterRows(ids.cuda(), count)
    scaled = lambda t, dim: t * torch.where(first, 2.0**10, 2.0**-10).view([-1 if i == dim else 1 for i in range(3)])
    without = lambda t, dim: t * (~first).view([-1 if i == dim else 1 for i in range(3)])
    p, q, xh = scaled(a, 1).mul(k**-0.5).to(FP16), without(b, 2).to(FP16), x.to(FP16)
    exact, off = products(xh, p, q, ids, k)
    assert exact.abs().median() > 2.0**-13  # (normal fp16 values, unless the rank is all large)
    check(f8.low_rank_adapters(xh.cuda(), p.cuda(), q.cuda(), rows), exact, off)
    p, q, g = without(a, 1).to(FP16), scaled(b, 2).mul(n**-0.5).to(FP16), dout.to(FP16)
    exact, off = products(g, q.transpose(1, 2).contiguous(), p.transpose(1, 2).contiguous(), ids, n)
    v = xh.cuda().requires_grad_()
    f8.low_rank_adapters(v, p.cuda(), q.cuda(), rows).backward(g.cuda())
    check(v.grad, exact, off)


def test_rows_at_the_ends_of_fp32(f8):
    """A row's largest inner value near fp32's largest or far below its normal ones: the power of two stays one that fp32 has."""
    k = n = 64
    ones = torch.ones(1, 4, k, dtype=FP16)
    for scale in (2.0**100, 2.0**-100, 2.0**-130):
        x, b = torch.full((3, k), 2.0**9, dtype=FP16), torch.full((1, n, 4), 2.0**-8, dtype=FP16)
        h = 2.0**9 * k * scale
        got = f8.low_rank_adapters(x.cuda(), ones.cuda(), b.cuda(), torch.zeros(3, dtype=torch.int64, device="cuda"), None, torch.tensor([scale], device="cuda"))
        want = torch.tensor(h * 4 * 2.0**-8, dtype=torch.float64).to(FP16)  # powers of two throughout: exact, infinite or zero
        assert (got.cpu() == want).all(), (scale, got[0, 0], want)
