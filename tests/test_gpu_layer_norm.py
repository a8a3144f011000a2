"""Layer norm, forward and backward, against the formula in 64 bits and against differences."""
import pytest
import torch
import torch.nn as nn

pytestmark = pytest.mark.gpu

BF16, FP16, FP32 = torch.bfloat16, torch.float16, torch.float32
EPS = {BF16: 2.0**-8, FP16: 2.0**-11, FP32: 2.0**-23}
FP = 2.0**-24  # a rounding of fp32


@pytest.fixture(scope="module")
def f8():
    import float8_experimental_amd

    return float8_experimental_amd


def made(rows, cols, dtype, p_dtype, seed=0, offset=0.5):
    g = torch.Generator().manual_seed(seed)
    x = (torch.randn(rows, cols, generator=g) * torch.randn(cols, generator=g).exp() + offset).to(dtype)
    w, b = (1 + 0.1 * torch.randn(cols, generator=g)).to(p_dtype), (0.1 * torch.randn(cols, generator=g)).to(p_dtype)
    return x.cuda(), w.cuda(), b.cuda(), (1e-2 * torch.randn(rows, cols, generator=g)).to(dtype).cuda()


def formula(x, w, b, dy, eps=1e-5):
    x, dy = x.detach().double(), dy.double()
    w = torch.ones_like(x[0]) if w is None else w.detach().double()
    b = torch.zeros_like(x[0]) if b is None else b.detach().double()
    mean = x.mean(1, keepdim=True)
    rstd = 1 / (x.var(1, keepdim=True, correction=0) + eps).sqrt()
    xh = (x - mean) * rstd
    g = dy * w
    m1, m2 = g.mean(1, keepdim=True), (g * xh).mean(1, keepdim=True)
    return xh, rstd, mean, w, b, {"y": xh * w + b, "dx": rstd * (g - m1 - xh * m2), "dw": (dy * xh).sum(0), "db": dy.sum(0)}


def check(x, w, b, dy, got, eps=1e-5):
    """One rounding to the output's type, and fp32 arithmetic: a sum over the columns goes through 64 additions a lane, 6 steps between lanes and 16
    between waves at most (C roundings in all), one over the rows through at most `rows` additions and 32 more."""
    xh, rstd, mean, wd, bd, want = formula(x, w, b, dy, eps)
    rows, cols = x.shape
    C = 96 * FP
    g, gx = (dy.double() * wd).abs(), (dy.double() * wd * xh).abs()
    # how far the fp32 xhat may be off: the mean by C of the mean magnitude, rstd by C of itself and through the mean
    off = 2 * C * (x.detach().double().abs().mean(1, keepdim=True) * rstd + xh.abs()) + 4 * FP * x.detach().double().abs() * rstd
    size = {"y": off * wd.abs() + 4 * FP * ((xh * wd).abs() + bd.abs()),
            "dx": rstd * (C * (g + g.mean(1, keepdim=True) + xh.abs() * gx.mean(1, keepdim=True)) + off * gx.mean(1, keepdim=True)
                          + xh.abs() * (g * off).mean(1, keepdim=True)) * 2 + C * want["dx"].abs(),
            "dw": (rows + 32) * FP * (dy.double() * xh).abs().sum(0) + (dy.double().abs() * off).sum(0),
            "db": (rows + 32) * FP * dy.double().abs().sum(0)}
    for name, value in got.items():
        if value is None:
            continue
        tol = EPS[value.dtype] * want[name].abs() + size[name] + (2.0**-25 if value.dtype is FP16 else 0) + 1e-37
        worst = ((value.detach().double() - want[name]).abs() / tol).max().item()
        assert worst <= 1.0, (name, worst)


def run(f8, x, w, b, dy, eps=1e-5):
    x, w, b = (None if t is None else t.clone().requires_grad_() for t in (x, w, b))
    y = f8.layer_norm(x, x.shape[1], w, b, eps)
    y.backward(dy)
    return {"y": y, "dx": x.grad, "dw": None if w is None else w.grad, "db": None if b is None else b.grad}


# columns: one, odd, each number of lanes and pieces a row, and rows that do not fit in registers
COLS = [1, 7, 64, 100, 512, 513, 1024, 1500, 2048, 4096, 4097, 5000, 8192, 8200, 16384, 16390, 20011]


@pytest.mark.parametrize("dtype,p_dtype", [(BF16, BF16), (BF16, FP32), (FP16, FP16), (FP32, FP32)])
@pytest.mark.parametrize("cols", COLS)
def test_forward_and_backward(f8, cols, dtype, p_dtype):
    for rows in (1, 3, 70):
        x, w, b, dy = made(rows, cols, dtype, p_dtype, cols + rows)
        check(x, w, b, dy, run(f8, x, w, b, dy))


@pytest.mark.parametrize("rows,cols", [(5000, 64), (2500, 1000), (3000, 4096), (1100, 9000), (600, 20000)])
def test_many_rows(f8, rows, cols):
    x, w, b, dy = made(rows, cols, BF16, FP32)
    first = run(f8, x, w, b, dy)
    check(x, w, b, dy, first)
    again = run(f8, x, w, b, dy)  # sums have a fixed order
    assert all(torch.equal(first[k], again[k]) for k in first)


def test_without_parameters_and_with_either(f8):
    x, w, b, dy = made(20, 300, FP32, FP32)
    for ww, bb in ((None, None), (w, None), (None, b)):
        check(x, ww, bb, dy, run(f8, x, ww, bb, dy))


def test_large_means_and_constant_rows(f8):
    """The variance is that of the row less its mean: a mean a thousand times the spread costs fp32's rounding of the inputs, no more."""
    x, w, b, dy = made(64, 1000, FP32, FP32, offset=1000.0)
    check(x, w, b, dy, run(f8, x, w, b, dy))
    x[5] = 3.0
    x[6] = 0.0
    check(x, w, b, dy, run(f8, x, w, b, dy))


def test_values_that_are_not_finite_stay_in_their_row(f8):
    x, w, b, dy = made(9, 500, BF16, BF16)
    clean = run(f8, x, w, b, dy)
    x[4, 17] = float("nan")
    x[7, 3] = float("inf")
    got = run(f8, x, w, b, dy)
    for r in range(9):
        for name in ("y", "dx"):
            assert got[name][r].isnan().all() if r in (4, 7) else torch.equal(got[name][r], clean[name][r])


def test_strides_and_shapes(f8):
    x, w, b, dy = made(60, 400, BF16, BF16)
    for view in (x[:, 3:260], x[::2, :129], x[:1, 1:].expand(60, 399), x.t()):
        check(view, w[:view.shape[1]] if view.shape[1] <= 400 else None, None, dy[: view.shape[0], : view.shape[1]] if view.shape == (view.shape[0], view.shape[1]) and view.shape[0] <= 60 else
              torch.ones(view.shape, dtype=BF16, device="cuda"),
              run_view(f8, view, w, dy))
    y = f8.layer_norm(x.view(3, 20, 20, 20), (20, 20), w.view(20, 20), b.view(20, 20))
    assert torch.equal(y.view(60, 400), f8.layer_norm(x, 400, w, b))
    z = x.clone().requires_grad_()
    f8.layer_norm(z, 400).sum().backward()  # a gradient that is one number expanded
    assert z.grad.abs().max() < 1e-2
    assert f8.layer_norm(x[:0], 400, w, b).shape == (0, 400)


def run_view(f8, view, w, dy):
    g = dy[: view.shape[0], : view.shape[1]] if view.shape[0] <= 60 else torch.ones(view.shape, dtype=BF16, device="cuda")
    v = view.detach().requires_grad_()
    y = f8.layer_norm(v, v.shape[1], w[: v.shape[1]])
    y.backward(g)
    return {"y": y, "dx": v.grad}


def test_no_rows(f8):
    x, w = torch.zeros((0, 64), device="cuda", requires_grad=True), torch.ones(64, device="cuda", requires_grad=True)
    f8.layer_norm(x, 64, w).sum().backward()
    assert x.grad.shape == (0, 64) and (w.grad == 0).all()


def test_gradients_against_differences(f8):
    """Central differences of the formula in 64 bits."""
    x, w, b, dy = made(6, 50, FP32, FP32)
    got = run(f8, x, w, b, dy)
    loss = lambda x, w, b: (formula(x, w, b, dy)[5]["y"] * dy.double()).sum().item()
    g, h = torch.Generator().manual_seed(1), 1e-4
    for i, name in enumerate(("dx", "dw", "db")):
        for _ in range(6):
            ts = [t.double() for t in (x, w, b)]
            at = tuple(int(torch.randint(0, s, (1,), generator=g)) for s in ts[i].shape)
            ts[i][at] += h
            up = loss(*ts)
            ts[i][at] -= 2 * h
            want = (up - loss(*ts)) / (2 * h)
            # differences: h^2 of the third derivative and the roundings of the loss over h
            assert abs(got[name][at].item() - want) <= 1e-5 * abs(want) + 1e-7


def test_only_the_gradients_that_are_asked_for(f8):
    x, w, b, dy = made(33, 700, BF16, BF16)
    full = run(f8, x, w, b, dy)
    for which in ((1, 0, 0), (0, 1, 0), (0, 0, 1), (0, 1, 1), (1, 0, 1)):
        ts = [t.clone().requires_grad_(bool(r)) for t, r in zip((x, w, b), which)]
        f8.layer_norm(ts[0], 700, *ts[1:]).backward(dy)
        for t, r, name in zip(ts, which, ("dx", "dw", "db")):
            assert (t.grad is not None) == bool(r) and (not r or torch.equal(t.grad, full[name]))


def test_parameters_of_other_types(f8):
    x, w, b, dy = made(10, 90, FP16, FP32)
    got = run(f8, x, w.to(BF16), b, dy)
    assert got["dw"].dtype == BF16 and got["db"].dtype == FP32
    check(x, w.to(BF16), b, dy, got)


def test_module_compile_stream_and_graph(f8):
    x, w, b, dy = made(40, 256, BF16, BF16)
    model = nn.Sequential(nn.LayerNorm(256), nn.Sequential(nn.LayerNorm(256, bias=False))).to("cuda", BF16)
    params = list(model.parameters())
    f8.convert_layer_norms(model)
    assert type(model[0]) is f8.LayerNorm and type(model[1][0]) is f8.LayerNorm and all(p is q for p, q in zip(params, model.parameters()))
    assert type(f8.convert_layer_norms(nn.LayerNorm(4))) is f8.LayerNorm
    runs = []
    for fn in (f8.layer_norm, torch.compile(f8.layer_norm, fullgraph=True)):
        ts = [t.clone().requires_grad_() for t in (x, w, b)]
        y = fn(ts[0], 256, ts[1], ts[2])
        y.backward(dy)
        runs.append([y] + [t.grad for t in ts])
    assert all(torch.equal(p, q) for p, q in zip(*runs))
    x, w, b = (t.clone().requires_grad_() for t in (x, w, b))

    def step():  # autograd.grad: nothing is left behind that accumulates gradients on the stream it first ran on
        y = f8.layer_norm(x, 256, w, b)
        return (y.detach(),) + torch.autograd.grad(y, (x, w, b), dy)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
        got = step()
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    assert all(torch.equal(p, q) for p, q in zip(got, runs[0]))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = step()
    for i in range(3):
        with torch.no_grad():
            x.copy_(made(40, 256, BF16, BF16, i)[0])
        graph.replay()
        torch.cuda.synchronize()
        recorded = [t.clone() for t in got]
        assert all(torch.equal(p, q) for p, q in zip(recorded, step()))


def test_refusals(f8):
    x, w, b, _ = made(4, 64, BF16, BF16)
    for bad in (lambda: f8.layer_norm(x, 63), lambda: f8.layer_norm(x, ()), lambda: f8.layer_norm(x, 64, w[:63]), lambda: f8.layer_norm(x, 64, w, b.double()),
                lambda: f8.layer_norm(x[:, :0], 0), lambda: f8.layer_norm(x, (2, 4, 64))):
        with pytest.raises(ValueError):
            bad()
    with pytest.raises(TypeError):
        f8.layer_norm(x.double(), 64)
    with pytest.raises(RuntimeError):
        f8.layer_norm(x, 64, w.cpu())
    y = f8.layer_norm(x.requires_grad_(), 64)
    with pytest.raises(RuntimeError, match="second derivative"):
        torch.autograd.grad(y.sum(), x, create_graph=True)
