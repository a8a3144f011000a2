"""RMS norm with and without a residual, forward and backward, and its output in block scales, against the formula in 64 bits and against differences."""
import pytest
import torch
import torch.nn as nn

pytestmark = pytest.mark.gpu

BF16, FP16, FP32 = torch.bfloat16, torch.float16, torch.float32
FP = 2.0**-24  # a rounding of fp32
C = 96 * FP    # a sum over the columns: 64 additions a lane, 6 steps between lanes and 16 between waves at most, the wide rows' ones too


@pytest.fixture(scope="module")
def f8():
    import float8_experimental_amd

    return float8_experimental_amd


def half(dtype):
    return torch.finfo(dtype).eps / 2


def made(rows, cols, dtype, p_dtype, seed=0):
    g = torch.Generator().manual_seed(seed)
    x, r = (torch.randn(rows, cols, generator=g) * torch.randn(cols, generator=g).exp()).to(dtype), torch.randn(rows, cols, generator=g).to(dtype)
    w = (1 + 0.1 * torch.randn(cols, generator=g)).to(p_dtype)
    dy, ds = ((1e-2 * torch.randn(rows, cols, generator=g)).to(dtype) for _ in range(2))
    return [t.cuda() for t in (x, r, w, dy, ds)]


def formula(x, r, w, dy=None, ds=None, eps=1e-6):
    """({name: (value, what fp32 arithmetic may be off by)}, s)"""
    s = (x if r is None else (x.double() + r.double()).to(x.dtype)).detach().double()
    w = torch.ones_like(s[0]) if w is None else w.detach().double()
    rstd = 1 / (s.square().mean(1, keepdim=True) + eps).sqrt()
    xh = s * rstd
    y = xh * w
    # the mean of squares by C of itself, so rstd by C / 2, and five more roundings
    out = {"y": (y, (C + 5 * FP) * y.abs())}
    if r is not None:
        out["s"] = (s, torch.zeros_like(s))
    if dy is not None:
        g = dy.double() * w
        m, size = (g * xh).mean(1, keepdim=True), (g * xh).abs().mean(1, keepdim=True)
        dx = rstd * (g - xh * m)
        off = rstd * ((C + 8 * FP) * g.abs() + xh.abs() * size * 3 * (C + 8 * FP))
        if ds is not None:
            dx, off = dx + ds.double(), off + 4 * FP * ds.double().abs()
        out["dx"] = (dx, off)
        prod = (dy.double() * xh)
        # up to `rows` additions and 64 between groups, workgroups and their sums; xhat off by C / 2 and three roundings
        out["dw"] = (prod.sum(0), ((len(s) + 64) * FP + C + 5 * FP) * prod.abs().sum(0))
    return out, s


def check(got, want):
    for name, value in got.items():
        if value is None:
            continue
        exact, off = want[name]
        tol = half(value.dtype) * exact.abs() + (1 + half(value.dtype)) * off + (2.0**-25 if value.dtype is FP16 else 2.0**-140)
        worst = ((value.detach().double() - exact).abs() / tol).max().item()
        assert worst <= 1.0, (name, worst)


def run(f8, x, r, w, dy, ds, eps=1e-6):
    x, w = x.clone().requires_grad_(), None if w is None else w.clone().requires_grad_()
    if r is None:
        y = f8.rms_norm(x, x.shape[1], w, eps)
        y.backward(dy)
        return {"y": y, "dx": x.grad, "dw": None if w is None else w.grad}
    r = r.clone().requires_grad_()
    y, s = f8.rms_norm(x, x.shape[1], w, eps, residual=r)
    torch.autograd.backward([y, s], [dy, ds])
    assert torch.equal(x.grad.view(torch.uint8), r.grad.view(torch.uint8))  # (the bits: of NaN too)
    return {"y": y, "s": s, "dx": x.grad, "dw": None if w is None else w.grad}


# columns: one, odd, each number of lanes and pieces a row, and rows that do not fit in registers
COLS = [1, 7, 64, 100, 512, 513, 1000, 1024, 2048, 2050, 4096, 4097, 8192, 8200, 12289, 16384, 16390, 20011, 32768, 33001]


@pytest.mark.parametrize("dtype,p_dtype", [(BF16, BF16), (BF16, FP32), (FP16, FP16), (FP16, FP32), (FP32, FP32)])
@pytest.mark.parametrize("cols", COLS)
def test_forward_and_backward(f8, cols, dtype, p_dtype):
    for rows in (1, 3, 70):
        x, r, w, dy, ds = made(rows, cols, dtype, p_dtype, cols + rows)
        check(run(f8, x, r, w, dy, ds), formula(x, r, w, dy, ds)[0])
        check(run(f8, x, None, w, dy, None), formula(x, None, w, dy)[0])


@pytest.mark.parametrize("rows,cols", [(5000, 64), (2500, 1000), (3000, 4096), (1100, 9000), (600, 20000)])
def test_many_rows(f8, rows, cols):
    x, r, w, dy, ds = made(rows, cols, BF16, FP32)
    first = run(f8, x, r, w, dy, ds)
    check(first, formula(x, r, w, dy, ds)[0])
    again = run(f8, x, r, w, dy, ds)  # sums have a fixed order
    assert all(torch.equal(first[k], again[k]) for k in first)


def test_without_a_weight(f8):
    x, r, _, dy, ds = made(20, 300, FP32, FP32)
    check(run(f8, x, r, None, dy, ds), formula(x, r, None, dy, ds)[0])
    check(run(f8, x, None, None, dy, None), formula(x, None, None, dy)[0])


def test_default_eps_is_that_of_torch(f8):
    x = torch.full((2, 64), 1e-3, device="cuda", dtype=BF16)
    want = torch.nn.functional.rms_norm(x.cpu(), (64,)).cuda()
    assert torch.equal(f8.rms_norm(x, 64), want) and torch.equal(f8.RMSNorm(64, device="cuda", dtype=BF16)(x), want)


def test_either_result_alone_has_gradients(f8):
    x, r, w, dy, ds = made(40, 700, BF16, FP32)
    for use in ("y", "s"):
        a, b, p = (t.clone().requires_grad_() for t in (x, r, w))
        y, s = f8.rms_norm(a, 700, p, 1e-6, residual=b)
        if use == "y":
            y.backward(dy)
            check({"dx": a.grad, "dw": p.grad}, formula(x, r, w, dy)[0])
        else:
            s.backward(ds)
            assert torch.equal(a.grad, ds) and p.grad is None
        assert torch.equal(a.grad, b.grad)


def test_only_the_gradients_that_are_asked_for(f8):
    x, r, w, dy, ds = made(33, 700, BF16, BF16)
    full = run(f8, x, r, w, dy, ds)
    for which in ((1, 0, 0), (0, 1, 0), (0, 0, 1), (0, 1, 1), (1, 0, 1)):
        ts = [t.clone().requires_grad_(bool(q)) for t, q in zip((x, r, w), which)]
        y, s = f8.rms_norm(ts[0], 700, ts[2], 1e-6, residual=ts[1])
        torch.autograd.backward([y] + [s] * s.requires_grad, [dy] + [ds] * s.requires_grad)
        for t, q, name in zip(ts, which, ("dx", "dx", "dw")):
            assert (t.grad is not None) == bool(q) and (not q or torch.equal(t.grad, full[name]))


def test_values_that_are_not_finite_stay_in_their_row(f8):
    x, r, w, dy, ds = made(9, 500, BF16, BF16)
    clean = run(f8, x, r, w, dy, ds)
    x[4, 17], x[7, 3] = float("nan"), float("inf")
    got = run(f8, x, r, w, dy, ds)
    assert got["y"][4].isnan().all() and got["dx"][4].isnan().all() and got["y"][7, 3].isnan() and got["dx"][7, 3].isnan()
    for row in (0, 1, 2, 3, 5, 6, 8):
        assert all(torch.equal(got[name][row], clean[name][row]) for name in ("y", "s", "dx"))


def test_zero_rows_and_small_ones(f8):
    x, _, w, dy, _ = made(6, 1000, FP32, FP32)
    x[2] = 0.0
    x[3] *= 1e-25  # squares that fp32 does not hold: eps is all there is
    check(run(f8, x, None, w, dy, None), formula(x, None, w, dy)[0])


def test_strides_and_shapes(f8):
    x, r, w, dy, ds = made(60, 400, BF16, BF16)
    for cut in (lambda t: t[:, 3:260], lambda t: t[::2, :129], lambda t: t[:1, 1:].expand(60, 399)):
        a, b = cut(x), cut(r)
        v = w[:a.shape[1]]
        g, e = dy[:len(a), :a.shape[1]], ds[:len(a), 1:1 + a.shape[1]]
        xs, rs, ws = a.detach().requires_grad_(), b.detach().requires_grad_(), v.clone().requires_grad_()
        y, s = f8.rms_norm(xs, a.shape[1], ws, 1e-6, residual=rs)
        grads = torch.autograd.grad([y, s], [xs, ws], [g, e])
        check({"y": y, "s": s, "dx": grads[0], "dw": grads[1]}, formula(a, b, v, g, e)[0])
    y = f8.rms_norm(x.view(3, 20, 20, 20), (20, 20), w.view(20, 20), 1e-6)
    assert torch.equal(y.view(60, 400), f8.rms_norm(x, 400, w, 1e-6))
    check({"y": f8.rms_norm(x.t(), 60, None, 1e-6)}, formula(x.t(), None, None)[0])
    z = x.clone().requires_grad_()
    f8.rms_norm(z, 400, w).sum().backward()  # a gradient that is one number expanded
    check({"dx": z.grad}, formula(x, None, w, torch.ones_like(x), eps=torch.finfo(FP32).eps)[0])
    assert f8.rms_norm(x[:0], 400, w).shape == (0, 400)


def test_no_rows(f8):
    x, w = torch.zeros((0, 64), device="cuda", requires_grad=True), torch.ones(64, device="cuda", requires_grad=True)
    y, s = f8.rms_norm(x, 64, w, residual=torch.zeros(0, 64, device="cuda"))
    (y.sum() + s.sum()).backward()
    assert x.grad.shape == (0, 64) and (w.grad == 0).all()


def test_gradients_against_differences(f8):
    """Central differences of the formula in 64 bits."""
    x, _, w, dy, _ = made(6, 50, FP32, FP32)
    got = run(f8, x, None, w, dy, None)
    loss = lambda x, w: (x / (x.square().mean(1, keepdim=True) + 1e-6).sqrt() * w * dy.double()).sum().item()
    g, h = torch.Generator().manual_seed(1), 1e-4
    for i, name in enumerate(("dx", "dw")):
        for _ in range(6):
            ts = [t.double() for t in (x, w)]
            at = tuple(int(torch.randint(0, n, (1,), generator=g)) for n in ts[i].shape)
            ts[i][at] += h
            up = loss(*ts)
            ts[i][at] -= 2 * h
            want = (up - loss(*ts)) / (2 * h)
            # differences: h^2 of the third derivative and the roundings of the loss over h
            assert abs(got[name][at].item() - want) <= 1e-5 * abs(want) + 1e-7


def test_weights_of_other_types(f8):
    x, _, w, dy, _ = made(10, 90, FP16, FP32)
    p = w.to(BF16).requires_grad_()
    y = f8.rms_norm(x, 90, p, 1e-6)
    y.backward(dy)
    assert p.grad.dtype == BF16
    check({"y": y, "dw": p.grad}, formula(x, None, p, dy)[0])


# ---- block scales


def exponents(most):
    """S of a block with this largest magnitude (64 bits): the smallest >= -126 with most <= 448 * 2^S"""
    fraction, exponent = torch.frexp(most)
    return (exponent - 9 + (fraction > 0.875)).clamp(min=-126)


def blocks_of(kept):
    """(S of each block [rows, blocks], fp64 values [rows, padded k])"""
    rows = kept.data.shape[1]
    values = kept.data.double().permute(1, 0, 2).reshape(rows, -1)
    order = torch.arange(128, device="cuda")
    bytes_ = kept.scales.view(len(kept.scales), -1, 128)[:, :, order % 16 * 8 + order // 16].reshape(len(kept.scales), -1)[:, :rows].t()
    s = bytes_.long() - 127
    return s, values * torch.exp2(s.double()).repeat_interleave(128, 1)


def check_kept(kept, y):
    """Each value is e4m3's nearest to y / 2^S but for fp32's arithmetic, S the smallest but for a maximum on its border; zeros fill the last block up."""
    rows, cols = y.shape
    s, values = blocks_of(kept)
    padded = torch.nn.functional.pad(y, (0, values.shape[1] - cols)).view(rows, -1, 128)
    most, off = padded.abs().amax(2), C + 5 * FP
    assert ((exponents(most * (1 - off)) <= s) & (s <= exponents(most * (1 + off)))).all()
    assert (values[:, cols:] == 0).all()
    step = torch.exp2(s.double()).repeat_interleave(128, 1)[:, :cols] * 2.0**-9  # of the subnormals
    tol = torch.maximum(2.0**-4 * y.abs(), step / 2) + 2 * off * y.abs()
    assert ((values[:, :cols] - y).abs() <= tol).all()


@pytest.mark.parametrize("dtype,p_dtype", [(BF16, BF16), (BF16, FP32), (FP16, FP16), (FP32, FP32)])
@pytest.mark.parametrize("cols", [1, 100, 128, 512, 700, 1000, 4096, 4097, 8192, 10000, 16384, 24576, 24600, 33001])
def test_block_scales(f8, cols, dtype, p_dtype):
    for rows in (1, 5, 130):
        x, r, w, _, _ = made(rows, cols, dtype, p_dtype, cols + rows)
        x[:, cols // 2:] *= 2.0**-9  # blocks of different sizes
        kept, s = f8.rms_norm_blockwise(x, cols, w, 1e-6, residual=r)
        want, sums = formula(x, r, w)
        assert torch.equal(s.double(), sums) and kept.shape == (rows, cols) and kept.dtype == dtype
        check_kept(kept, want["y"][0])
        check_kept(f8.rms_norm_blockwise(x, cols, None, 1e-6), formula(x, None, None)[0]["y"][0])
        assert torch.equal(kept.dequantized().double(), blocks_of(kept)[1][:, :cols])


def test_block_scales_of_small_and_broken_rows(f8):
    x, _, w, _, _ = made(8, 300, BF16, BF16)
    x[1] = 0.0
    x[2, 5] = float("nan")
    x[3, 140] = float("inf")
    x[4, :128] = 0.0
    kept = f8.rms_norm_blockwise(x, 300, w, 1e-6)
    values = kept.dequantized()
    assert (values[1] == 0).all() and values[2].isnan().all() and values[3, 128:256].isnan().all() and (values[4, :128] == 0).all()
    ok = [0, 4, 5, 6, 7]
    assert torch.equal(values[ok], f8.rms_norm_blockwise(x[ok], 300, w, 1e-6).dequantized())


@pytest.mark.parametrize("rows", [1, 16, 17, 300])
@pytest.mark.parametrize("k,n", [(256, 128), (1000, 333), (4096, 1024)])
def test_served_linears_take_the_kept_values(f8, rows, k, n):
    x, r, w, _, _ = made(rows, k, BF16, BF16, rows)
    g = torch.Generator().manual_seed(1)
    lin = nn.Linear(k, n, device="cuda", dtype=BF16)
    with torch.no_grad():
        lin.weight.copy_((torch.randn(n, k, generator=g) / k**0.5).cuda())
    served = f8.Float8BlockwiseInferenceLinear.from_float(lin)
    with torch.no_grad():
        kept, _ = f8.rms_norm_blockwise(x.view(rows, 1, k), k, w, 1e-6, residual=r.view(rows, 1, k))
        y = served(kept)
    a, b = kept.dequantized().double().view(rows, k), served.dequantized_weight().double()
    want, size = a @ b.t() + lin.bias.double(), a.abs() @ b.abs().t()
    # eight products cut to 2^-13 of the largest, k / 8 additions, one rounding
    tol = half(BF16) * want.abs() + (8 * 2.0**-13 + (k / 8 + 16) * FP) * size + FP * lin.bias.double().abs()
    assert y.shape == (rows, 1, n) and y.dtype == BF16 and ((y.view(rows, n).double() - want).abs() <= tol).all()


def test_block_scales_refuse_gradients_and_other_linears(f8):
    x, r, w, _, _ = made(4, 256, BF16, BF16)
    with pytest.raises(RuntimeError, match="no backward"):
        f8.rms_norm_blockwise(x, 256, w.requires_grad_())
    served = f8.Float8BlockwiseInferenceLinear.from_float(nn.Linear(128, 64, device="cuda", dtype=BF16))
    with torch.no_grad():
        kept = f8.rms_norm_blockwise(x, 256, w)
        with pytest.raises(ValueError, match="in_features"):
            served(kept)
        with pytest.raises(ValueError, match="last dimension"):
            f8.rms_norm_blockwise(x.view(4, 2, 128), (2, 128))
        assert f8.rms_norm_blockwise(x[:0], 256, w).data.shape == (4, 0, 64)
        assert f8.Float8BlockwiseInferenceLinear.from_float(nn.Linear(256, 64, device="cuda", dtype=BF16))(f8.rms_norm_blockwise(x[:0], 256, w)).shape == (0, 64)


# ---- modules, compilers, streams and graphs


def test_module_compile_stream_and_graph(f8):
    x, r, w, dy, ds = made(40, 256, BF16, BF16)
    model = nn.Sequential(nn.RMSNorm(256, eps=1e-6), nn.Sequential(nn.RMSNorm(256, elementwise_affine=False))).to("cuda", BF16)
    params = list(model.parameters())
    f8.convert_rms_norms(model)
    assert type(model[0]) is f8.RMSNorm and type(model[1][0]) is f8.RMSNorm and all(p is q for p, q in zip(params, model.parameters())) and model[0].eps == 1e-6
    assert type(f8.convert_rms_norms(nn.RMSNorm(4))) is f8.RMSNorm and torch.equal(model[0](x), f8.rms_norm(x, 256, params[0], 1e-6))
    runs = []
    for fn in (f8.rms_norm, torch.compile(f8.rms_norm, fullgraph=True, backend="aot_eager")):
        ts = [t.clone().requires_grad_() for t in (x, w, r)]
        y, s = fn(ts[0], 256, ts[1], 1e-6, ts[2])
        torch.autograd.backward([y, s], [dy, ds])
        alone = [t.clone().requires_grad_() for t in (x, w)]
        z = fn(alone[0], 256, alone[1])
        z.backward(dy)
        runs.append([y, s, z] + [t.grad for t in ts + alone])
    assert all(torch.equal(p, q) for p, q in zip(*runs))
    with torch.no_grad():
        kept = [fn(x, 256, w, 1e-6, r) for fn in (f8.rms_norm_blockwise, torch.compile(f8.rms_norm_blockwise, fullgraph=True, backend="aot_eager"))]
    assert torch.equal(kept[0][1], kept[1][1]) and torch.equal(kept[0][0].dequantized(), kept[1][0].dequantized())
    x, w, r = (t.clone().requires_grad_() for t in (x, w, r))

    def step():  # autograd.grad: nothing is left behind that accumulates gradients on the stream it first ran on
        y, s = f8.rms_norm(x, 256, w, 1e-6, r)
        return (y.detach(), s.detach()) + torch.autograd.grad([y, s], (x, w), [dy, ds])

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
        got = step()
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    assert all(torch.equal(p, q) for p, q in zip(got, runs[0][:2] + runs[0][3:5]))
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
    x, r, w, _, _ = made(4, 64, BF16, BF16)
    for bad in (lambda: f8.rms_norm(x, 63), lambda: f8.rms_norm(x, ()), lambda: f8.rms_norm(x, 64, w[:63]), lambda: f8.rms_norm(x, 64, w.double()), lambda: f8.rms_norm(x[:, :0], 0),
                lambda: f8.rms_norm(x, (2, 4, 64)), lambda: f8.rms_norm(x, (4, 64), w), lambda: f8.rms_norm(x, 64, residual=r[:3]), lambda: f8.rms_norm(x, 64, residual=r.float())):
        with pytest.raises(ValueError):
            bad()
    with pytest.raises(TypeError):
        f8.rms_norm(x.double(), 64)
    for bad in (lambda: f8.rms_norm(x, 64, w.cpu()), lambda: f8.rms_norm(x, 64, w, residual=r.cpu())):
        with pytest.raises(RuntimeError):
            bad()
    y = f8.rms_norm(x.requires_grad_(), 64)
    with pytest.raises(RuntimeError, match="second derivative"):
        torch.autograd.grad(y.sum(), x, create_graph=True)
