"""Low-rank adapters of many requests beside one projection, forward and backward, against the formula in 64 bits and against differences."""
import pytest
import torch
import torch.nn as nn

pytestmark = pytest.mark.gpu
BF16, FP16, FP32 = torch.bfloat16, torch.float16, torch.float32
FP = 2.0**-24  # a rounding of fp32


@pytest.fixture(scope="module")
def f8():
    import float8_experimental_amd

    return float8_experimental_amd


def made(m, k, n, r, count, dtype, seed=0, p_dtype=None):
    g = torch.Generator().manual_seed(seed)
    x, y = (torch.randn(m, k, generator=g) * torch.randn(k, generator=g).exp()).to(dtype), torch.randn(m, n, generator=g).to(dtype)
    a, b = (torch.randn(count, r, k, generator=g) / k**0.5).to(p_dtype or dtype), (torch.randn(count, n, r, generator=g) / r**0.5).to(p_dtype or dtype)
    return [t.cuda() for t in (x, a, b, y, (1 + 0.1 * torch.randn(count, generator=g)), (1e-2 * torch.randn(m, n, generator=g)).to(dtype))]


def formula(x, a, b, ids, y, scale, dout=None):
    """{name: (value, what fp32 arithmetic and h in two 16-bit parts may be off by)}"""
    (m, k), (count, r, _), n = x.shape, a.shape, b.shape[1]
    dtype, x = x.dtype, x.detach().double()
    ad, bd = (t.detach().to(dtype).double() for t in (a, b))
    z = lambda *s: torch.zeros(s, dtype=torch.float64, device="cuda")
    out = z(m, n) if y is None else y.detach().double()
    off = FP * out.abs()
    g = {"dx": z(m, k), "da": z(*a.shape), "db": z(*b.shape)}
    goff = {name: torch.zeros_like(v) for name, v in g.items()}

    def kept(h, h_off):  # in two 16-bit parts: 2^-16 of itself, fp16 also 2^-24 of the row's largest
        return h_off + (0 if dtype is FP32 else 2.0**-16 * h.abs()) + (2.0**-23 * h.abs().amax(1, keepdim=True) if dtype is FP16 and len(h) else 0)

    for e in range(count):
        at = (ids == e).nonzero().flatten()
        f = float(scale[e]) if isinstance(scale, torch.Tensor) else scale
        xe = x[at]
        h, h_off = xe @ ad[e].t(), (k + 40) * FP * (xe.abs() @ ad[e].abs().t())
        size = h.abs() @ bd[e].abs().t()
        out[at] += f * (h @ bd[e].t())
        off[at] += abs(f) * (kept(h, h_off) @ bd[e].abs().t() + (2 * r + 16) * FP * size) + FP * out[at].abs()
        if dout is not None:
            ge = dout[at].double()
            dh, dh_off = ge @ bd[e], (n + 40) * FP * (ge.abs() @ bd[e].abs())
            g["dx"][at] = f * (dh @ ad[e])
            goff["dx"][at] = abs(f) * (kept(dh, dh_off) @ ad[e].abs() + (2 * r + 16) * FP * (dh.abs() @ ad[e].abs()))
            rows = (len(at) + 40) * FP
            g["da"][e], g["db"][e] = f * (dh.t() @ xe), f * (ge.t() @ h)
            # (the gradients' products may take dh and h in two parts as well)
            goff["da"][e] = abs(f) * (kept(dh, dh_off).t() @ xe.abs() + rows * (dh.abs().t() @ xe.abs()))
            goff["db"][e] = abs(f) * (ge.abs().t() @ kept(h, h_off) + rows * (ge.abs().t() @ h.abs()))
    result = {"out": (out, off)}
    if dout is not None:
        result.update({name: (g[name], goff[name]) for name in g})
    return result


def check(got, want):
    for name, value in got.items():
        exact, off = want[name]
        half = torch.finfo(value.dtype).eps / 2
        tol = half * exact.abs() + (1 + half) * off + (2.0**-25 if value.dtype is FP16 else 2.0**-140)
        worst = ((value.detach().double() - exact).abs() / tol).max().item()
        assert value.isfinite().all() and worst <= 1.0, (name, worst)


def run(f8, x, a, b, rows, y, scale, dout):
    x, a, b = (t.clone().requires_grad_() for t in (x, a, b))
    out = f8.low_rank_adapters(x, a, b, rows, y, scale)
    out.backward(dout)
    return {"out": out, "dx": x.grad, "da": a.grad, "db": b.grad}


def whose(kind, m, count, seed=0):
    g = torch.Generator().manual_seed(seed)
    if kind == "any":
        ids = torch.randint(-1, count, (m,), generator=g)
    elif kind == "runs":  # of a request each, some without an adapter
        ids = (torch.randint(0, 5, (m,), generator=g).eq(0).cumsum(0) * 7) % (count + 1) - 1
    elif kind == "one":
        ids = torch.full((m,), count - 1)
    else:
        ids = torch.full((m,), -1)
    return ids.cuda()


SHAPES = [  # m, k, n, rank, count
    (1, 64, 64, 8, 1), (1, 1000, 333, 16, 5), (3, 4096, 1024, 4, 64), (17, 129, 65, 1, 3), (40, 500, 260, 12, 7), (64, 2048, 2048, 16, 64), (100, 96, 40, 33, 2), (130, 130, 515, 64, 2),
    (300, 257, 129, 16, 3), (513, 640, 384, 48, 4), (700, 100, 1030, 128, 5), (1000, 72, 200, 256, 2), (2500, 320, 96, 16, 1), (70, 8, 8, 100, 4), (90, 1, 1, 2, 3), (5, 16384, 17, 7, 2),
]


@pytest.mark.parametrize("dtype", [BF16, FP16, FP32])
@pytest.mark.parametrize("shape", SHAPES, ids=lambda s: "x".join(map(str, s)))
def test_forward_and_backward(f8, shape, dtype):
    m, k, n, r, count = shape
    for kind in ("any", "runs"):
        x, a, b, y, scale, dout = made(m, k, n, r, count, dtype, m + k)
        ids = whose(kind, m, count, n)
        got = run(f8, x, a, b, f8.AdapterRows(ids, count), y, scale, dout)
        check(got, formula(x, a, b, ids, y, scale, dout))
        again = run(f8, x, a, b, f8.AdapterRows(ids, count), y, scale, dout)  # sums have a fixed order
        assert all(torch.equal(got[name], again[name]) for name in got)


FEW = [  # on both sides of what goes in one launch: the length of the contractions, the number of columns, the rank, the workgroups
    (1, 4096, 513, 8, 3), (1, 4097, 513, 8, 3), (5, 2048, 1100, 5, 2), (5, 2056, 4096, 16, 2), (20, 300, 512, 16, 20), (20, 300, 63, 16, 20), (20, 63, 300, 16, 20), (20, 300, 64, 17, 20),
    (16, 64, 7000, 16, 64), (16, 64, 9000, 16, 64), (33, 1, 64, 1, 40),
]


@pytest.mark.parametrize("dtype", [BF16, FP16, FP32])
@pytest.mark.parametrize("shape", FEW, ids=lambda s: "x".join(map(str, s)))
def test_few_rows_in_one_launch_and_in_two(f8, shape, dtype):
    m, k, n, r, count = shape
    x, a, b, y, scale, dout = made(m, k, n, r, count, dtype, m + n)
    ids = whose("any", m, count, k)
    rows, want = f8.AdapterRows(ids, count), formula(x, a, b, ids, y, scale, dout)
    got = run(f8, x, a, b, rows, y, scale, dout)
    check(got, want)
    assert torch.equal(got["out"], f8.low_rank_adapters(x, a, b, rows, y, scale))  # (without h kept for backward)
    for name, t in (("dx", x), ("da", a), ("db", b)):  # each gradient alone, the same bits
        leaf = t.clone().requires_grad_()
        f8.low_rank_adapters(*(leaf if u is t else u for u in (x, a, b)), rows, y, scale).backward(dout)
        assert torch.equal(leaf.grad, got[name]), name


@pytest.mark.parametrize("kind", ["one", "none"])
@pytest.mark.parametrize("m", [1, 16, 200])
def test_all_rows_of_one_adapter_and_of_none(f8, kind, m):
    x, a, b, y, _, dout = made(m, 200, 120, 16, 3, BF16)
    y[0, 0] = -0.0
    ids = whose(kind, m, 3)
    got = run(f8, x, a, b, f8.AdapterRows(ids, 3), y, 0.5, dout)
    check(got, formula(x, a, b, ids, y, 0.5, dout))
    unused = slice(0, 2) if kind == "one" else slice(0, 3)
    assert (got["da"][unused] == 0).all() and (got["db"][unused] == 0).all()
    if kind == "none":
        assert torch.equal(got["out"].view(torch.int16), y.view(torch.int16)) and (got["dx"] == 0).all()


def test_numbers_of_no_adapter_and_of_other_types(f8):
    x, a, b, y, _, _ = made(40, 100, 60, 8, 4, BF16)
    ids = torch.randint(0, 4, (40,), generator=torch.Generator().manual_seed(1)).cuda()
    want = f8.low_rank_adapters(x, a, b, f8.AdapterRows(ids, 4), y)
    for dtype in (torch.int32, torch.int16, torch.int8, torch.uint8):
        assert torch.equal(f8.low_rank_adapters(x, a, b, ids.to(dtype), y), want)
    for none in (4, 1000, -7, 2**40, -(2**62)):
        other = ids.clone()
        other[::3] = none
        got = f8.low_rank_adapters(x, a, b, other, y)
        assert torch.equal(got[::3], y[::3]) and torch.equal(got[1::3], want[1::3])


def test_the_table_lists_every_row_once(f8):
    from float8_experimental_amd import _native

    for m, count in ((1, 1), (63, 3), (5000, 17), (300, 500), (70000, 2)):
        ids = torch.randint(-1, count, (m,), generator=torch.Generator().manual_seed(m)).cuda()
        words = f8.AdapterRows(ids, count).table.cpu()
        up4 = lambda v: (v + 3) // 4 * 4
        groups = count + 1
        at = up4(groups) + up4(groups + 1)
        order = words[at:at + m].long()
        want = torch.where(ids < 0, count, ids).cpu()
        assert torch.equal(order, torch.sort(want, stable=True).indices)
        at += up4(m)
        chunk = 64
        while chunk < 512 and chunk * 32 < m:
            chunk *= 2
        for height in (16, 64, chunk):
            tiles = words[at:at + 4 * (m // height + min(groups, m))].view(-1, 4)
            at += tiles.numel()
            tiles = tiles[tiles[:, 2] > 0]
            counts = torch.bincount(want, minlength=groups)
            assert len(tiles) == ((counts + height - 1) // height).sum() and (tiles[:, 2] <= height).all()
            assert torch.equal(torch.cat([order[f:f + c] for _, f, c, _ in tiles.tolist()]), order) and all((want[order[f:f + c]] == g).all() for g, f, c, _ in tiles.tolist())
        assert at == len(words) == _native.lib().f8mi_adapter_rows_words(m, count)


def test_without_a_projection_and_with_numbers_for_scale(f8):
    x, a, b, y, _, dout = made(50, 100, 70, 8, 3, BF16)
    ids = whose("any", 50, 3)
    for scale in (1.0, 0, -2.5):
        check(run(f8, x, a, b, f8.AdapterRows(ids, 3), None, scale, dout), formula(x, a, b, ids, None, scale, dout))
    out = f8.low_rank_adapters(x, a, b, ids, None)
    assert (out[ids < 0] == 0).all()


def test_adapters_of_other_types(f8):
    for dtype, p_dtype in ((BF16, FP32), (FP16, FP32), (FP32, BF16)):
        x, a, b, y, scale, dout = made(60, 90, 70, 8, 3, dtype, 3, p_dtype)
        ids = whose("any", 60, 3)
        got = run(f8, x, a, b, f8.AdapterRows(ids, 3), y, scale, dout)
        assert got["da"].dtype == got["db"].dtype == p_dtype and got["dx"].dtype == dtype
        check(got, formula(x, a, b, ids, y, scale, dout))
    x, a, b, y, scale, dout = made(60, 90, 70, 8, 3, BF16, 3)
    got = run(f8, x, a, b.float(), f8.AdapterRows(ids, 3), y, scale.bfloat16(), dout)
    assert got["da"].dtype == BF16 and got["db"].dtype == FP32
    check(got, formula(x, a, b, ids, y, scale.bfloat16(), dout))


def test_fp16_keeps_small_and_large_inner_values(f8):
    """h beyond fp16's largest value and below its subnormals: kept after a power of two for each row."""
    x, a, b, y, _, dout = made(40, 256, 128, 16, 2, FP16)
    ids = whose("any", 40, 2)
    x *= torch.logspace(-3, 3, 40, device="cuda")[:, None].half()
    a *= 50
    b *= 2.0**-14
    y *= 0.01
    assert (x.double() @ a[0].double().t()).abs().max() > 1e5
    check(run(f8, x, a, b, f8.AdapterRows(ids, 2), y, 1.0, dout * 2.0**-4), formula(x, a, b, ids, y, 1.0, dout * 2.0**-4))


def test_values_that_are_not_finite_stay_in_their_row(f8):
    x, a, b, y, _, dout = made(40, 300, 130, 12, 2, BF16)
    ids = torch.arange(40, device="cuda") % 3 - 1
    clean = f8.low_rank_adapters(x, a, b, ids, y)
    x[3, 299], x[10, 0], x[7, 5], y[5, 1] = float("nan"), float("inf"), float("inf"), float("nan")
    b[ids[7]][b[ids[7]] == 0] = 1.0
    assert ids[3] < 0
    got = f8.low_rank_adapters(x, a, b, ids, y)
    assert torch.equal(got[3], clean[3]) and not got[10].isfinite().any() and got[5, 1].isnan()
    rest = [i for i in range(40) if i not in (3, 5, 7, 10)]
    assert torch.equal(got[rest], clean[rest])


def test_strides_and_shapes(f8):
    x, a, b, y, scale, dout = made(60, 400, 300, 16, 3, BF16)
    ids = whose("any", 60, 3)
    for cut in (slice(3, 260), slice(1, 258)):
        xs, ys, gs, aa, bb = x[:, cut], y[:, cut], dout[:, cut], a[:, :, cut], b[:, cut]
        v = xs.detach().requires_grad_()
        p, q = aa.detach().requires_grad_(), bb.detach().requires_grad_()
        out = f8.low_rank_adapters(v, p, q, ids, ys, scale)
        grads = torch.autograd.grad(out, (v, p, q), gs)
        check(dict(zip(("out", "dx", "da", "db"), (out, *grads))), formula(xs, aa, bb, ids, ys, scale, gs))
    half = f8.low_rank_adapters(x[::2], a, b, ids[::2], y[::2], scale)
    check({"out": half}, formula(x[::2], a, b, ids[::2], y[::2], scale))
    same = f8.low_rank_adapters(x[:1].expand(60, 400), a, b, ids, y[:1].expand(60, 300), scale)
    check({"out": same}, formula(x[:1].expand(60, 400), a, b, ids, y[:1].expand(60, 300), scale))
    three = f8.low_rank_adapters(x.view(3, 20, 400), a, b, ids.view(3, 20), y.view(3, 20, 300), scale)
    assert three.shape == (3, 20, 300) and torch.equal(three.view(60, 300), f8.low_rank_adapters(x, a, b, ids, y, scale))
    v = x.clone().requires_grad_()
    f8.low_rank_adapters(v, a, b, ids, y, scale).sum().backward()  # a gradient that is one number expanded
    check({"dx": v.grad}, {"dx": formula(x, a, b, ids, y, scale, torch.ones_like(dout))["dx"]})


def test_no_rows(f8):
    x, a, b, y, scale, dout = made(0, 64, 32, 8, 2, BF16)
    got = run(f8, x, a, b, f8.AdapterRows(torch.zeros(0, dtype=torch.int64, device="cuda"), 2), y, scale, dout)
    assert got["out"].shape == (0, 32) and got["dx"].shape == (0, 64) and (got["da"] == 0).all() and (got["db"] == 0).all() and got["da"].shape == a.shape and got["db"].shape == b.shape


def test_only_the_gradients_that_are_asked_for(f8):
    x, a, b, y, scale, dout = made(90, 130, 70, 16, 3, BF16)
    rows = f8.AdapterRows(whose("runs", 90, 3), 3)
    full = run(f8, x, a, b, rows, y, scale, dout)
    full["dy"] = dout
    for which in ((1, 0, 0, 0), (0, 1, 0, 0), (0, 0, 1, 0), (0, 0, 0, 1), (0, 1, 1, 0), (1, 0, 1, 1)):
        ts = [t.clone().requires_grad_(bool(q)) for t, q in zip((x, a, b, y), which)]
        f8.low_rank_adapters(ts[0], ts[1], ts[2], rows, ts[3], scale).backward(dout)
        for t, q, name in zip(ts, which, ("dx", "da", "db", "dy")):
            assert (t.grad is not None) == bool(q) and (not q or torch.equal(t.grad, full[name]))


def test_gradients_against_differences(f8):
    """Central differences of the formula in 64 bits."""
    x, a, b, y, _, dout = made(12, 30, 20, 5, 2, FP32)
    ids = whose("any", 12, 2)
    got = run(f8, x, a, b, f8.AdapterRows(ids, 2), y, 0.7, dout)
    at_e = ids.clamp(min=0)

    def loss(x, a, b):
        h = (a[at_e] @ x[:, :, None])
        return (0.7 * (b[at_e] @ h)[:, :, 0] * (ids >= 0)[:, None] * dout.double()).sum().item()

    g, h = torch.Generator().manual_seed(1), 1e-4
    for i, name in enumerate(("dx", "da", "db")):
        for _ in range(8):
            ts = [t.double() for t in (x, a, b)]
            at = tuple(int(torch.randint(0, s, (1,), generator=g)) for s in ts[i].shape)
            ts[i][at] += h
            up = loss(*ts)
            ts[i][at] -= 2 * h
            want = (up - loss(*ts)) / (2 * h)
            # the loss is linear in each factor: the roundings of the loss over h, and fp32's in what is compared
            assert abs(got[name][at].item() - want) <= 1e-5 * abs(want) + 1e-7


def test_offsets_that_pass_32_bits(f8):
    """The last rows have the values that they have by themselves, and gradients of far rows arrive."""
    m, k, n = 600_000, 4096, 64
    x = torch.zeros(m, k, device="cuda", dtype=BF16)
    _, a, b, _, _, _ = made(1, k, n, 8, 2, BF16)
    tail = made(200, k, n, 8, 2, BF16)
    x[-200:] = tail[0]
    ids = torch.zeros(m, dtype=torch.int64, device="cuda")
    ids[-100:] = 1
    dout = torch.zeros(m, n, device="cuda", dtype=BF16)
    dout[-200:] = tail[5]
    got = run(f8, x, a, b, f8.AdapterRows(ids, 2), None, 1.0, dout)
    want = formula(tail[0], a, b, ids[-200:], None, 1.0, tail[5])
    check({"out": got["out"][-200:], "dx": got["dx"][-200:], "da": got["da"], "db": got["db"]}, want)
    assert (got["out"][:-200] == 0).all() and (got["dx"][:-200] == 0).all()


def test_compile_streams_and_graphs(f8):
    x, a, b, y, scale, dout = made(90, 256, 128, 16, 3, BF16)
    ids = whose("runs", 90, 3)
    rows = f8.AdapterRows(ids, 3)
    runs = []
    for fn in (f8.low_rank_adapters, torch.compile(lambda *t: f8.low_rank_adapters(*t), fullgraph=True, backend="aot_eager")):
        for which in (rows, ids):
            ts = [t.clone().requires_grad_() for t in (x, a, b)]
            out = fn(*ts, which, y, scale)
            out.backward(dout)
            runs.append([out] + [t.grad for t in ts])
    assert all(torch.equal(p, q) for other in runs[1:] for p, q in zip(runs[0], other))
    x, a, b = (t.clone().requires_grad_() for t in (x, a, b))

    def step():
        out = f8.low_rank_adapters(x, a, b, f8.AdapterRows(ids, 3), y, scale)
        return (out.detach(),) + torch.autograd.grad(out, (x, a, b), dout)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
        got = step()
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    assert all(torch.equal(p, q) for p, q in zip(got, runs[0]))
    graphs, outs = [torch.cuda.CUDAGraph(), torch.cuda.CUDAGraph()], []
    for graph in graphs:  # two of them in one pool
        with torch.cuda.graph(graph, pool=graphs[0].pool() if outs else None):
            outs.append(step())
    for i in range(3):
        ids.copy_(whose("any", 90, 3, i))  # the rows are sorted at each replay
        with torch.no_grad():
            x.copy_(made(90, 256, 128, 16, 3, BF16, i)[0])
        want = step()
        for graph, out in zip(graphs, outs):
            graph.replay()
            torch.cuda.synchronize()
            assert all(torch.equal(p, q) for p, q in zip([t.clone() for t in out], want))


def test_refusals(f8):
    x, a, b, y, scale, dout = made(8, 64, 32, 4, 2, BF16)
    rows = f8.AdapterRows(torch.zeros(8, dtype=torch.int64, device="cuda"), 2)
    for bad in (lambda: f8.low_rank_adapters(x[:7], a, b, rows, y[:7]), lambda: f8.low_rank_adapters(x[:, :60], a, b, rows, y), lambda: f8.low_rank_adapters(x, a[:1], b, rows, y),
                lambda: f8.low_rank_adapters(x, a, b[:, :, :3], rows, y), lambda: f8.low_rank_adapters(x, a, b, rows, y[:, :31]), lambda: f8.low_rank_adapters(x, a, b, rows, y.float()),
                lambda: f8.low_rank_adapters(x, a[:1], b[:1], rows, y), lambda: f8.low_rank_adapters(x, a, b, rows, y, scale[:1]), lambda: f8.AdapterRows(torch.zeros(3, dtype=torch.int64, device="cuda"), 0),
                lambda: f8.AdapterRows(torch.zeros(3, dtype=torch.int64, device="cuda"), 40000),
                lambda: f8.low_rank_adapters(x, torch.ones(2, 300, 64, device="cuda", dtype=BF16), torch.ones(2, 32, 300, device="cuda", dtype=BF16), rows, y)):
        with pytest.raises(ValueError):
            bad()
    for bad in (lambda: f8.low_rank_adapters(x.double(), a, b, rows), lambda: f8.low_rank_adapters(x, a.double(), b.double(), rows), lambda: f8.AdapterRows(torch.zeros(3, device="cuda"), 2)):
        with pytest.raises(TypeError):
            bad()
    for bad in (lambda: f8.low_rank_adapters(x, a.cpu(), b, rows), lambda: f8.AdapterRows(torch.zeros(3, dtype=torch.int64), 2)):
        with pytest.raises(RuntimeError):
            bad()
    with pytest.raises(NotImplementedError):
        f8.low_rank_adapters(x, a, b, rows, y, scale.clone().requires_grad_())
    out = f8.low_rank_adapters(x.requires_grad_(), a, b, rows, y)
    with pytest.raises(RuntimeError, match="second derivative"):
        torch.autograd.grad(out.sum(), x, create_graph=True)


# ---- modules


def test_adapted_linears_of_every_kind(f8):
    """Beside each kind of linear: what the linear gives plus what the adapters add, gradients of the adapters alone, and of what is in front where the linear has a backward pass."""
    from float8_experimental_amd.inference import ActivationCasting, QuantConfig, quantize_to_float8

    blk = f8.CastConfig(scaling_type=f8.ScalingType.BLOCKWISE)
    blockwise = f8.Float8LinearConfig(cast_config_input=blk, cast_config_weight=blk, cast_config_grad_output=blk)
    kinds = {"plain": lambda m: m, "float8": f8.convert_to_float8_training, "blockwise": lambda m: f8.convert_to_float8_training(m, config=blockwise),
             "served": lambda m: quantize_to_float8(m, QuantConfig(ActivationCasting.DYNAMIC)), "served blockwise": lambda m: quantize_to_float8(m, QuantConfig(ActivationCasting.BLOCKWISE))}
    x, ids = torch.randn(40, 256, device="cuda", dtype=BF16), whose("any", 40, 3)
    for name, make in kinds.items():
        torch.manual_seed(0)
        base = make(nn.Sequential(nn.Linear(256, 128)).to("cuda", BF16))
        model = f8.adapt_linears(base, 3, 8, alpha=16)
        layer = model[0]
        assert type(layer) is f8.AdaptedLinear and [n for n, p in model.named_parameters() if p.requires_grad] == ["0.adapter_a", "0.adapter_b"] and layer.adapter_a.dtype == BF16
        with torch.no_grad():
            plain = layer.linear(x)
            assert torch.equal(model(x), plain)  # no rows have one
            rows = f8.select_adapters(model, ids)
            assert torch.equal(model(x), plain)  # b is zero
            layer.adapter_b.normal_()
            got = model(x)
            assert torch.equal(got, f8.low_rank_adapters(x, layer.adapter_a, layer.adapter_b, rows, plain, 2.0)) and not torch.equal(got, plain)
            f8.select_adapters(model, None)
            assert torch.equal(model(x), plain)
        if not name.startswith("served"):
            f8.select_adapters(model, rows)
            v = x.clone().requires_grad_()
            model(v).square().sum().backward()
            assert all(t.grad is not None and t.grad.isfinite().all() and t.grad.abs().max() > 0 for t in (v, layer.adapter_a, layer.adapter_b))
    with pytest.raises(ValueError):
        f8.select_adapters(model, f8.AdapterRows(ids, 4))
    with pytest.raises(ValueError):
        f8.select_adapters(nn.Linear(2, 2), ids)
    with pytest.raises(ValueError):
        f8.AdaptedLinear(nn.Linear(4, 4, device="cuda"), 2, 1000)


def test_adapted_models_are_served_quantised_afterwards(f8):
    """Adapters first, then the shared weights in block scales: the adapters stay as they are."""
    from float8_experimental_amd.inference import ActivationCasting, QuantConfig, quantize_to_float8

    torch.manual_seed(0)
    model = f8.adapt_linears(nn.Sequential(nn.Linear(256, 384), nn.SiLU(), nn.Linear(384, 128)).to("cuda", BF16), 2, 8, module_filter_fn=lambda m, fqn: fqn != "2")
    served = quantize_to_float8(model, QuantConfig(ActivationCasting.BLOCKWISE))
    assert type(served[0]) is f8.AdaptedLinear and type(served[0].linear) is f8.Float8BlockwiseInferenceLinear and type(served[2]) is f8.Float8BlockwiseInferenceLinear
    f8.select_adapters(served, torch.tensor([0, 1, -1], device="cuda"))
    with torch.no_grad():
        served[0].adapter_b.normal_()
        x = torch.randn(3, 256, device="cuda", dtype=BF16)
        y = served(x)
    assert y.isfinite().all() and set(served.state_dict()) == {"0.adapter_a", "0.adapter_b", "0.linear.weight_data", "0.linear.weight_scales", "0.linear.bias", "2.weight_data", "2.weight_scales", "2.bias"}


def test_dropout_of_the_adapters_input(f8):
    torch.manual_seed(0)
    layer = f8.AdaptedLinear(nn.Linear(64, 32, device="cuda", dtype=BF16), 2, 4, dropout=0.5)
    rows, x = f8.select_adapters(layer, torch.zeros(10, dtype=torch.int64, device="cuda")), torch.randn(10, 64, device="cuda", dtype=BF16)
    with torch.no_grad():
        layer.adapter_b.normal_()
        torch.manual_seed(5)
        got = layer.train()(x)
        torch.manual_seed(5)
        want = f8.low_rank_adapters(f8.dropout(x, 0.5), layer.adapter_a, layer.adapter_b, rows, layer.linear(x))
        assert torch.equal(got, want) and not torch.equal(got, layer(x))
        assert torch.equal(layer.eval()(x), layer(x))


# ---- a run of the operators together


class Block(nn.Module):
    """The residual goes along: norm and addition are one operator."""

    def __init__(self, dim, hidden):
        super().__init__()
        self.norm, self.up, self.down, self.drop = nn.RMSNorm(dim, eps=1e-6), nn.Linear(dim, hidden, bias=False), nn.Linear(hidden, dim, bias=False), nn.Dropout(0.1)

    def forward(self, branch, stream):
        normed, stream = self.norm(branch, residual=stream)
        return self.drop(self.down(nn.functional.silu(self.up(normed)))), stream


class Model(nn.Module):
    def __init__(self, dim, hidden, layers):
        super().__init__()
        self.blocks, self.norm = nn.ModuleList([Block(dim, hidden) for _ in range(layers)]), nn.RMSNorm(dim, eps=1e-6)

    def forward(self, x):
        branch, stream = torch.zeros_like(x), x
        for block in self.blocks:
            branch, stream = block(branch, stream)
        return self.norm(branch, residual=stream)[0]


def reference(model, x, ids, seeds, keeps):
    """The same model in fp64 with the given masks of its dropouts"""
    norm = lambda v, m: v / (v.square().mean(1, keepdim=True) + 1e-6).sqrt() * m.weight.double()

    def linear(v, m, a, b):
        y = v @ m.linear.weight.double().t()
        at = ids.clamp(min=0)
        return y + m.scaling * (ids >= 0)[:, None] * (b[at] @ (a[at] @ v[:, :, None]))[:, :, 0]

    branch, stream, params = torch.zeros_like(x), x, iter(seeds)
    for block, keep in zip(model.blocks, keeps):
        stream = stream + branch
        up = linear(norm(stream, block.norm), block.up, next(params), next(params))
        branch = linear(nn.functional.silu(up), block.down, next(params), next(params)) * keep / 0.9
    return norm(stream + branch, model.norm)


def test_fine_tuning_and_serving_together(f8):
    """A model of the norms, dropouts and adapters in fp32: its output and the gradients of all adapters against the same model in fp64, and the served
    copy (norms into block scales, frozen weights in block scales) against its own operators."""
    torch.manual_seed(0)
    model = f8.convert_dropouts(f8.convert_rms_norms(Model(96, 160, 2))).cuda()
    f8.adapt_linears(model, 3, 8, alpha=16)
    adapters = [p for m in model.modules() if isinstance(m, f8.AdaptedLinear) for p in (m.adapter_a, m.adapter_b)]
    with torch.no_grad():
        for p in adapters[1::2]:
            p.normal_(std=0.1)
    ids = whose("runs", 70, 3)
    f8.select_adapters(model, ids)
    x, g = torch.randn(70, 96, device="cuda"), torch.randn(70, 96, device="cuda")
    torch.manual_seed(9)
    keeps = [f8.dropout(torch.ones(70, 96, device="cuda"), 0.1) != 0 for _ in range(2)]
    torch.manual_seed(9)
    y = model.train()(x)
    got = torch.autograd.grad(y, adapters, g)
    doubles = [p.detach().double().requires_grad_() for p in adapters]
    want_y = reference(model, x.double(), ids, doubles, keeps)
    want = torch.autograd.grad(want_y, doubles, g.double())
    # fp32 throughout: a chain of eight products and five norms, each off by a few hundred roundings of what goes in
    for a, b in zip((y, *got), (want_y, *want)):
        assert (a.double() - b).norm() <= 1e-4 * b.norm()
    model.eval()
    with torch.no_grad():
        stream = torch.randn(5, 96, device="cuda")
        block = model.blocks[0]
        up = f8.Float8BlockwiseInferenceLinear.from_float(block.up.linear)
        kept, s = block.norm.blockwise(stream, residual=stream)
        normed, s2 = block.norm(stream, residual=stream)
        rows = f8.AdapterRows(ids[:5], 3)
        out = f8.low_rank_adapters(normed, block.up.adapter_a, block.up.adapter_b, rows, up(kept), 2.0)
        assert torch.equal(s, s2)
        base = kept.dequantized().double() @ up.dequantized_weight().double().t()
        check({"out": out}, {name: (v, off + 2.0**-9 * (kept.dequantized().double().abs() @ up.dequantized_weight().double().abs().t()))
                             for name, (v, off) in formula(normed, block.up.adapter_a, block.up.adapter_b, ids[:5], base, 2.0).items()})
