"""Dropout without a stored mask: which values are kept against the generator's definition, values against the formula in 64 bits."""
import numpy as np
import pytest
import torch
import torch.nn as nn

pytestmark = pytest.mark.gpu
BF16, FP16, FP32 = torch.bfloat16, torch.float16, torch.float32


@pytest.fixture(scope="module")
def f8():
    import float8_experimental_amd

    return float8_experimental_amd


def words(seed, first, count):
    """Random words first .. first + count - 1 of a seed: Philox 4x32 with 7 rounds in numpy's 64-bit integers."""
    low = np.uint64(0xFFFFFFFF)
    block = np.arange(first // 4, (first + count + 3) // 4, dtype=np.uint64)
    c = [block & low, block >> np.uint64(32), np.zeros_like(block), np.zeros_like(block)]
    key = [seed % 2**32, seed % 2**64 >> 32]
    for _ in range(7):
        p, q = c[0] * np.uint64(0xD2511F53), c[2] * np.uint64(0xCD9E8D57)
        c = [(q >> np.uint64(32)) ^ c[1] ^ np.uint64(key[0]), q & low, (p >> np.uint64(32)) ^ c[3] ^ np.uint64(key[1]), p & low]
        key = [(key[0] + 0x9E3779B9) % 2**32, (key[1] + 0xBB67AE85) % 2**32]
    return np.stack(c, 1).reshape(-1)[first % 4:][:count]


def kept(seed, p, shape):
    n = int(np.prod(shape))
    return torch.from_numpy(words(seed, 0, n) >= round(p * 2**32)).view(shape).cuda()


def seed_of(value):
    return torch.tensor([value], dtype=torch.int64, device="cuda")


def made(shape, dtype, seed=0):
    g = torch.Generator().manual_seed(seed)
    return [torch.randn(shape, generator=g).to(dtype).cuda() for _ in range(3)]


def test_the_generator_has_its_published_values():
    """The first block of counter 0 and key 0 after 7 rounds, from the generator's known-answer vectors."""
    assert [f"{v:08x}" for v in words(0, 0, 4)] == ["5f6fb709", "0d893f64", "4f121f81", "4f730a48"]


def check(f8, shape, dtype, p, seed, residual=True):
    x, r, g = made(shape, dtype, seed % 1000)
    xs, rs = x.clone().requires_grad_(), r.clone().requires_grad_()
    out = f8.dropout(xs, p, seed_of(seed), rs if residual else None)
    out.backward(g)
    keep, half = kept(seed, p, shape), torch.finfo(dtype).eps / 2
    for got, value, add in ((out, x, r if residual else None), (xs.grad, g, None)):
        want = torch.where(keep, value.double() / (1 - p), 0.0)
        # 1 / (1 - p) and the product are rounded in fp32, the sum too, and the result once to its type
        off = 2.0**-23 * want.abs()
        if add is not None:
            want = want + add.double()
            off += 2.0**-24 * want.abs()
        assert got.dtype == dtype and ((got.detach().double() - want).abs() <= half * want.abs() + (1 + half) * off + (2.0**-25 if dtype is FP16 else 0)).all()
        if add is None:
            assert ((got.detach() == 0) | keep).all()
    if residual:
        assert torch.equal(rs.grad, g)


@pytest.mark.parametrize("dtype", [BF16, FP16, FP32])
@pytest.mark.parametrize("shape", [(1,), (3,), (4,), (7, 9), (8, 1000), (129, 1023), (3, 5, 77), (1000, 4096)])
def test_forward_and_backward(f8, shape, dtype):
    for p, seed, residual in ((0.1, 0, True), (0.5, -1, False), (0.0, 2**62 + 12345, True), (0.937, -(2**63), True)):
        check(f8, shape, dtype, p, seed, residual)


def test_probabilities_at_the_ends(f8):
    x, r, g = made((50, 70), FP32)
    for residual in (None, r):
        xs = x.clone().requires_grad_()
        out = f8.dropout(xs, 1.0, seed_of(3), residual)
        out.backward(g)
        assert torch.equal(out, torch.zeros_like(x) if residual is None else r) and (xs.grad == 0).all()
    assert torch.equal(f8.dropout(x, 0.0, seed_of(3)), x)
    few = f8.dropout(torch.ones(1 << 16, device="cuda"), 1 - 2.0**-12, seed_of(5))
    assert 0 < (few != 0).sum() < 64 and (few[few != 0] == 4096).all()


def test_what_is_dropped_is_zero_whatever_it_was(f8):
    x, r, _ = made((64, 64), BF16)
    keep = kept(11, 0.5, (64, 64))
    x[~keep] = float("nan")
    x[0, 0] = float("inf")
    out = f8.dropout(x, 0.5, seed_of(11), r)
    assert torch.equal(out[~keep], r[~keep]) and not out[keep].isnan().any()


def test_strides(f8):
    x, r, g = made((60, 300), BF16)
    for cut in (lambda t: t[:, 3:260], lambda t: t.t(), lambda t: t[::2], lambda t: t[:1].expand(60, 300), lambda t: t.reshape(-1)[1:1001]):
        a = cut(x).detach().requires_grad_()
        out = f8.dropout(a, 0.3, seed_of(9), cut(r))
        (da,) = torch.autograd.grad(out, a, cut(g))
        same = f8.dropout(cut(x).contiguous(), 0.3, seed_of(9), cut(r).contiguous())
        assert torch.equal(out, same) and torch.equal(da, f8.dropout(cut(g).contiguous(), 0.3, seed_of(9)))
    a = x.clone().requires_grad_()
    f8.dropout(a, 0.3, seed_of(9)).sum().backward()  # a gradient that is one number expanded
    assert torch.equal(a.grad, f8.dropout(torch.ones_like(x), 0.3, seed_of(9)))
    assert f8.dropout(x[:0], 0.3).shape == (0, 300)


def test_seeds_of_torchs_generator(f8):
    x = torch.ones(1000, 1000, device="cuda")
    torch.manual_seed(3)
    a, b = f8.dropout(x, 0.25), f8.dropout(x, 0.25)
    torch.manual_seed(3)
    assert torch.equal(f8.dropout(x, 0.25), a) and not torch.equal(a, b)
    # a share of a million independent trials: ten standard deviations
    assert abs((a == 0).float().mean().item() - 0.25) < 10 * (0.25 * 0.75 / 1e6) ** 0.5


def test_far_elements_have_their_own_words(f8):
    """Elements past 2^34, whose counters need more than 32 bits."""
    n = 2**34 + 1001
    x = torch.ones(n, device="cuda", dtype=BF16)
    out = f8.dropout(x, 0.5, seed_of(77))
    del x
    for first in (0, 2**32 - 500, 2**34 - 500):
        want = torch.from_numpy(words(77, first, 1000) >= 2**31)
        assert torch.equal(out[first:first + 1000].cpu() != 0, want)
    assert torch.equal(out[-3:].cpu() != 0, torch.from_numpy(words(77, n - 3, 3) >= 2**31))


def test_module_compile_stream_and_graph(f8):
    x, r, g = made((40, 256), BF16)
    model = f8.convert_dropouts(nn.Sequential(nn.Dropout(0.2), nn.Sequential(nn.Dropout(0.4))))
    assert [m.p for m in model.modules() if type(m) is f8.Dropout] == [0.2, 0.4] and type(f8.convert_dropouts(nn.Dropout())) is f8.Dropout
    assert (model.train()(x) == 0).any() and torch.equal(model.eval()(x), x) and torch.equal(model[0](x, r), x + r)
    with pytest.raises(NotImplementedError):
        f8.convert_dropouts(nn.Dropout(0.5, inplace=True))
    seed, runs = seed_of(5), []
    for fn in (f8.dropout, torch.compile(f8.dropout, fullgraph=True, backend="aot_eager")):
        a, b = x.clone().requires_grad_(), r.clone().requires_grad_()
        out = fn(a, 0.2, seed, b)
        out.backward(g)
        runs.append([out, a.grad, b.grad])
    assert all(torch.equal(p, q) for p, q in zip(*runs))
    a = x.clone().requires_grad_()

    def step():
        out = f8.dropout(a, 0.2, seed, r)
        return (out.detach(),) + torch.autograd.grad(out, a, g)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
        got = step()
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    assert torch.equal(got[0], runs[0][0]) and torch.equal(got[1], runs[0][1])
    graph, drawn = torch.cuda.CUDAGraph(), torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = step()
    with torch.cuda.graph(drawn):  # the seed is drawn inside: another at each replay
        other = f8.dropout(x, 0.5)
    seen = []
    for i in range(3):
        seed.fill_(100 + i)  # the seed is read at each replay
        graph.replay()
        drawn.replay()
        torch.cuda.synchronize()
        recorded = [t.clone() for t in got]
        assert all(torch.equal(p, q) for p, q in zip(recorded, step()))
        seen.append(other.clone())
    assert not torch.equal(seen[0], seen[1]) and not torch.equal(seen[1], seen[2])


def test_refusals(f8):
    x, r, g = made((4, 64), BF16)
    for bad in (lambda: f8.dropout(x, -0.1), lambda: f8.dropout(x, 1.5), lambda: f8.dropout(x, float("nan")), lambda: f8.dropout(x, 0.5, torch.zeros(2, dtype=torch.int64, device="cuda")),
                lambda: f8.dropout(x, 0.5, torch.zeros(1, device="cuda")), lambda: f8.dropout(x, 0.5, residual=r[:3]), lambda: f8.dropout(x, 0.5, residual=r.float())):
        with pytest.raises(ValueError):
            bad()
    with pytest.raises(TypeError):
        f8.dropout(x.double(), 0.5)
    for bad in (lambda: f8.dropout(x, 0.5, torch.zeros(1, dtype=torch.int64)), lambda: f8.dropout(x, 0.5, residual=r.cpu()), lambda: f8.dropout(x.cpu(), 0.5)):
        with pytest.raises(RuntimeError):
            bad()
    a, seed = x.clone().requires_grad_(), seed_of(1)
    out = f8.dropout(a, 0.5, seed)
    with pytest.raises(RuntimeError, match="second derivative"):
        torch.autograd.grad(out.sum(), a, create_graph=True)
    out = f8.dropout(a, 0.5, seed)
    seed.add_(1)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        out.backward(g)
