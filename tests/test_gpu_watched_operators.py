"""Blockwise linears, layer norm and clipping where somebody has to see operators: under a trace, a function mode or a dispatch mode the calls are
operators (or raise), with the values of the plain call."""
import copy
import warnings

import pytest
import torch
import torch.nn as nn
from torch.utils._python_dispatch import TorchDispatchMode

pytestmark = pytest.mark.gpu
BF16 = torch.bfloat16


@pytest.fixture(scope="module")
def f8():
    import float8_experimental_amd

    return float8_experimental_amd


def normal(*shape, dtype=BF16, seed=0):
    return torch.randn(shape, generator=torch.Generator().manual_seed(seed)).to(dtype).cuda()


class Dispatch(TorchDispatchMode):
    def __init__(self, seen):
        super().__init__()
        self.seen = seen

    def __torch_dispatch__(self, func, types, args=(), kwargs=None):
        self.seen.append(str(func))
        return func(*args, **(kwargs or {}))


class Function(torch.overrides.TorchFunctionMode):
    def __init__(self, seen):
        super().__init__()
        self.seen = seen

    def __torch_function__(self, func, types, args=(), kwargs=None):
        self.seen.append(str(func))
        return func(*args, **(kwargs or {}))


def forwards(f8, trains=True):
    """(name, name of its operator, call, x): what a model runs forward"""
    w, b = normal(128, 256, seed=1), normal(128, seed=2)
    p, q = normal(256, seed=3, dtype=torch.float32), normal(256, seed=4, dtype=torch.float32)
    lin = nn.Linear(256, 128, device="cuda", dtype=BF16)
    served = f8.Float8BlockwiseInferenceLinear.from_float(lin)
    norm = f8.LayerNorm.from_float(nn.LayerNorm(256, device="cuda", dtype=BF16).requires_grad_(trains))
    return [("linear", "f8mi.blockwise_linear_fwd", lambda x: f8.blockwise_linear(x, w, b), normal(40, 256)),
            ("linear, 3-D", "f8mi.blockwise_linear_fwd", lambda x: f8.blockwise_linear(x, w), normal(2, 20, 256)),
            ("served, few", "f8mi.blockwise_inference_linear", served, normal(3, 256)),
            ("served, many", "f8mi.blockwise_inference_linear", served, normal(2, 150, 256)),
            ("norm", "f8mi.layer_norm_fwd", lambda x: f8.layer_norm(x, 256, p, q), normal(40, 256)),
            ("norm, module", "f8mi.layer_norm_fwd", norm, normal(4, 10, 256))]


TRACED = {"f8mi.blockwise_linear_fwd": "f8mi::blockwise_linear", "f8mi.blockwise_inference_linear": "f8mi::blockwise_inference_linear",
          "f8mi.layer_norm_fwd": "f8mi::layer_norm"}  # training and inference are the same trace


def same(got, want):
    """The served linear of a few rows adds its parts in another order where cast and product are two kernels."""
    return got.shape == want.shape and got.dtype == want.dtype and ((got.double() - want.double()).abs() <= 2.0**-7 * want.double().abs() + 2.0**-6).all()


def test_traces_hold_operators_and_their_values(f8):
    for name, op, call, x in forwards(f8):
        with torch.no_grad(), warnings.catch_warnings():
            warnings.simplefilter("ignore")
            traced = torch.jit.trace(call, x)
            assert f"{TRACED[op]}(" in str(traced.inlined_graph), name
            for seed in (7, 8):
                other = normal(*x.shape, seed=seed)
                assert same(traced(other), call(other)), name


def test_traced_modules_train_and_are_saved(f8, tmp_path):
    blk = f8.CastConfig(scaling_type=f8.ScalingType.BLOCKWISE)
    config = f8.Float8LinearConfig(cast_config_input=blk, cast_config_weight=blk, cast_config_grad_output=blk)
    torch.manual_seed(0)
    model = f8.convert_layer_norms(f8.convert_to_float8_training(nn.Sequential(nn.LayerNorm(256), nn.Linear(256, 384)).to("cuda", BF16), config=config))
    x, dy = normal(40, 256), normal(40, 384, seed=5)
    with warnings.catch_warnings():
        warnings.simplefilter("ignore")
        traced = torch.jit.trace(model, normal(40, 256, seed=9))
    torch.jit.save(traced, str(tmp_path / "traced.pt"))
    loaded = torch.jit.load(str(tmp_path / "traced.pt"))
    with torch.no_grad():
        assert torch.equal(loaded(x), model(x))
    runs = []
    for call in (model, traced):
        model.zero_grad()
        xs = x.clone().requires_grad_()
        y = call(xs)
        y.backward(dy)
        runs.append([y, xs.grad] + [p.grad.clone() for p in model.parameters()])
    assert all(torch.equal(p, q) for p, q in zip(*runs))


@pytest.mark.parametrize("mode", [Dispatch, Function])
def test_modes_see_operators(f8, mode):
    for name, op, call, x in forwards(f8):
        with torch.no_grad():
            want, seen = call(x), []
            with mode(seen):
                got = call(x)
        assert same(got, want) and any(op in s for s in seen), (name, seen)


def test_a_default_device_asks_for_nothing(f8):
    """torch.set_default_device is a function mode: the calls stay the fast ones, with their bits."""
    for name, op, call, x in forwards(f8):
        with torch.no_grad():
            want = call(x)
            with torch.device("cuda"):
                assert torch.equal(call(x), want), name
    grads = [normal(100, seed=1), normal(30, 7, seed=2)]
    want = f8.clip_grads(grads, 1.0)
    with torch.device("cuda"):
        got = f8.clip_grads(grads, 1.0)
    assert torch.equal(got[0], want[0]) and all(torch.equal(p, q) for p, q in zip(got[1], want[1]))


def test_function_modes_see_training_and_clipping(f8):
    x, w = normal(40, 256).requires_grad_(), normal(128, 256, seed=1).requires_grad_()
    dy = normal(40, 128, seed=2)
    want = f8.blockwise_linear(x, w)
    want_grads = torch.autograd.grad(want, (x, w), dy)
    seen = []
    with Function(seen):
        got = f8.blockwise_linear(x, w)
    assert torch.equal(got, want) and all(torch.equal(p, q) for p, q in zip(torch.autograd.grad(got, (x, w), dy), want_grads))
    assert any("blockwise_linear_fwd" in s for s in seen)
    grads = [normal(100, seed=1), normal(30, 7, seed=2)]
    norm, clipped = f8.clip_grads(grads, 1.0)
    params = [nn.Parameter(torch.zeros_like(g)) for g in grads]
    for p, g in zip(params, copy.deepcopy(grads)):
        p.grad = g
    for call, name in ((lambda: f8.grad_norm(grads), "grad_norm"), (lambda: f8.clip_grads(grads, 1.0)[0], "clip_grads"), (lambda: f8.clip_grad_norm_(params, 1.0), "clip_grad_norm_")):
        seen.clear()
        with Function(seen):
            assert torch.equal(call(), norm)
        assert any(name in s for s in seen), (name, seen)
    assert all(torch.equal(p.grad, q) for p, q in zip(params, clipped))


def test_clipping_is_not_traced(f8):
    """It has no operators that a trace could hold: an error, not a trace of the allocations."""
    g = normal(100)
    p = nn.Parameter(torch.zeros_like(g))
    p.grad = g
    for call in (lambda t: f8.grad_norm([t]), lambda t: f8.clip_grads([t], 1.0)[1][0], lambda t: f8.clip_grad_norm_([p], 1.0)):
        with pytest.raises(RuntimeError, match="trace"), warnings.catch_warnings():
            warnings.simplefilter("ignore")
            torch.jit.trace(call, g)


def test_calls_inside_functional_transforms_of_something_else(f8):
    """Tensors that a transform does not know are constants to it; a history inside one is refused, as by any C++ autograd function."""
    scale = torch.tensor([1.0, 2.0], device="cuda")
    for name, op, call, x in forwards(f8, trains=False):
        with torch.no_grad():
            want = call(x).float()
            for got in (torch.func.grad(lambda s: (call(x).float() * s).sum())(scale[0]), torch.func.jvp(lambda s: (call(x).float() * s).sum(), (scale[0],), (scale[0],))[1]):
                assert abs(got - want.sum()) <= 2.0**-7 * want.abs().sum(), name
            batch = torch.func.vmap(lambda s: call(x).float() * s)(scale)
            assert torch.equal(batch, want * scale.view(2, *[1] * want.dim())), name
    x, w = normal(40, 256), normal(128, 256, seed=1).requires_grad_()
    with pytest.raises(RuntimeError, match="functorch"):
        torch.func.vmap(lambda s: f8.blockwise_linear(x, w).float() * s)(scale)
