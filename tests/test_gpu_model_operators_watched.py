"""RMS norm, dropout and the adapters where somebody has to see operators (traces, modes, functional transforms), where derivatives are of another kind, and under hooks on saved
tensors.  The refusals of what hooks hand back run over a stand-in library, whose entry points count their calls and queue nothing."""
import ctypes
import importlib.util
import shutil
import subprocess
import warnings

import pytest
import torch
import torch.autograd.forward_ad as fwd
import torch.nn as nn
from torch.utils._python_dispatch import TorchDispatchMode

pytestmark = pytest.mark.gpu
BF16, FP32 = torch.bfloat16, torch.float32


@pytest.fixture(scope="module")
def f8():
    import float8_experimental_amd

    return float8_experimental_amd


def normal(*shape, dtype=BF16, seed=0):
    return torch.randn(shape, generator=torch.Generator().manual_seed(seed)).to(dtype).cuda()


def calls(f8):
    """name -> (name of its operator, its name in a trace, call, differentiable arguments)"""
    rows = f8.AdapterRows(torch.arange(40, device="cuda") % 4 - 1, 3)
    seed = torch.full((1,), 5, dtype=torch.int64, device="cuda")
    served = f8.Float8BlockwiseInferenceLinear.from_float(nn.Linear(256, 64, device="cuda", dtype=BF16))
    x, r, w = normal(40, 256), normal(40, 256, seed=1), normal(256, seed=2, dtype=FP32)
    a, b, y = normal(3, 8, 256, seed=3), normal(3, 128, 8, seed=4), normal(40, 128, seed=5)
    return {
        "norm": ("f8mi.rms_norm_fwd", "f8mi::rms_norm", lambda x, w: f8.rms_norm(x, 256, w, 1e-6), [x, w]),
        "norm, 3-D": ("f8mi.rms_norm_fwd", "f8mi::rms_norm", lambda x, w: f8.rms_norm(x.view(2, 20, 256), 256, w, 1e-6), [x, w]),
        "norm, residual": ("f8mi.rms_norm_fwd", "f8mi::rms_norm_add", lambda x, w, r: f8.rms_norm(x, 256, w, 1e-6, r), [x, w, r]),
        "dropout": ("f8mi.dropout_masked", "f8mi::dropout", lambda x, r: f8.dropout(x, 0.25, seed, r), [x, r]),
        "adapters": ("f8mi.adapters_fwd", "f8mi::low_rank_adapters", lambda x, a, b, y: f8.low_rank_adapters(x, a, b, rows, y, 0.5), [x, a, b, y]),
        "served": ("f8mi.rms_norm_blockwise", "f8mi::rms_norm_blockwise", lambda x: served(f8.rms_norm_blockwise(x, 256, w, 1e-6)), [x]),
    }


NAMES = ["norm", "norm, 3-D", "norm, residual", "dropout", "adapters", "served"]


def flat(out):
    return list(out) if isinstance(out, tuple) else [out]


def equal(got, want):
    return all(p.shape == q.shape and torch.equal(p, q) for p, q in zip(flat(got), flat(want)))


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


@pytest.mark.parametrize("name", NAMES)
def test_modes_and_traces_see_operators(f8, name):
    op, traced_op, call, args = calls(f8)[name]
    with torch.no_grad():
        want = call(*args)
        for mode in (Dispatch, Function):
            seen = []
            with mode(seen):
                got = call(*args)
            assert equal(got, want) and any(op in s for s in seen), (mode, seen)
        with torch.device("cuda"):  # a function mode that asks for nothing
            assert equal(call(*args), want)
        with warnings.catch_warnings():
            warnings.simplefilter("ignore")
            traced = torch.jit.trace(call, tuple(normal(*t.shape, dtype=t.dtype, seed=9) for t in args))
        assert f"{traced_op}(" in str(traced.inlined_graph)
        assert equal(traced(*args), want)


@pytest.mark.parametrize("name", NAMES[:5])
def test_gradients_through_modes_and_traces(f8, name):
    _, _, call, args = calls(f8)[name]

    def grads(call):
        ts = [t.clone().requires_grad_() for t in args]
        out = flat(call(*ts))
        return torch.autograd.grad(out, ts, [normal(*o.shape, seed=20 + i) for i, o in enumerate(out)])

    want = grads(call)
    with warnings.catch_warnings():
        warnings.simplefilter("ignore")
        traced = torch.jit.trace(call, tuple(t.clone().requires_grad_() for t in args))
    assert equal(tuple(grads(traced)), tuple(want))
    with Function([]):
        assert equal(tuple(grads(call)), tuple(want))
    assert equal(tuple(grads(torch.compile(call, fullgraph=True, backend="aot_eager"))), tuple(want))


def test_compiled_calls_without_gradients(f8):
    for name, (_, _, call, args) in calls(f8).items():
        with torch.no_grad():
            assert equal(torch.compile(call, fullgraph=True, backend="aot_eager")(*args), call(*args)), name
    x = torch.ones(100, 100, device="cuda")
    drawn = torch.compile(lambda t: f8.dropout(t, 0.5), fullgraph=True, backend="aot_eager")
    a, b = drawn(x), drawn(x)  # a seed of its own each time
    assert 0.4 < (a == 0).float().mean() < 0.6 and not torch.equal(a, b)


def test_autocast(f8):
    """The norm and dropout keep x's type; the adapters and the served linear take the autocast type, as the linears do."""
    x, w = normal(40, 256, dtype=FP32), normal(256, dtype=FP32, seed=1)
    a, b, y = normal(3, 8, 256, seed=3, dtype=FP32), normal(3, 128, 8, seed=4, dtype=FP32), normal(40, 128, seed=5, dtype=FP32)
    rows = f8.AdapterRows(torch.arange(40, device="cuda") % 3, 3)
    served = f8.Float8BlockwiseInferenceLinear.from_float(nn.Linear(256, 64, device="cuda", dtype=FP32))
    layer = f8.AdaptedLinear(nn.Linear(256, 128, device="cuda"), 3, 8)
    f8.select_adapters(layer, rows)
    with torch.no_grad():
        layer.adapter_b.normal_()
        plain = f8.low_rank_adapters(x.bfloat16(), a, b, rows, y.bfloat16())
        with torch.autocast("cuda", dtype=BF16):
            assert f8.rms_norm(x, 256, w).dtype == FP32 and f8.dropout(x, 0.5).dtype == FP32
            out = f8.low_rank_adapters(x, a, b, rows, y)
            assert out.dtype == BF16 and torch.equal(out, plain)
            assert served(f8.rms_norm_blockwise(x, 256, w)).dtype == BF16 and layer(x).dtype == BF16
    xs = x.clone().requires_grad_()
    with torch.autocast("cuda", dtype=BF16):
        layer(xs).sum().backward()
    assert xs.grad.dtype == FP32 and layer.adapter_a.grad.dtype == FP32 and xs.grad.isfinite().all()


@pytest.mark.parametrize("name", NAMES)
def test_tangents_raise(f8, name):
    _, _, call, args = calls(f8)[name]
    for i in range(len(args)):
        for context in (torch.no_grad, torch.enable_grad):
            with fwd.dual_level(), context():
                with pytest.raises(NotImplementedError, match="forward-mode"):
                    call(*[fwd.make_dual(t, torch.ones_like(t)) if j == i else t for j, t in enumerate(args)])
    with torch.no_grad():
        want = call(*args)
        with fwd.dual_level():
            assert equal(call(*args), want)


@pytest.mark.parametrize("name", NAMES)
def test_calls_inside_functional_transforms_of_something_else(f8, name):
    _, _, call, args = calls(f8)[name]
    scale = torch.tensor([1.0, 2.0], device="cuda")
    with torch.no_grad():
        want = flat(call(*args))[0].float()
        got = torch.func.grad(lambda s: (flat(call(*args))[0].float() * s).sum())(scale[0])
        assert abs(got - want.sum()) <= 2.0**-7 * want.abs().sum()
        batch = torch.func.vmap(lambda s: flat(call(*args))[0].float() * s)(scale)
        assert torch.equal(batch, want * scale.view(2, *[1] * want.dim()))


# ---- hooks on saved tensors

_LIBRARY = """
#include <stdint.h>
int backwards = 0;
const char* f8mi_last_error(void) { return ""; }
int64_t f8mi_block_scale_bytes(int64_t rows, int64_t k) { return 256; }
int f8mi_block_gemm(void) { return 0; }
int64_t f8mi_block_gemm_workspace_bytes(int64_t m, int64_t n, int64_t k) { return 0; }
int f8mi_rms_norm(void) { return 0; }
int f8mi_rms_norm_block(void) { return 0; }
int f8mi_rms_norm_backward(void) { backwards++; return 0; }
int64_t f8mi_rms_norm_workspace_bytes(int64_t rows, int64_t cols, int dtype, int p_dtype) { return 0; }
int calls = 0;
int f8mi_dropout(void) { calls++; return 0; }
int64_t f8mi_adapter_rows_words(int64_t m, int64_t count) { return 40; }
int f8mi_adapters(void) { return 0; }
int64_t f8mi_adapters_workspace_bytes(int64_t m, int64_t k, int64_t n, int64_t r, int64_t count, int dtype) { return 0; }
int f8mi_adapters_backward(void) { backwards++; return 0; }
int64_t f8mi_adapters_backward_workspace_bytes(int64_t m, int64_t k, int64_t n, int64_t r, int64_t count, int dtype, int a, int b, int c) { return 0; }
"""


@pytest.fixture(scope="module")
def stand_in(tmp_path_factory):
    """(the host path over the stand-in, the stand-in)"""
    from float8_experimental_amd import _native

    d = tmp_path_factory.mktemp("stand_in")
    (d / "stand_in.c").write_text(_LIBRARY)
    subprocess.run(["gcc", "-shared", "-fPIC", "-o", str(d / "stand_in.so"), str(d / "stand_in.c")], check=True)
    spec = importlib.util.spec_from_file_location("_f8mi_torch_model", shutil.copy(_native._MODEL_PATH, d / "_f8mi_torch_model.so"))
    module = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(module)
    module.load(str(d / "stand_in.so"), RuntimeError)
    return module, ctypes.CDLL(str(d / "stand_in.so"))


CHANGES = {
    "on the CPU": lambda t: t.cpu(), "of another type": lambda t: t.double(), "shorter": lambda t: t[:-1], "longer": lambda t: torch.cat([t, t]), "flat": lambda t: t.reshape(-1)[: t.numel() - 1],
    "sparse": lambda t: t.to_sparse(), "meta": lambda t: t.to("meta"),
}


def refuses(module, library, counter, forward, tensor_of, which, alter):
    seen = []

    def pack(t):
        seen.append(tensor_of(t))
        return tensor_of(t), t.detach()

    with torch.autograd.graph.saved_tensors_hooks(pack, lambda p: alter(p[1]) if p[0] == which else p[1]):
        out = forward()
        out = out[0] if isinstance(out, tuple) else out
        before = ctypes.c_int.in_dll(library, counter).value
        with pytest.raises(RuntimeError):
            out.backward(torch.ones_like(out))
    assert ctypes.c_int.in_dll(library, counter).value == before and which in seen


@pytest.mark.parametrize("change", list(CHANGES))
@pytest.mark.parametrize("which", ["s", "weight", "rstd"])
def test_rms_norm_refuses_what_was_not_saved(stand_in, which, change):
    module, library = stand_in
    x, r, w = (torch.randn(s, device="cuda", dtype=d, requires_grad=True) for s, d in (((12, 64), BF16), ((12, 64), BF16), ((64,), FP32)))
    refuses(module, library, "backwards", lambda: module.rms_norm(x, 64, w, 1e-6, r), lambda t: {(12, 64): "s", (64,): "weight", (12,): "rstd"}[tuple(t.shape)], which, CHANGES[change])


@pytest.mark.parametrize("change", [c for c in CHANGES if c not in ("flat", "shorter")] + ["shorter"])
def test_dropout_refuses_what_was_not_saved(stand_in, change):
    module, library = stand_in
    x = torch.randn(12, 64, device="cuda", requires_grad=True)
    refuses(module, library, "calls", lambda: module.dropout(x, 0.5, torch.zeros(1, dtype=torch.int64, device="cuda"), None), lambda t: "seed", "seed", CHANGES[change])


@pytest.mark.parametrize("change", list(CHANGES))
@pytest.mark.parametrize("which", ["x", "a", "b", "table", "scale", "h"])
def test_adapters_refuse_what_was_not_saved(stand_in, which, change):
    module, library = stand_in
    x, a, b = (torch.randn(s, device="cuda", dtype=BF16, requires_grad=True) for s in ((12, 64), (3, 8, 64), (3, 48, 8)))
    table, scale = torch.zeros(40, dtype=torch.int32, device="cuda"), torch.ones(3, device="cuda")
    kinds = {(12, 64): "x", (3, 8, 64): "a", (3, 48, 8): "b", (40,): "table", (3,): "scale", (12, 16): "h"}
    refuses(module, library, "backwards", lambda: module.low_rank_adapters(x, a, b, table, 12, 3, None, scale, 1.0), lambda t: kinds[tuple(t.shape)], which, CHANGES[change])


@pytest.mark.parametrize("name", NAMES[:5])
def test_saved_tensors_may_be_kept_elsewhere(f8, name):
    _, _, call, args = calls(f8)[name]

    def grads():
        ts = [t.clone().requires_grad_() for t in args]
        out = flat(call(*ts))
        return torch.autograd.grad(out, ts, [normal(*o.shape, seed=20 + i) for i, o in enumerate(out)])

    want = grads()
    for context in (torch.autograd.graph.save_on_cpu(), torch.autograd.graph.saved_tensors_hooks(lambda t: t.detach().clone(), lambda t: t)):
        with context:
            assert equal(tuple(grads()), tuple(want))


# ---- other callers of the allocator, streams and threads


def test_two_threads_on_two_streams(f8):
    """The calls share nothing: each thread's results are those of a call alone."""
    import threading

    want = {name: flat(call(*args)) for name, (_, _, call, args) in calls(f8).items() if name != "served"}
    wrong = []

    def work(i):
        with torch.cuda.stream(torch.cuda.Stream()):
            mine = calls(f8)
            torch.cuda.current_stream().synchronize()
            for _ in range(20):
                for name in want:
                    got = flat(mine[name][2](*mine[name][3]))
                    torch.cuda.current_stream().synchronize()
                    if not equal(tuple(got), tuple(want[name])):
                        wrong.append((i, name))

    threads = [threading.Thread(target=work, args=(i,)) for i in range(4)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not wrong


def test_offsets_that_pass_32_bits(f8):
    """The last rows have the values that they have by themselves."""
    x = normal(1000, 4096).repeat(600, 1)  # 4.9 GB
    w = normal(4096, seed=1, dtype=FP32)
    tail = x[-1000:].clone().requires_grad_()
    y, s = f8.rms_norm(tail, 4096, w, 1e-6, residual=tail.detach())
    (want,) = torch.autograd.grad([y, s], tail, [tail.detach(), tail.detach()])
    whole = x.requires_grad_()
    z, t = f8.rms_norm(whole, 4096, w, 1e-6, residual=x.detach())
    assert torch.equal(z[-1000:], y) and torch.equal(t[-1000:], s)
    (got,) = torch.autograd.grad([z, t], whole, [x.detach(), x.detach()])
    assert torch.equal(got[-1000:], want)
    del z, t, got
    with torch.no_grad():
        kept, small = f8.rms_norm_blockwise(x, 4096, w, 1e-6), f8.rms_norm_blockwise(tail, 4096, w, 1e-6)
        assert torch.equal(kept.data[:, -1000:].view(torch.uint8), small.data.view(torch.uint8))
