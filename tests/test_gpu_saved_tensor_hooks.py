"""Layer norm and the blockwise linear under hooks on saved tensors: what comes back as it was saved is used, anything else raises before a kernel is queued.
The refusals run over a stand-in library, whose entry points count their calls and queue nothing."""
import ctypes
import importlib.util
import shutil
import subprocess

import pytest
import torch

pytestmark = pytest.mark.gpu
BF16, FP32 = torch.bfloat16, torch.float32

_LIBRARY = """
#include <stdint.h>
int backwards = 0, casts = 0;
const char* f8mi_last_error(void) { return ""; }
int64_t f8mi_block_scale_bytes(int64_t rows, int64_t k) { return 256; }
int f8mi_block_cast(void) { casts++; return 0; }
int f8mi_block_gemm(void) { return 0; }
int64_t f8mi_block_gemm_workspace_bytes(int64_t m, int64_t n, int64_t k) { return 0; }
int f8mi_block_linear_few_rows(void) { return 0; }
int f8mi_column_sum_finish(void) { return 0; }
int f8mi_layer_norm(void) { return 0; }
int f8mi_layer_norm_backward(void) { backwards++; return 0; }
int64_t f8mi_layer_norm_workspace_bytes(int64_t rows, int64_t cols, int dtype) { return 0; }
int f8mi_grad_clip(void) { return 0; }
int64_t f8mi_grad_clip_workspace_bytes(int64_t count) { return 8; }
"""


@pytest.fixture(scope="module")
def f8():
    import float8_experimental_amd

    return float8_experimental_amd


@pytest.fixture(scope="module")
def stand_in(tmp_path_factory):
    """(the host path over the stand-in, the stand-in)"""
    from float8_experimental_amd import _native

    d = tmp_path_factory.mktemp("stand_in")
    (d / "stand_in.c").write_text(_LIBRARY)
    subprocess.run(["gcc", "-shared", "-fPIC", "-o", str(d / "stand_in.so"), str(d / "stand_in.c")], check=True)
    spec = importlib.util.spec_from_file_location("_f8mi_torch_ops", shutil.copy(_native._OPS_PATH, d / "_f8mi_torch_ops.so"))
    module = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(module)
    module.load(str(d / "stand_in.so"), RuntimeError)
    return module, ctypes.CDLL(str(d / "stand_in.so"))


ROWS, COLS = 12, 64
CHANGES = {
    "on the CPU": lambda t: t.cpu(), "of another type": lambda t: t.half(), "in 64 bits": lambda t: t.double(), "shorter": lambda t: t[:-1], "longer": lambda t: torch.cat([t, t]),
    "flat": lambda t: t.reshape(-1)[: t.numel() - 1], "sparse": lambda t: t.to_sparse(), "meta": lambda t: t.to("meta"),
}
EXPANDED = [("weight", lambda t: t[:1].expand(COLS + 1)), ("stats", lambda t: t[:1].expand(t.shape))]  # (rows of x that are all the same one are read as such)


def saved_kind(t):
    return {(ROWS, COLS): "x", (COLS,): "weight", (ROWS, 2): "stats"}[tuple(t.shape)]


@pytest.mark.parametrize("which,alter", [pytest.param(which, alter, id=f"{which}-{name}") for name, alter in CHANGES.items() for which in ("x", "weight", "stats")] + EXPANDED)
def test_layer_norm_refuses_what_was_not_saved(stand_in, which, alter):
    module, library = stand_in
    x, w, b = (torch.randn(s, device="cuda", dtype=d, requires_grad=True) for s, d in (((ROWS, COLS), BF16), ((COLS,), FP32), ((COLS,), FP32)))
    seen = []
    with torch.autograd.graph.saved_tensors_hooks(lambda t: (saved_kind(t), t.detach()), lambda p: seen.append(p[0]) or (alter(p[1]) if p[0] == which else p[1])):
        y = module.layer_norm(x, COLS, w, b, 1e-5)
        before = ctypes.c_int.in_dll(library, "backwards").value
        with pytest.raises(RuntimeError):
            y.backward(torch.ones_like(y))
    assert ctypes.c_int.in_dll(library, "backwards").value == before and set(seen) == {"x", "weight", "stats"}


def test_layer_norm_over_the_stand_in_without_a_change(stand_in):
    module, library = stand_in
    x, w = torch.randn(ROWS, COLS, device="cuda", requires_grad=True), torch.ones(COLS, device="cuda", requires_grad=True)
    before = ctypes.c_int.in_dll(library, "backwards").value
    with torch.autograd.graph.saved_tensors_hooks(lambda t: t.detach().clone(), lambda t: t):
        module.layer_norm(x, COLS, w, None, 1e-5).sum().backward()
    assert ctypes.c_int.in_dll(library, "backwards").value == before + 1


@pytest.mark.parametrize("change", list(CHANGES))
def test_linear_refuses_what_was_not_saved(stand_in, change):
    module, library = stand_in
    x, w = torch.randn(ROWS, COLS, device="cuda", dtype=BF16, requires_grad=True), torch.randn(32, COLS, device="cuda", dtype=BF16, requires_grad=True)
    with torch.autograd.graph.saved_tensors_hooks(lambda t: t.detach(), CHANGES[change]):
        y = module.blockwise_linear(x, w, None)
        before = ctypes.c_int.in_dll(library, "casts").value
        with pytest.raises(RuntimeError):
            y.backward(torch.ones_like(y))
    assert ctypes.c_int.in_dll(library, "casts").value == before


def test_saved_tensors_may_be_kept_elsewhere_and_in_another_order(f8):
    g = torch.Generator().manual_seed(0)
    made = [torch.randn(s, generator=g).to(BF16).cuda() for s in ((50, 256), (256,), (256,), (128, 256), (50, 128))]

    def step():
        x, w, b, weight = (t.clone().requires_grad_() for t in made[:4])
        y = f8.blockwise_linear(f8.layer_norm(x, 256, w, b), weight)
        return [y] + list(torch.autograd.grad(y, (x, w, b, weight), made[4]))

    want = step()
    columns = lambda t: t.t().contiguous().t() if t.shape == (50, 256) else t
    for context in (torch.autograd.graph.save_on_cpu(), torch.autograd.graph.saved_tensors_hooks(lambda t: t.detach().clone(), columns)):
        with context:
            got = step()
        assert all(torch.equal(p, q) for p, q in zip(got, want))
