"""What RMS norm, dropout and the low-rank adapters refuse or decide on the host, and their operators as a compiler sees them: no GPU needed."""
import pytest
import torch
import torch.nn as nn
from torch._subclasses.fake_tensor import FakeTensorMode

import float8_experimental_amd as f8
from float8_experimental_amd import _custom_ops_model as ops
from float8_experimental_amd import _native

BF16, FP32 = torch.bfloat16, torch.float32


def test_tensors_on_the_cpu_are_refused():
    x, ids = torch.ones(4, 8), torch.zeros(4, dtype=torch.int64)
    for call in (lambda: f8.rms_norm(x, 8), lambda: f8.rms_norm_blockwise(x, 8), lambda: f8.RMSNorm(8)(x, x), lambda: f8.dropout(x, 0.5), lambda: f8.dropout(x, 0.5, torch.zeros(1, dtype=torch.int64)),
                 lambda: f8.AdapterRows(ids, 2), lambda: f8.low_rank_adapters(x, torch.ones(2, 4, 8), torch.ones(2, 6, 4), ids)):
        with pytest.raises(_native.Float8NativeError):
            call()


def test_arguments_are_checked_before_tensors():
    x = torch.ones(4, 8)
    for p in (-1e-9, 1.0000001, float("nan")):
        with pytest.raises(ValueError, match="probability"):
            f8.dropout(x, p)
    for kw in ({"count": 0, "rank": 4}, {"count": 2, "rank": 0}, {"count": 2, "rank": 257}, {"count": 2, "rank": 4, "dropout": 2.0}):
        with pytest.raises(ValueError):
            f8.AdaptedLinear(nn.Linear(4, 4), **kw)
    with pytest.raises(NotImplementedError):
        f8.Dropout.from_float(nn.Dropout(0.5, inplace=True))


def test_adapting_twice_keeps_the_first_adapters():
    model = nn.Sequential(nn.Linear(8, 6), nn.Linear(6, 4))
    f8.adapt_linears(model, 3, 2, module_filter_fn=lambda m, fqn: fqn == "0")
    first = model[0]
    assert f8.adapt_linears(model, 3, 4, module_filter_fn=lambda m, fqn: True) is model
    assert model[0] is first and type(first.linear) is nn.Linear and type(model[1]) is f8.AdaptedLinear and (first.rank, model[1].rank) == (2, 4)
    assert [n for n, p in model.named_parameters() if p.requires_grad] == ["0.adapter_a", "0.adapter_b", "1.adapter_a", "1.adapter_b"]
    assert f8.adapt_linears(first, 3, 4) is first and type(first.linear) is nn.Linear


def test_activations_that_have_been_cast_are_refused_beside_adapters():
    layer = f8.AdaptedLinear(nn.Linear(8, 6), 2, 2)
    layer.linear, layer.rows = nn.Identity(), object()  # (as a linear that takes them, and any rows)
    with pytest.raises(TypeError, match="BlockwiseActivations"):
        layer(f8.BlockwiseActivations(torch.empty(2, 1, 64), torch.empty(1), (1, 8), BF16))


def test_modules_are_swapped_and_share_their_parameters():
    model = nn.Sequential(nn.RMSNorm(8, eps=1e-3), nn.Dropout(0.3), nn.Linear(8, 6), nn.Sequential(nn.RMSNorm(6), nn.Linear(6, 4, bias=False)))
    weights = dict(model.named_parameters())
    f8.adapt_linears(f8.convert_dropouts(f8.convert_rms_norms(model)), 3, 2, alpha=4, dropout=0.1, module_filter_fn=lambda m, fqn: fqn != "3.1")
    assert [type(m) for m in model] == [f8.RMSNorm, f8.Dropout, f8.AdaptedLinear, nn.Sequential] and type(model[3][0]) is f8.RMSNorm and type(model[3][1]) is nn.Linear
    assert model[0].weight is weights["0.weight"] and model[2].linear.weight is weights["2.weight"] and model[0].eps == 1e-3 and model[1].p == 0.3
    assert [n for n, p in model.named_parameters() if p.requires_grad] == ["2.adapter_a", "2.adapter_b"]
    assert model[2].adapter_a.shape == (3, 2, 8) and model[2].adapter_b.shape == (3, 6, 2) and (model[2].adapter_b == 0).all() and model[2].scaling == 2.0
    x = torch.randn(5, 8)
    assert torch.equal(model[2](x), model[2].linear(x))  # no rows are selected
    assert type(f8.adapt_linears(nn.Linear(4, 4), 1, 1)) is f8.AdaptedLinear


def test_sizes_of_the_table():
    lib = _native.lib()
    for m, count in ((0, 1), (1, 1), (16, 3), (17, 1000), (64, 64), (2049, 7), (16384, 16), (16385, 2), (1 << 24, 32768)):
        assert ops.adapter_rows_words(m, count) == lib.f8mi_adapter_rows_words(m, count)
    assert lib.f8mi_adapter_rows_words(-1, 2) == 0 and lib.f8mi_adapter_rows_words(5, 0) == 0


def test_arguments_of_the_library_are_checked_on_the_host():
    lib, p = _native.lib(), 1 << 20  # no address is read
    err = lambda: lib.f8mi_last_error().decode()

    def norm(x=p, ld=8, res=None, ld_res=8, rows=4, cols=8, dt=0, pt=0, y=p, total=None):
        return lib.f8mi_rms_norm(x, ld, res, ld_res, rows, cols, dt, None, pt, 1e-6, y, total, None, None)

    assert norm(x=None) == -1 and norm(y=None) == -1 and norm(ld=7) == -1 and norm(ld=-8) == -1 and norm(res=p) == -1 and norm(res=p, total=p, ld_res=7) == -1
    assert norm(cols=0) == -1 and norm(rows=-1) == -1 and norm(dt=3) == -1 and norm(pt=1) == -1 and "weight" in err() and norm(rows=1 << 40) == -2 and norm(rows=0) == 0

    def block(out=p, scales=p, **kw):
        a = dict(x=p, ld=8, res=None, total=None, rows=4, cols=8, dt=0) | kw
        return lib.f8mi_rms_norm_block(a["x"], a["ld"], a["res"], 8, a["rows"], a["cols"], a["dt"], None, a["dt"], 1e-6, out, scales, a["total"], None)

    assert block(out=None) == -1 and block(scales=None) == -1 and block(out=p + 8) == -1 and "aligned" in err() and block(res=p) == -1 and block(ld=3) == -1 and block(rows=0) == 0
    assert lib.f8mi_rms_norm_backward(p, 8, p, 8, None, 0, 4, 8, 0, None, 0, p, p, p, None, 0, None) == -1 and "workspace" in err()
    assert lib.f8mi_rms_norm_backward(p, 8, p, 8, p, 7, 4, 8, 0, None, 0, p, p, None, None, 0, None) == -1
    assert lib.f8mi_rms_norm_backward(p, 8, p, 8, None, 0, 4, 8, 0, None, 0, None, p, None, None, 0, None) == -1
    assert lib.f8mi_rms_norm_backward(p, 8, p, 8, None, 0, 4, 8, 0, None, 0, p, None, None, None, 0, None) == 0

    def dropout(x=p, n=4, dt=0, q=0.5, seed=p, out=p):
        return lib.f8mi_dropout(x, None, n, dt, q, seed, out, None)

    assert dropout(x=None) == -1 and dropout(seed=None) == -1 and dropout(seed=p + 4) == -1 and dropout(out=None) == -1 and dropout(n=-1) == -1 and dropout(dt=7) == -1
    assert dropout(q=1.0) == -1 and dropout(q=-0.5) == -1 and dropout(q=float("nan")) == -1 and dropout(n=0, x=None) == 0

    assert lib.f8mi_adapter_rows(p, 2, 4, 2, p, None) == -1 and lib.f8mi_adapter_rows(p, 8, 4, 0, p, None) == -1 and lib.f8mi_adapter_rows(p + 4, 8, 4, 2, p, None) == -1
    assert lib.f8mi_adapter_rows(p, 8, 4, 2, p + 4, None) == -1 and lib.f8mi_adapter_rows(p, 8, (1 << 24) + 1, 2, p, None) == -2 and lib.f8mi_adapter_rows(p, 8, 4, 32769, p, None) == -2
    assert lib.f8mi_adapter_rows(None, 8, 0, 2, None, None) == 0

    def adapters(m=4, k=8, n=6, r=4, count=2, dt=0, ld=8, x=p, y=None, ldy=6, table=p, ws=None, ws_bytes=0):
        return lib.f8mi_adapters(x, ld, p, p, None, 1.0, table, m, k, n, r, count, dt, y, ldy, p, None, ws, ws_bytes, None)

    assert adapters(m=-1) == -1 and adapters(k=0) == -1 and adapters(dt=3) == -1 and adapters(r=257) == -2 and adapters(x=None) == -1 and adapters(table=None) == -1 and adapters(ld=7) == -1
    assert adapters(y=p, ldy=5) == -1 and adapters(ws=p, ws_bytes=10) == -1 and "workspace" in err() and adapters(m=0) == 0
    assert lib.f8mi_adapters_backward(p, 6, p, 8, p, p, None, 1.0, p, None, 4, 8, 6, 4, 2, 0, None, None, p, 0, p, 1 << 30, None) == -1  # h is needed
    assert lib.f8mi_adapters_backward(p, 6, p, 8, p, p, None, 1.0, p, p, 4, 8, 6, 4, 2, 0, None, None, p, 0, p, 16, None) == -1 and "workspace" in err()
    assert lib.f8mi_adapters_backward(p, 6, p, 8, p, p, None, 1.0, p, p, 4, 8, 6, 4, 2, 0, None, None, None, 0, None, 0, None) == 0


def shapes(outputs):
    return [(tuple(t.shape), t.dtype, t.stride()) for t in outputs]


def test_compiled_operators_have_the_shapes_that_a_compiler_is_told(monkeypatch):
    """The kernels are stood in for by what their wrappers allocate."""
    z = lambda *s, dtype=BF16: torch.zeros(s, dtype=dtype)
    monkeypatch.setattr(_native, "rms_norm", lambda x, w, r, eps: (torch.zeros_like(x), None if r is None else torch.zeros_like(x), z(x.shape[0], dtype=FP32)))
    monkeypatch.setattr(_native, "rms_norm_block", lambda x, w, r, eps: (_native._blocks_alloc(*x.shape, "cpu"), None if r is None else torch.zeros_like(x)))
    monkeypatch.setattr(_native, "rms_norm_backward", lambda dy, s, ds, w, rstd, a, b: (torch.zeros_like(s) if a else None, z(s.shape[1], dtype=s.dtype if w is None else w.dtype) if b else None))
    monkeypatch.setattr(_native, "adapters", lambda x, a, b, t, y, s, f, h: (z(len(x), b.shape[1]), z(len(x), -(-a.shape[1] // 16) * 16, dtype=FP32) if h else None))
    monkeypatch.setattr(_native, "adapters_backward", lambda g, x, a, b, t, s, f, h, p, q, r: (z(len(g), a.shape[2]) if p else None, torch.zeros_like(a) if q else None, torch.zeros_like(b) if r else None))

    def calls():
        x, w, r, rstd = z(5, 200), z(200, dtype=FP32), z(5, 200), z(5, dtype=FP32)
        a, b, table = z(3, 4, 200, dtype=FP32), z(3, 70, 4, dtype=FP32), torch.zeros(ops.adapter_rows_words(5, 3), dtype=torch.int32)
        for res in (None, r):
            yield ops.rms_norm_fwd(x, w, res, 1e-6)
            yield ops.rms_norm_blockwise(x, None, res, 1e-6)
        for need in ((True, True), (True, False), (False, True)):
            yield ops.rms_norm_bwd(x, x, None, w, rstd, *need)
            yield ops.rms_norm_bwd(x, x, r, None, rstd, *need)
            yield ops.adapters_bwd(z(5, 70), x, a, b, table, None, 1.0, z(5, 16, dtype=FP32), *need, True)
            yield ops.adapters_bwd(z(0, 70), z(0, 200), a, b, table, None, 1.0, z(0, 16, dtype=FP32), *need, True)
        for need_h in (False, True):
            yield ops.adapters_fwd(x, a, b, table, None, None, 1.0, need_h)

    real = [shapes(out) for out in calls()]
    with FakeTensorMode():
        fake = [shapes(out) for out in calls()]
    assert real == fake
