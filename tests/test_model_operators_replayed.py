"""A trace holds registered operators and is replayed with other tensors than it was made with: what does not fit is refused before a kernel reads it.  No GPU needed: the kernels are stood in
for, and none is reached."""
import pytest
import torch
import torch.fx.experimental.proxy_tensor

import float8_experimental_amd as f8
from float8_experimental_amd import _custom_ops_model as ops
from float8_experimental_amd import _native

BF16, FP16, FP32 = torch.bfloat16, torch.float16, torch.float32
z = lambda *s, dtype=BF16: torch.zeros(s, dtype=dtype)


@pytest.fixture
def reached(monkeypatch):
    """Names of the kernels' wrappers that have been called."""
    seen = []
    for name in ("rms_norm", "rms_norm_block", "rms_norm_backward", "dropout", "adapter_rows", "adapters", "adapters_backward"):
        monkeypatch.setattr(_native, name, lambda *args, name=name: seen.append(name) or pytest.fail(f"{name} was reached"))
    return seen


def refused(reached, call, match):
    with pytest.raises(_native.Float8NativeError, match=match):
        call()
    assert not reached


@pytest.mark.parametrize("weight", [z(199), z(201), z(200, dtype=FP16), z(1, 200), z(0)])
def test_norms_of_another_weight(reached, weight):
    x, rstd = z(5, 200), z(5, dtype=FP32)
    for call in (lambda: ops.rms_norm_fwd(x, weight, None, 1e-6), lambda: ops.rms_norm_blockwise(x, weight, None, 1e-6), lambda: ops.rms_norm_bwd(x, x, None, weight, rstd, True, True)):
        refused(reached, call, "weight")


@pytest.mark.parametrize("other", [z(4, 200), z(5, 199), z(1, 200), z(5, 200, dtype=FP32)])
def test_norms_of_another_residual_or_gradient(reached, other):
    x, rstd = z(5, 200), z(5, dtype=FP32)
    refused(reached, lambda: ops.rms_norm_fwd(x, None, other, 1e-6), "residual")
    refused(reached, lambda: ops.rms_norm_blockwise(x, None, other, 1e-6), "residual")
    refused(reached, lambda: ops.rms_norm_bwd(other, x, None, None, rstd, True, True), "gradient")
    refused(reached, lambda: ops.rms_norm_bwd(x, x, other, None, rstd, True, True), "sum's gradient")


def test_norms_of_other_statistics_and_shapes(reached):
    x = z(5, 200)
    for rstd in (z(4, dtype=FP32), z(6, dtype=FP32), z(5), z(5, 1, dtype=FP32)):
        refused(reached, lambda: ops.rms_norm_bwd(x, x, None, None, rstd, True, True), "rstd")
    for bad in (z(200), z(1, 5, 200), z(5, 200, dtype=torch.float64)):
        refused(reached, lambda: ops.rms_norm_fwd(bad, None, None, 1e-6), "no matrix")


def test_dropout_of_another_residual_or_seed(reached):
    x, seed = z(5, 200), torch.zeros(1, dtype=torch.int64)
    for residual in (z(4, 200), z(5, 200, dtype=FP32), z(1000)):
        refused(reached, lambda: ops.dropout_masked(x, residual, seed, 0.5), "residual")
    for other in (torch.zeros(0, dtype=torch.int64), torch.zeros(2, dtype=torch.int64), torch.zeros(1, dtype=torch.int32)):
        refused(reached, lambda: ops.dropout_masked(x, None, other, 0.5), "seed")


def operands(**other):
    return {"x": z(5, 200), "a": z(3, 4, 200), "b": z(3, 70, 4), "table": torch.zeros(ops.adapter_rows_words(5, 3), dtype=torch.int32), "y": z(5, 70), "scale": z(3, dtype=FP32),
            "g": z(5, 70), "h": z(5, 16, dtype=FP32)} | other


ADAPTERS = {
    "more rows": ({"x": z(60, 200), "y": z(60, 70), "g": z(60, 70), "h": z(60, 16, dtype=FP32)}, "table"), "fewer columns": ({"x": z(5, 199)}, "x "), "rows of x": ({"x": z(4, 200)}, "x |table|y "),
    "another rank": ({"a": z(3, 5, 200)}, "a "), "another count": ({"a": z(2, 4, 200)}, "a "), "more adapters": ({"a": z(9, 4, 200), "b": z(9, 70, 4), "scale": z(9, dtype=FP32)}, "table"),
    "two types": ({"a": z(3, 4, 200, dtype=FP32)}, "a "), "a matrix": ({"a": z(4, 200)}, "a "), "no table": ({"table": torch.zeros(0, dtype=torch.int32)}, "table"),
    "a table of 64 bits": ({"table": torch.zeros(ops.adapter_rows_words(5, 3), dtype=torch.int64)}, "table"),
    "a short scale": ({"scale": z(2, dtype=FP32)}, "scale"), "a scale of 16 bits": ({"scale": z(3)}, "scale"),
}


@pytest.mark.parametrize("name", list(ADAPTERS))
def test_adapters_of_other_operands(reached, name):
    other, match = ADAPTERS[name]
    t = operands(**other)
    refused(reached, lambda: ops.adapters_fwd(t["x"], t["a"], t["b"], t["table"], t["y"], t["scale"], 1.0, True), match)
    refused(reached, lambda: ops.adapters_bwd(t["g"], t["x"], t["a"], t["b"], t["table"], t["scale"], 1.0, t["h"], True, True, True), match)


def test_adapters_of_other_rows_beside_them(reached):
    for y in (z(4, 70), z(5, 69), z(5, 70, dtype=FP32)):
        t = operands(y=y)
        refused(reached, lambda: ops.adapters_fwd(t["x"], t["a"], t["b"], t["table"], y, None, 1.0, False), "y ")
    for key, bad in (("g", z(5, 69)), ("g", z(5, 70, dtype=FP16)), ("h", z(5, 15, dtype=FP32)), ("h", z(4, 16, dtype=FP32)), ("h", z(5, 16)), ("h", z(0, dtype=FP32))):
        t = operands(**{key: bad})
        refused(reached, lambda: ops.adapters_bwd(t["g"], t["x"], t["a"], t["b"], t["table"], None, 1.0, t["h"], True, True, True), "gradient|x |h ")


def test_rows_of_numbers_that_are_not_whole(reached):
    for ids in (z(5, dtype=FP32), torch.zeros(5, dtype=torch.int16)):
        refused(reached, lambda: ops.adapter_rows(ids, 3), "ids")


# ---- the rows that a table was made for


@pytest.mark.parametrize("rows, count", [(8, 3), (6, 3), (5, 2), (5, 4), (0, 0)])
def test_a_table_that_is_as_long_but_of_other_rows(reached, rows, count):
    assert ops.adapter_rows_words(8, 3) == ops.adapter_rows_words(6, 3) == ops.adapter_rows_words(5, 3)
    t = operands()
    refused(reached, lambda: ops.adapters_fwd(t["x"], t["a"], t["b"], t["table"], t["y"], None, 1.0, True, rows, count), f"table of {rows} rows and {count} adapters")
    refused(reached, lambda: ops.adapters_bwd(t["g"], t["x"], t["a"], t["b"], t["table"], None, 1.0, t["h"], True, True, True, rows, count), f"table of {rows} rows and {count} adapters")


@pytest.fixture
def stand_ins(monkeypatch):
    """The adapters' kernels, on the CPU: (rows of x, rows of the ids that the table was made of) of each call."""
    seen = []

    def adapters(x, a, b, table, y, scale, factor, need_h):
        seen.append((len(x), int(table[0])))
        return torch.zeros(len(x), b.shape[1], dtype=x.dtype), torch.zeros(len(x), 16) if need_h else None

    def adapter_rows(ids, count):
        table = torch.zeros(ops.adapter_rows_words(ids.numel(), count), dtype=torch.int32)
        table[0] = ids.numel()
        return table

    monkeypatch.setattr(_native, "_require_gpu", lambda t, name: None)
    monkeypatch.setattr(_native, "adapters", adapters)
    monkeypatch.setattr(_native, "adapter_rows", adapter_rows)
    return seen


@pytest.mark.filterwarnings("ignore")
def test_traces_with_a_table_from_outside_take_its_rows_alone(stand_ins):
    a, b, rows = z(2, 4, 8), z(2, 6, 4), f8.AdapterRows(torch.zeros(8, dtype=torch.int64), 2)
    graphed = torch.fx.experimental.proxy_tensor.make_fx(lambda x, a, b: f8.low_rank_adapters(x, a, b, rows))(z(8, 8), a, b)
    traced = torch.jit.trace(lambda x, a, b: f8.low_rank_adapters(x, a, b, rows), (z(8, 8), a, b))
    stand_ins.clear()
    for call in (graphed, traced):
        assert call(z(8, 8), a, b).shape == (8, 6)
        for x, p, q in ((z(5, 8), a, b), (z(9, 8), a, b), (z(8, 8), z(3, 4, 8), z(3, 6, 4)), (z(8, 8), a[:1], b[:1])):
            with pytest.raises(RuntimeError, match="table of 8 rows and 2 adapters"):
                call(x, p, q)
    assert stand_ins == [(8, 8)] * 2


@pytest.mark.filterwarnings("ignore")
def test_traces_that_make_the_table_take_any_rows(stand_ins):
    a, b = z(2, 4, 8), z(2, 6, 4)
    traced = torch.jit.trace(lambda x, ids: f8.low_rank_adapters(x, a, b, f8.AdapterRows(ids, 2)), (z(5, 8), torch.zeros(5, dtype=torch.int64)))
    stand_ins.clear()
    for m in (5, 6, 8, 70, 1):
        assert traced(z(m, 8), torch.zeros(m, dtype=torch.int64)).shape == (m, 6)
    assert stand_ins == [(m, m) for m in (5, 6, 8, 70, 1)]
    with pytest.raises(RuntimeError, match="table of 8 rows"):
        traced(z(5, 8), torch.zeros(8, dtype=torch.int64))
