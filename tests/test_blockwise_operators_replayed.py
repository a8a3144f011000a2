"""The operators of layer norm and of the blockwise linears, as a replayed trace calls them: what does not fit is refused before a kernel reads it.  No GPU needed: the kernels are stood in for,
and none is reached."""
import pytest
import torch

from float8_experimental_amd import _custom_ops_norm_blockwise as ops
from float8_experimental_amd import _native

BF16, FP16, FP32, E4M3, U8 = torch.bfloat16, torch.float16, torch.float32, torch.float8_e4m3fn, torch.uint8
z = lambda *s, dtype=BF16: torch.zeros(s, dtype=dtype)


@pytest.fixture
def refused(monkeypatch):
    for name in ("layer_norm", "layer_norm_backward", "block_cast", "block_gemm"):
        monkeypatch.setattr(_native, name, lambda *args, name=name, **kw: pytest.fail(f"{name} was reached"))

    def check(call, match):
        with pytest.raises(_native.Float8NativeError, match=match):
            call()

    return check


@pytest.mark.parametrize("p", [z(199), z(201), z(200, dtype=FP16), z(1, 200), z(0)])
def test_layer_norm_of_other_parameters(refused, p):
    x, w = z(5, 200), z(200)
    refused(lambda: ops.layer_norm_fwd(x, p, None, 1e-5), "weight")
    refused(lambda: ops.layer_norm_fwd(x, w, p, 1e-5), "bias")
    refused(lambda: ops.layer_norm_bwd(x, x, p, BF16, z(5, 2, dtype=FP32), True, True, True), "weight")
    refused(lambda: ops.layer_norm_fwd(x, w, z(200, dtype=FP32), 1e-5), "bias")  # the kernels read both in one type


def test_layer_norm_of_other_gradients_and_statistics(refused):
    x, w, stats = z(5, 200), z(200), z(5, 2, dtype=FP32)
    for g in (z(4, 200), z(5, 199), z(5, 200, dtype=FP32)):
        refused(lambda: ops.layer_norm_bwd(g, x, w, BF16, stats, True, True, True), "gradient")
    for s in (z(4, 2, dtype=FP32), z(5, 2), z(5, dtype=FP32)):
        refused(lambda: ops.layer_norm_bwd(x, x, w, BF16, s, True, True, True), "statistics")
    refused(lambda: ops.layer_norm_fwd(z(200), None, None, 1e-5), "no matrix")


def test_blockwise_linear_of_other_copies(refused):
    m, k, n = 5, 200, 70
    kept = {"xt": z(*ops._data_shape(k, m), dtype=E4M3), "xts": z(*ops._scales_shape(k, m), dtype=U8), "w": z(*ops._data_shape(k, n), dtype=E4M3), "ws": z(*ops._scales_shape(k, n), dtype=U8)}
    for name, bad in (("xt", z(*ops._data_shape(k, 200), dtype=E4M3)), ("xt", z(*ops._data_shape(k, m))), ("xts", z(*ops._scales_shape(k, 200), dtype=U8)), ("w", z(0, dtype=E4M3)),
                      ("w", z(*ops._data_shape(k, n), dtype=U8)), ("ws", z(1, 1, dtype=U8))):
        t = kept | {name: bad}
        refused(lambda: ops.blockwise_linear_bwd(z(m, n), t["xt"], t["xts"], t["w"], t["ws"], k, BF16, None, True, True), "x|weight")
