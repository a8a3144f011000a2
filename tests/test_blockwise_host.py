"""What the blockwise linears, layer norm and clipping refuse or decide on the host: no GPU needed."""
import ctypes

import pytest
import torch
import torch.nn as nn

import float8_experimental_amd as f8
from float8_experimental_amd import _native

BLK = f8.CastConfig(scaling_type=f8.ScalingType.BLOCKWISE)


def test_config_is_blockwise_for_all_three_tensors_or_none():
    config = f8.Float8LinearConfig(cast_config_input=BLK, cast_config_weight=BLK, cast_config_grad_output=BLK)
    assert f8.ScalingType.BLOCKWISE.short_str() == "blk" and not f8.linear_requires_sync(config)
    with pytest.raises(ValueError, match="all three"):
        f8.Float8LinearConfig(cast_config_input=BLK)
    with pytest.raises(ValueError, match="Float8BlockwiseLinear"):
        f8.Float8Linear(4, 4, config=config)
    model = f8.convert_to_float8_training(nn.Sequential(nn.Linear(4, 8), nn.Linear(8, 4, bias=False)), config=config)
    assert [type(m) for m in model] == [f8.Float8BlockwiseLinear] * 2 and model[1].bias is None
    assert type(f8.convert_to_float8_training(nn.Linear(4, 8))) is f8.Float8Linear
    for kw in ({"emulate": True}, {"enable_fsdp_float8_all_gather": True}):
        with pytest.raises(NotImplementedError):
            f8.convert_to_float8_training(nn.Linear(4, 8), config=f8.Float8LinearConfig(cast_config_input=BLK, cast_config_weight=BLK, cast_config_grad_output=BLK, **kw))


def test_tensors_on_the_cpu_are_refused():
    x, w = torch.ones(4, 8), torch.ones(6, 8)
    for call in (lambda: f8.blockwise_linear(x, w), lambda: f8.layer_norm(x, 8), lambda: f8.Float8BlockwiseInferenceLinear.from_float(nn.Linear(8, 6)),
                 lambda: f8.clip_grads([x], 1.0), lambda: f8.grad_norm([x])):
        with pytest.raises(_native.Float8NativeError):
            call()
    with pytest.raises(ValueError, match="norm_type"):
        f8.grad_norm([x], 3.0)


def test_arguments_of_the_library_are_checked_on_the_host():
    lib, p = _native.lib(), 1 << 20  # no address is read
    err = lambda: lib.f8mi_last_error().decode()
    assert lib.f8mi_block_scale_bytes(130, 200) == 2 * 256 and lib.f8mi_block_scale_bytes(0, 5) == 0
    job = lambda **kw: (_native.BlockCastJob * 1)(_native.BlockCastJob(**{**dict(x=p, rows=4, cols=8, ld=8, dtype=0, square=0, out=p, out_scales=p), **kw}))
    for kw, said in ((dict(rows=0), "shape"), (dict(ld=7), "shape"), (dict(dtype=5), "dtype"), (dict(out=None), "null"), (dict(out_scales=None), "null"), (dict(out=p + 8), "aligned"),
                     (dict(x=p + 1), "aligned"), (dict(out_t_scales=p), "null")):
        assert lib.f8mi_block_cast(job(**kw), 1, None) == -1 and said in err(), kw
    assert lib.f8mi_block_cast(job(), 3, None) == -1 and lib.f8mi_block_cast(job(rows=1 << 40, cols=1 << 40, ld=1 << 40), 1, None) == -2

    def gemm(m=4, n=8, k=128, ldc=8, dt=0, tr=0, a=p, c=p):
        return lib.f8mi_block_gemm(a, p, p, p, tr, m, n, k, c, dt, ldc, None, None, 0, None)

    assert gemm(m=-1) == -1 and gemm(ldc=7) == -1 and gemm(dt=3) == -1 and gemm(k=100) == -1 and gemm(a=None) == -1 and gemm(a=p + 4) == -1 and gemm(k=1 << 30) == -2
    assert gemm(tr=1) == -2 and "multiple of 128" in err()
    assert gemm(m=0) == 0

    assert lib.f8mi_layer_norm(None, 4, 8, 8, 0, None, None, 0, 1e-5, p, None, None) == -1 and lib.f8mi_layer_norm(p, 4, 8, 7, 0, None, None, 0, 1e-5, p, None, None) == -1
    assert lib.f8mi_layer_norm(p, 4, 8, 8, 0, None, None, 1, 1e-5, p, None, None) == -1 and "parameters" in err()
    assert lib.f8mi_layer_norm(p, 4, 0, 8, 0, None, None, 0, 1e-5, p, None, None) == -1 and lib.f8mi_layer_norm(p, 0, 8, 8, 0, None, None, 0, 1e-5, p, None, None) == 0
    assert lib.f8mi_layer_norm_backward(p, 8, p, 8, 4, 8, 0, None, 0, p, p, p, None, None, 0, None) == -1 and "workspace" in err()
    assert lib.f8mi_layer_norm_backward(p, 8, p, 8, 4, 8, 0, None, 0, None, p, None, None, None, 0, None) == -1

    grad = lambda **kw: (_native.Grad * 1)(_native.Grad(**{**dict(x=p, out=p, n=5, dtype=0, out_dtype=0), **kw}))
    clip = lambda g, count=1, kind=2, norm=p, ws=p, size=1 << 20: lib.f8mi_grad_clip(g, count, kind, 1.0, 1, norm, ws, size, None)
    for g in (grad(n=-1), grad(dtype=4), grad(x=None), grad(out=None), grad(out_dtype=2)):
        assert clip(g) == -1 and "tensor 0" in err()
    assert clip(grad(), kind=3) == -1 and clip(None) == -1 and clip(grad(), norm=None) == -1 and clip(grad(), size=8) == -1 and "workspace" in err()
    assert lib.f8mi_grad_clip_workspace_bytes(1) == 8192 and lib.f8mi_grad_clip_workspace_bytes(96 * 2000) >= 2000 * 8
    assert isinstance(ctypes.sizeof(_native.Grad), int)
