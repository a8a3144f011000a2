"""The library's gradients of low-rank adapters for a batch without rows: zeros, whole."""
import pytest
import torch

pytestmark = pytest.mark.gpu
BF16, FP16, FP32 = torch.bfloat16, torch.float16, torch.float32


@pytest.mark.parametrize("which", [(True, True), (True, False), (False, True)])
@pytest.mark.parametrize("dtype", [BF16, FP16, FP32])
@pytest.mark.parametrize("shape", [(3, 4, 200, 70), (1, 1, 1, 1), (5, 7, 4097, 333)])
def test_gradients_of_no_rows(shape, dtype, which):
    from float8_experimental_amd import _native

    count, r, k, n = shape
    # in the middle of other values, which stay
    buffers = [torch.full((count * r * size + 2,), 7.0, device="cuda", dtype=dtype) for size in (k, n)]
    da, db = (b[1:].data_ptr() if wanted else None for b, wanted in zip(buffers, which))
    stream = torch.cuda.current_stream().cuda_stream
    assert _native.lib().f8mi_adapters_backward(None, n, None, k, None, None, None, 1.0, None, None, 0, k, n, r, count, _native._DT[dtype], None, da, db, _native._DT[dtype], None, 0, stream) == 0
    for b, wanted in zip(buffers, which):
        assert (b[1:-1] == (0.0 if wanted else 7.0)).all() and b[0] == 7.0 and b[-1] == 7.0


def test_gradients_of_no_rows_in_a_graph():
    from float8_experimental_amd import _native

    da, db = torch.empty(2, 4, 64, device="cuda"), torch.empty(2, 32, 4, device="cuda")
    call = lambda: _native.lib().f8mi_adapters_backward(None, 32, None, 64, None, None, None, 1.0, None, None, 0, 64, 32, 4, 2, 2, None, da.data_ptr(), db.data_ptr(), 2, None, 0,
                                                        torch.cuda.current_stream().cuda_stream)
    assert call() == 0
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        assert call() == 0
    for _ in range(3):
        da.fill_(7.0), db.fill_(7.0)
        graph.replay()
        torch.cuda.synchronize()
        assert (da == 0).all() and (db == 0).all()


def test_an_unknown_type_is_refused_without_rows_too():
    from float8_experimental_amd import _native

    p = 1 << 20  # no address is read
    assert _native.lib().f8mi_adapters_backward(None, 32, None, 64, None, None, None, 1.0, None, None, 0, 64, 32, 4, 2, 2, None, p, None, 3, None, 0, None) == -1
    assert _native.lib().f8mi_adapters_backward(None, 32, None, 64, None, None, None, 1.0, None, None, 0, 64, 32, 4, 2, 2, p, None, None, 2, None, 0, None) == 0
