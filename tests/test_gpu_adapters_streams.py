"""A batch's table that is let go while another stream still reads it: its memory is not handed out again before that stream is done."""
import pytest
import torch
import torch.nn as nn
from torch.overrides import TorchFunctionMode

pytestmark = pytest.mark.gpu
BF16 = torch.bfloat16


@pytest.fixture(scope="module")
def f8():
    import float8_experimental_amd

    return float8_experimental_amd


class Watch(TorchFunctionMode):  # the call goes through the registered operators
    def __torch_function__(self, func, types, args=(), kwargs=None):
        return func(*args, **(kwargs or {}))


def elsewhere(call):
    """What `call` gives on a stream of its own that is busy for some milliseconds first, and that waits for this one."""
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        torch.cuda._sleep(20_000_000)
        return call()


@pytest.mark.parametrize("watched", [False, True])
@pytest.mark.parametrize("grad", [False, True])
def test_a_table_that_another_stream_reads(f8, grad, watched):
    x, a, b = torch.randn(8, 64, device="cuda", dtype=BF16), torch.randn(3, 4, 64, device="cuda", dtype=BF16), torch.randn(3, 128, 4, device="cuda", dtype=BF16)
    ids = torch.tensor([0, 1, 2, -1, 1, 0, 2, 2], device="cuda")
    rows = f8.AdapterRows(ids, 3)
    want = f8.low_rank_adapters(x, a, b, rows)
    a.requires_grad_(grad)
    torch.cuda.synchronize()
    at, words = rows.table.data_ptr(), rows.table.numel()

    def call():
        if watched:
            with Watch():
                return f8.low_rank_adapters(x, a, b, rows).detach()
        return f8.low_rank_adapters(x, a, b, rows).detach()  # (nothing keeps the table for backward)

    got = elsewhere(call)
    del rows
    taken = [torch.empty(words, dtype=torch.int32, device="cuda") for _ in range(256)]  # (nothing is written there)
    assert all(t.data_ptr() != at for t in taken)
    torch.cuda.synchronize()
    assert torch.equal(got, want)


def test_batches_one_after_another_on_another_stream(f8):
    torch.manual_seed(0)
    layer = f8.AdaptedLinear(nn.Linear(64, 128, device="cuda", dtype=BF16), 3, 4).eval()
    with torch.no_grad():
        layer.adapter_b.normal_()
        batches = [(torch.randn(m, 64, device="cuda", dtype=BF16), torch.arange(m, device="cuda") * 7 % 4 - 1) for m in (8, 7, 6, 5, 8, 5)]
        want = []
        for x, ids in batches:
            f8.select_adapters(layer, ids)
            want.append(layer(x))
        torch.cuda.synchronize()
        side, got = torch.cuda.Stream(), []
        for x, ids in batches:
            f8.select_adapters(layer, ids)  # on this stream, which does not wait for the other
            side.wait_stream(torch.cuda.current_stream())
            with torch.cuda.stream(side):
                torch.cuda._sleep(2_000_000)
                got.append(layer(x))
        torch.cuda.synchronize()
    assert all(torch.equal(p, q) for p, q in zip(got, want))


def test_a_captured_graph_reads_a_table_from_outside(f8):
    """Made on another stream than the capturing one, read at each replay, and let go once the graph is."""
    torch.manual_seed(1)
    layer = f8.AdaptedLinear(nn.Linear(64, 128, device="cuda", dtype=BF16), 3, 4).eval()
    x, ids = torch.randn(9, 64, device="cuda", dtype=BF16), torch.arange(9, device="cuda") % 4 - 1
    with torch.no_grad():
        layer.adapter_b.normal_()
        f8.select_adapters(layer, ids)
        layer(x)
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = layer(x)
        for i in range(3):
            x.copy_(torch.randn(9, 64, generator=torch.Generator().manual_seed(i)).to(BF16))
            want = layer(x)
            graph.replay()
            torch.cuda.synchronize()
            assert torch.equal(out, want)
        del graph, out
        f8.select_adapters(layer, ids[:5])
        assert layer(x[:5]).isfinite().all()
