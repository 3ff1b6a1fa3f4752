"""Embedding gradients whose time must follow their work, not a few waves': a
few ids in a large table, a few classes, widths that end inside a 16-byte
chunk."""
import pytest
import torch

from riemannengine_amd import abi
from helpers import DEV

pytestmark = pytest.mark.gpu

F32, BF16 = torch.float32, torch.bfloat16


def best(call):
    """Least time of a call, microseconds."""
    times = []
    for _ in range(8):
        start, end = (torch.cuda.Event(enable_timing=True) for _ in range(2))
        start.record()
        call()
        end.record()
        end.synchronize()
        times.append(start.elapsed_time(end) * 1e3)
    return min(times[1:])


def replayed(call):
    """Time of a call without the host's, microseconds: ten in a graph."""
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        call()
    torch.cuda.current_stream().wait_stream(stream)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        for _ in range(10):
            call()
    return best(graph.replay) / 10


@pytest.mark.parametrize("n", [0, 1, 50, 5000])
def test_a_few_ids_in_a_large_table(n):
    """A million rows of 16: within 100 us of clearing the table (64 MB, and 4
    MB of positions; a wave on its own would take half a millisecond)."""
    V, C = 1_000_000, 16
    ids = torch.randint(0, V, (n,), device=DEV)
    dy = torch.randn(n, C, device=DEV)
    table = torch.empty(V, C, device=DEV)
    clear = replayed(lambda: table.zero_())
    got = replayed(lambda: abi.embed_backward(dy, ids, V))
    print("few ids", n, clear, got, flush=True)
    assert got <= clear + 100
    want = torch.zeros(V, C, dtype=torch.float64, device=DEV).index_add_(0, ids, dy.double())
    assert (abi.embed_backward(dy, ids, V).double() - want).abs().max() <= 1e-5


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("n,V", [(1000, 16), (3500, 56)])
def test_classes_of_62_ids_each(dtype, n, V):
    """Rows just short of being cut into parts: at most 1.5 times all ids in one
    class, which are, and 5 us."""
    dy = torch.randn(n, 512, device=DEV).to(dtype)
    ids = torch.arange(n, device=DEV) % V
    one = replayed(lambda: abi.embed_backward(dy, torch.zeros_like(ids), 1))
    got = replayed(lambda: abi.embed_backward(dy, ids, V))
    print("classes", n, V, dtype, one, got, flush=True)
    assert got <= 1.5 * one + 5


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("n,V,C", [(3780, 51, 383), (900, 21, 1677), (20000, 30, 63)])
def test_widths_that_end_inside_a_chunk(dtype, n, V, C):
    """At most 1.1 times the next width of whole chunks, and 5 us."""
    ids = torch.arange(n, device=DEV) % V
    times = []
    for width in (C, (C + 7) // 8 * 8):
        dy = torch.randn(n, width, device=DEV).to(dtype)
        times.append(replayed(lambda: abi.embed_backward(dy, ids, V)))
    print("widths", n, V, C, dtype, times, flush=True)
    assert times[0] <= 1.1 * times[1] + 5
