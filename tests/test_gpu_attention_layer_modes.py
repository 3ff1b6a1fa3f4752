"""RiemannAttention's rotation keeps its frequencies from one call for the next:
whatever mode the first call runs in, those behind it get what they would
have got as the first."""
import pytest
import torch

import riemannengine as rie
from helpers import DEV

pytestmark = pytest.mark.gpu


def rows(n=90, seed=0):
    g = torch.Generator().manual_seed(seed)
    c = torch.unique(torch.stack([torch.randint(0, 2, (4 * n,), generator=g)]
                                 + [torch.randint(-40, 40, (4 * n,), generator=g)
                                    for _ in range(3)], 1), dim=0)[:n]
    return c.int().to(DEV), torch.randn(n, 64, generator=g).to(DEV)


def layer(head_norm):
    torch.manual_seed(1)
    attention = rie.nn.RiemannAttention(64, 4, 2, rotary=[3, 3, 2], head_norm=head_norm)
    attention.to(DEV)
    return attention


def step(attention, coords, x):
    """The output and all gradients of one training step."""
    x = x.clone().requires_grad_()
    out = attention(rie.SparseTensor(x, coords)).F
    return [out, *torch.autograd.grad(out.square().sum(),
                                      [x, *attention.named_parameters().values()])]


@pytest.mark.parametrize("mode", [torch.inference_mode, torch.no_grad])
@pytest.mark.parametrize("head_norm", [False, True])
def test_training_behind_an_evaluation(head_norm, mode):
    coords, x = rows()
    want = step(layer(head_norm), coords, x)
    attention = layer(head_norm)
    with mode():
        evaluated = attention(rie.SparseTensor(x, coords)).F
        assert torch.equal(evaluated, want[0])
    for got, ref in zip(step(attention, coords, x), want):
        assert torch.equal(got, ref)
    with mode():
        assert torch.equal(attention(rie.SparseTensor(x, coords)).F, want[0])


def test_frequencies_outlive_another_streams_kernels():
    """The layer is dropped while a second stream, which called it, has work queued:
    its frequencies, from the first stream's memory, are held until that is done."""
    coords, x = rows()
    attention = layer(False)
    a = torch.randn(8192, 8192, device=DEV)
    b = torch.empty_like(a)
    side = torch.cuda.Stream()
    with torch.no_grad():
        attention(rie.SparseTensor(x, coords))
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            out = attention(rie.SparseTensor(x, coords)).F
            for _ in range(10):  # some 70 ms
                torch.mm(a, a, out=b)

        def held():  # blocks that are free but for another stream
            stats = torch.cuda.memory_stats()
            return stats["active.all.current"] - stats["allocation.all.current"]

        before = held()
        del attention
        assert held() == before + 1
    torch.cuda.synchronize()
    assert out.isfinite().all()
