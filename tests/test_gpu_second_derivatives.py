"""Second derivatives through the transformer operators whose backward runs with
create_graph: the first ones are what they are without it, and to go
through them again is an error, not a result that lacks a part."""
import pytest
import torch

from helpers import DEV

pytestmark = pytest.mark.gpu


def attention(**options):
    def call(nn, dtype, g):
        q = torch.randn(40, 4, 16, generator=g, device=DEV).to(dtype)
        k, v = (torch.randn(40, 2, 16, generator=g, device=DEV).to(dtype) for _ in range(2))
        offsets = torch.tensor([0, 13, 40], dtype=torch.int32, device=DEV)
        return lambda *t: nn.packed_attention(*t, offsets, causal=True, **options), [q, k, v]
    return call


def layer_norm(nn, dtype, g):
    x = torch.randn(20, 24, generator=g, device=DEV).to(dtype)
    w, b = (torch.randn(24, generator=g, device=DEV) for _ in range(2))
    return lambda *t: nn.layer_norm(*t), [x, w, b]


def embedding(nn, dtype, g):
    table = torch.randn(9, 24, generator=g, device=DEV).to(dtype)
    ids = torch.randint(0, 9, (20,), generator=g, device=DEV)
    return lambda t: nn.embedding(ids, t), [table]


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("make,name", [(attention(), "attention"),
                                       (attention(window=5, sinks=2), "attention"),
                                       (layer_norm, "layer norm"), (embedding, "embedding")])
def test_second_derivatives(make, name, dtype):
    from riemannengine import nn
    g = torch.Generator(device=DEV).manual_seed(0)
    call, inputs = make(nn, dtype, g)
    leaves = [t.requires_grad_() for t in inputs]
    y = call(*leaves)
    loss = y.float().square().sum()
    want = torch.autograd.grad(loss, leaves, retain_graph=True)
    got = torch.autograd.grad(loss, leaves, create_graph=True)
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    assert not any(t.requires_grad for t in want)
    # a penalty on the gradients beside the loss
    both = loss + sum(t.float().square().sum() for t in got)
    with pytest.raises(RuntimeError, match=f"{name} has no second derivatives"):
        torch.autograd.grad(both, leaves)


def test_gradients_that_depend_on_nothing_recorded():
    """The embedding's gradient is linear in that of its rows: with a constant one
    there is nothing to differentiate, and nothing to refuse."""
    from riemannengine import nn
    call, (table,) = embedding(nn, torch.float32, torch.Generator(device=DEV).manual_seed(0))
    table.requires_grad_()
    y = call(table)
    grad, = torch.autograd.grad(y, table, torch.ones_like(y), create_graph=True)
    assert not grad.requires_grad
