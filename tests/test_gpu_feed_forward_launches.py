"""The gated feed-forward block at sizes that reach every launch of its products and
their joins (tests/test_abi_gated_plan_cpu.py shows that they do), against its
definition in fp64."""
import pytest
import torch

from feed_forward_launches import SIZES
from feed_forward_reference import assert_close, reference

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype,sizes", [(d, s) for d in SIZES for s in SIZES[d]],
                         ids=lambda v: "x".join(map(str, v)) if isinstance(v, tuple) else
                         str(v)[6:])
def test_sizes(dtype, sizes):
    from riemannengine import nn
    n, channels, hidden, outputs = sizes
    kind = "gelu" if n % 2 else "silu"
    g = torch.Generator(device="cuda").manual_seed(sum(sizes))

    def normal(*shape, scale=1.0):
        return (torch.randn(shape, generator=g, device="cuda") * scale).to(dtype)

    leaves = [normal(n, channels), normal(hidden, channels, scale=channels ** -0.5),
              normal(hidden, channels, scale=channels ** -0.5),
              normal(outputs, hidden, scale=hidden ** -0.5)]
    grad_y = normal(n, outputs)
    leaves = [t.requires_grad_() for t in leaves]
    y = nn.gated_feed_forward(*leaves, kind)
    got = [y.detach(), *torch.autograd.grad(y, leaves, grad_y)]
    want = reference(*leaves, kind, grad_y)
    for a, b, name in zip(got, want, ("y", "grad_x", "grad_gate", "grad_up", "grad_down")):
        assert_close(a, b, name)
