"""Inputs that the transformer functions cannot serve are refused, never
answered in part."""
import pytest
import torch
import torch.autograd.forward_ad as forward_ad

import riemannengine as rie
from helpers import DEV

pytestmark = pytest.mark.gpu


def test_forward_mode_tangents_are_refused():
    """As by the convolutions: a result without its tangent would be wrong."""
    nn = rie.nn
    x = torch.randn(12, 4, 16, device=DEV)
    rows = x.view(12, 64)
    w, b = torch.ones(64, device=DEV), torch.zeros(64, device=DEV)
    o = torch.tensor([0, 5, 12], dtype=torch.int32, device=DEV)
    ids = torch.zeros(3, dtype=torch.int64, device=DEV)
    with forward_ad.dual_level():
        for leaf, call in [
            (x, lambda t: nn.packed_attention(t, x, x, o)),
            (x, lambda t: nn.packed_attention(x, t, x, o)),
            (x, lambda t: nn.packed_attention(x, x, t, o, causal=True)),
            (rows, lambda t: nn.layer_norm(t, w, b)),
            (w, lambda t: nn.layer_norm(rows, t, b)),
            (b, lambda t: nn.layer_norm(rows, w, t)),
            (rows, lambda t: nn.embedding(ids, t)),
        ]:
            dual = forward_ad.make_dual(leaf, torch.ones_like(leaf))
            for grad in (True, False):
                with torch.set_grad_enabled(grad), pytest.raises(RuntimeError, match="jvp"):
                    call(dual)
        # without tangents nothing changes
        assert nn.packed_attention(x, x, x, o).shape == x.shape


def test_channels_past_32_bits():
    """2^32 + 8 channels are 8 in 32 bits."""
    one = torch.zeros(1, device=DEV, dtype=torch.bfloat16)
    wide = one.expand(2 ** 32 + 8)
    ids = torch.zeros(1, dtype=torch.int64, device=DEV)
    with pytest.raises(RuntimeError, match="channels"):
        rie.nn.layer_norm(torch.zeros(2 ** 32 + 8, device=DEV, dtype=torch.bfloat16))
    with pytest.raises(RuntimeError, match="channels"):
        rie.nn.embedding(ids, wide[None])


@pytest.mark.parametrize("eps", [0.0, 1e-60, -1e-5, float("nan")])
def test_eps_that_fp32_takes_for_zero(eps):
    """A constant row would come out as 0 / 0."""
    with pytest.raises(RuntimeError, match="eps"):
        rie.nn.layer_norm(torch.ones(3, 8, device=DEV), eps=eps)


@pytest.mark.parametrize("scale", [1e39, -1e300, float("nan"), float("inf")])
def test_scales_that_fp32_takes_for_infinity(scale):
    ids = torch.zeros(4, dtype=torch.int64, device=DEV)
    with pytest.raises(RuntimeError, match="finite"):
        rie.nn.embedding(ids, torch.ones(3, 8, device=DEV), scale)


def test_negative_key_heads():
    with pytest.raises(RuntimeError, match="multiple"):
        rie.nn.RiemannAttention(64, 4, -2)
    with pytest.raises(RuntimeError, match="multiple"):
        rie.nn.AttentionBlock(64, 4, kv_heads=-1)
    assert list(rie.nn.RiemannAttention(64, 4, 0).parameters())
