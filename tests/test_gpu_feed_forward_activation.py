"""The activation of the gated feed-forward block and its slope in fp32, to a few half
steps: with rows (g, 1), gate (1, 0), up (0, 1) and down 1, every sum is exact, y is
act(g), and the gradient of (g, 1) for ones is (act'(g), act(g)).

Tolerances count half steps (H = 2^-24): one for an operation, two for an exponential
(one unit in the last place), eight for erfc (four). The bf16 path's exponential, the
power of two of a rounded product, is further off than that for a third of the values
of the first activation."""
import math

import pytest
import torch

from helpers import DEV

pytestmark = pytest.mark.gpu
H = 2.0 ** -24


def silu(g):
    """(act, act', how far off either may be)"""
    s = torch.sigmoid(g)
    es = 2 * (1 - s) + 2  # the exponential's part of 1 + e^-g; the sum, the division
    act, slope = g * s, s * (1 + g * (1 - s))
    # 1 - s: s's error and its own; the product and sum with g; the product with s
    inner = g.abs() * (s * es + 0.5) + (1 + g * (1 - s)).abs()
    return act, slope, (es + 1) * act.abs(), s * inner + (es + 1) * slope.abs()


def gelu(g):
    cdf = 0.5 * torch.erfc(-g / math.sqrt(2))
    pdf = torch.exp(-g * g / 2) / math.sqrt(2 * math.pi)
    # erfc; its argument's constant and product, as pdf g of the argument's part
    ecdf = 8 * cdf + 2 * (pdf * g).abs()
    # the exponent g g / 2 and its exponential, the constant, three products and a sum
    return (g * cdf, cdf + g * pdf, g.abs() * ecdf + (g * cdf).abs(),
            ecdf + (pdf * g).abs() * (g * g / 2 + 2 + 4) + (cdf + g * pdf).abs())


@pytest.mark.parametrize("rows", [50, 20011])  # few rows, and tiles
@pytest.mark.parametrize("kind", [silu, gelu])
def test_activation(kind, rows):
    from riemannengine import nn
    reach = 80.0 if kind is silu else 12.0  # results above fp32's smallest normal ones
    g = torch.linspace(-reach, reach, rows, device=DEV)
    x = torch.stack([g, torch.ones_like(g)], 1).requires_grad_()
    gate, up = (torch.tensor([v], device=DEV) for v in ([1.0, 0.0], [0.0, 1.0]))
    y = nn.gated_feed_forward(x, gate, up, torch.ones(1, 1, device=DEV), kind.__name__)
    dx, = torch.autograd.grad(y, x, torch.ones_like(y))
    act, slope, e_act, e_slope = kind(g.double())
    for got, want, off, name in ((y.detach()[:, 0], act, e_act, "act"),
                                 (dx[:, 0], slope, e_slope, "act'"), (dx[:, 1], act, e_act, "u")):
        over = (got.double() - want).abs() - H * off - 1e-37
        assert over.max() <= 0, (name, float(over.max()), float(g[over.argmax()]))
