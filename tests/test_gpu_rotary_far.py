"""Rotation at far positions: the angle is the fp64 product of position and
frequency, however many turns that is, and its cosine and sine are off by no more
than at near ones.

The oracle's cosines and sines are math.cos and math.sin of that product on the
host, in fp64. Tolerance: a result's rounding, half a step of fp32; a product and
a sum of two, three half steps of the pair's magnitude; and the angle's, whose part
of a turn is rounded to fp32 (2^-26 of a turn, 2 pi 2^-26 < 2^-23) before a
cosine and a sine within 2^-23."""
import math

import pytest
import torch

from helpers import DEV

pytestmark = pytest.mark.gpu
STEP = 2.0 ** -24
ANGLE = 2.0 ** -22


def oracle(x, positions, freq, back=False):
    turn = -1.0 if back else 1.0
    angle = [[float(p) * f * turn for f in freq] for p in positions]
    c, s = (torch.tensor([[fn(t) for t in row] for row in angle], dtype=torch.float64)[:, None]
            for fn in (math.cos, math.sin))
    n = len(freq)
    a, b = x[..., :n], x[..., n:2 * n]
    return torch.cat([a * c - b * s, a * s + b * c], -1), (a.abs() + b.abs()).repeat(1, 1, 2)


def places(bits, dtype, generator):
    """48 positions of both signs of about so many bits, the power itself among them."""
    if dtype == torch.float32:
        p = torch.randn(48, generator=generator) * 2.0 ** bits
        p[0] = 2.0 ** bits
        return p
    p = torch.randint(2 ** (bits - 1), 2 ** bits, (48,), generator=generator)
    p[0] = 2 ** bits - 1
    p[1::2] *= -1
    return p.to(dtype)


@pytest.mark.parametrize("bits,dtype", [
    (10, torch.int32), (24, torch.float32), (31, torch.int32), (31, torch.int64),
    (40, torch.int64), (40, torch.float32), (47, torch.int64), (53, torch.int64),
])
def test_far_positions(bits, dtype):
    from riemannengine import nn
    g = torch.Generator().manual_seed(bits)
    pairs = 24
    freq = nn.rotary_frequencies([pairs])
    positions = places(bits, dtype, g)
    x, gy = (torch.randn(48, 2, 2 * pairs, generator=g) for _ in range(2))
    leaf = x.to(DEV).requires_grad_()
    y = nn.rotate_heads(leaf, positions.to(DEV), freq, [pairs])
    gx, = torch.autograd.grad(y, leaf, gy.to(DEV))
    # the products are rounded on the device as on the host
    freq = freq.cpu().tolist()
    for got, v, back in ((y.detach(), x, False), (gx, gy, True)):
        want, reach = oracle(v.double(), positions.tolist(), freq, back)
        off = STEP * want.abs() + (ANGLE + 3 * STEP) * reach
        over = (got.cpu().double() - want).abs() - off
        assert over.max() <= 0, (float(over.max()), int(over.argmax()))
