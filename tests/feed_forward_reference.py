"""The gated feed-forward block from its definition in fp64, with how far a
kernel's results may be off: every rounding counts half a step of its type,
every fp32 sum of k products k + 2 steps of 2^-24 of the sum of magnitudes."""
import math

import torch

STEP = 2.0 ** -24          # half a step of fp32
KEPT = 2.0 ** -17          # g and u kept to 16 significant bits (bf16)
ACT = 2.0 ** -17           # exponential and reciprocal at |g| up to 30
SLOPE, CURVE = 1.13, 1.0   # the activations' largest first and second derivatives


def half_step(dtype):
    return torch.finfo(dtype).eps / 2


def activation(g, kind):
    """act(g) and act'(g)."""
    if kind == "silu":
        s = torch.sigmoid(g)
        return g * s, s * (1 + g * (1 - s))
    cdf = 0.5 * torch.erfc(-g / math.sqrt(2))
    return g * cdf, cdf + g * torch.exp(-g * g / 2) / math.sqrt(2 * math.pi)


def reference(x, gate, up, down, kind, grad_y=None):
    """[(value, how far off it may be)] of y, and with grad_y of the gradients
    of x, gate, up and down."""
    dtype = x.dtype
    half = half_step(dtype)
    low = dtype != torch.float32  # h, dg and du are rounded
    x, gate, up, down = (t.detach().double() for t in (x, gate, up, down))
    n, (hidden, channels), outputs = x.shape[0], gate.shape, down.shape[0]

    def prod(a, b, ea, eb, k):
        """a @ b, and its error from the operands' and the sum's."""
        off = ea @ b.abs() + a.abs() @ eb + (k + 2) * STEP * (a.abs() @ b.abs())
        return a @ b, off

    zero = torch.zeros_like
    g, eg = prod(x, gate.t(), zero(x), zero(gate.t()), channels)
    u, eu = prod(x, up.t(), zero(x), zero(up.t()), channels)
    a, da = activation(g, kind)
    h = a * u
    eh = (SLOPE * eg * u.abs() + a.abs() * eu + SLOPE * eg * eu
          + (ACT + (half if low else STEP)) * h.abs())
    y, ey = prod(h, down.t(), eh, zero(down.t()), hidden)
    results = [(y, ey + half * y.abs())]
    if grad_y is None:
        return results
    dy = grad_y.detach().double()
    dh, edh = prod(dy, down, zero(dy), zero(down), outputs)
    if low:
        eg, eu = eg + KEPT * g.abs(), eu + KEPT * u.abs()
    dg, du = dh * u * da, dh * a
    one = ACT + (half if low else STEP)
    edg = (edh * (u * da).abs() + (dh * da).abs() * eu + (dh * u).abs() * (CURVE * eg + ACT)
           + one * dg.abs())
    edu = edh * a.abs() + dh.abs() * SLOPE * eg + one * du.abs()
    dx = dg @ gate + du @ up
    edx = (edg @ gate.abs() + edu @ up.abs()
           + (2 * hidden + 2) * STEP * (dg.abs() @ gate.abs() + du.abs() @ up.abs()))
    results.append((dx, edx + half * dx.abs()))
    for d, ed in ((dg, edg), (du, edu)):
        w, ew = prod(d.t(), x, ed.t(), zero(x), n)
        results.append((w, ew + half * w.abs()))
    w, ew = prod(dy.t(), h, zero(dy.t()), eh, n)
    results.append((w, ew + half * w.abs()))
    return results


def assert_close(got, want, name):
    value, off = want
    assert got.shape == value.shape and torch.isfinite(got).all(), name
    # what one more rounding of the smallest values (denormals) may add
    over = ((got.double() - value).abs() - off - 1e-37) if value.numel() else value
    assert not value.numel() or over.max() <= 0, (
        name, float(over.max()), int(over.argmax()), tuple(value.shape))
