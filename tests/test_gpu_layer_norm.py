"""rhip_ln_forward / rhip_ln_backward and riemannengine.nn.layer_norm against
the definition in fp64: widths of every kernel variant and both their edges,
odd widths, unaligned and strided rows, few and many rows, rows around a large
mean, refusals, gradients against differences.

Bounds, u = 2^-8 for bf16 results (unit roundoff) and 2^-23 for fp32 ones, and
e = 2^-24 (C + 16) for the fp32 sums of C terms, worst case:
  y       u |y| + e (1 + |xhat|) |w| (1 + |mean| rstd) + 2^-24 |b|
  grad_x  u |dx| + 4 e rstd (|g| + mean |g| + |xhat| mean |g xhat|) (1 + |mean| rstd)
  grad_w  2^-24 (n + 16) sum |dy| |xhat| + sum |dy| (xhat's error)
"""
import numpy as np
import pytest
import torch

import riemannengine as rie
from riemannengine_amd import abi
from helpers import DEV

pytestmark = pytest.mark.gpu

F32, BF16 = torch.float32, torch.bfloat16
U = {F32: 2.0 ** -23, BF16: torch.finfo(BF16).eps / 2}


def reference(x, w, b, dy, eps, dtype):
    x, w, b, dy = (t.detach().double().cpu().numpy() for t in (x, w, b, dy))
    n, C = x.shape
    u, e = U[dtype], 2.0 ** -24 * (C + 16)
    mean = x.mean(1, keepdims=True)
    rstd = 1 / np.sqrt(((x - mean) ** 2).mean(1, keepdims=True) + eps)
    hat = (x - mean) * rstd
    far = 1 + np.abs(mean) * rstd
    y = hat * w + b
    g = dy * w
    m1, m2 = g.mean(1, keepdims=True), (g * hat).mean(1, keepdims=True)
    dx = rstd * (g - m1 - hat * m2)
    hat_err = e * (1 + np.abs(hat)) * far
    a1, a2 = np.abs(g).mean(1, keepdims=True), np.abs(g * hat).mean(1, keepdims=True)
    return {
        "y": (y, u * np.abs(y) + hat_err * np.abs(w) + 2.0 ** -24 * np.abs(b)),
        "gx": (dx, u * np.abs(dx) + 4 * e * rstd * (np.abs(g) + a1 + (1 + np.abs(hat)) * a2
                                                    + np.abs(hat) * a1) * far),
        "gw": ((dy * hat).sum(0), 2.0 ** -24 * (n + 16) * (np.abs(dy * hat)).sum(0)
               + (np.abs(dy) * hat_err).sum(0) + 2.0 ** -23 * np.abs((dy * hat).sum(0))),
        "gb": (dy.sum(0), 2.0 ** -24 * (n + 16) * np.abs(dy).sum(0)),
    }


def within(got, want, what):
    val, err = want
    diff = np.abs(got.detach().double().cpu().numpy() - val)
    bad = ~(diff <= 1.01 * err + 1e-30)
    assert not bad.any(), (what, int(bad.sum()), float(diff.max()), float(err.max()))


def make(seed, n, C, dtype, shift=0.3):
    g = torch.Generator().manual_seed(seed)
    x = (torch.randn(n, C, generator=g) * (torch.rand(n, 1, generator=g) * 2 + 0.5) + shift)
    return (x.to(dtype).to(DEV), (1 + 0.1 * torch.randn(C, generator=g)).to(DEV),
            (0.1 * torch.randn(C, generator=g)).to(DEV),
            torch.randn(n, C, generator=g).to(dtype).to(DEV))


def check(x, w, b, dy, what):
    print(what, tuple(x.shape), x.dtype, flush=True)
    want = reference(x, w, b, dy, 1e-5, x.dtype)
    y, mean, rstd = abi.ln_forward(x, w, b)
    within(y, want["y"], what)
    for name, g in zip(("gx", "gw", "gb"), abi.ln_backward(dy, x, mean, rstd, w)):
        within(g, want[name], f"{what} {name}")


# both sides of each variant's edge in chunks of 4 (fp32) and 8 (bf16) channels
WIDTHS = [1, 2, 7, 16, 31, 64, 65, 96, 128, 129, 250, 256, 257, 512, 513, 1000, 1024, 1025, 2048,
          2049, 4096, 4099, 8192, 8200, 9001]


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("C", WIDTHS)
def test_widths(dtype, C):
    for n in (1, 37):
        check(*make(C, n, C, dtype), f"C {C}")


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("n,C", [(2, 64), (1023, 40), (5000, 32), (3000, 255), (40001, 24)])
def test_rows(dtype, n, C):
    check(*make(n, n, C, dtype), f"n {n}")


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_rows_around_a_large_mean(dtype):
    check(*make(1, 50, 300, dtype, shift=100.0), "mean 100")


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("shift", [0, 1, 3])
def test_strides(dtype, shift):
    """Columns of a wider matrix from an unaligned start; an expanded gradient
    (row stride 0) and one with a strided last axis."""
    n, C = 120, 70
    g = torch.Generator().manual_seed(shift)
    wide = torch.randn(n * 101 + 8, generator=g).to(dtype).to(DEV)
    x = torch.as_strided(wide, (n, C), (101, 1), shift)
    w, b = torch.randn(C, generator=g).to(DEV), torch.randn(C, generator=g).to(DEV)
    dy = torch.randn(1, C, generator=g).to(dtype).to(DEV).expand(n, C)
    check(x, w, b, dy, f"stride +{shift}")
    check(x, w, b, torch.randn(C, n, generator=g).to(dtype).to(DEV).t(), "strided gradient")


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_autograd_and_streams(dtype):
    x, w, b, dy = make(2, 300, 96, dtype)
    y, mean, rstd = abi.ln_forward(x, w, b)
    refs = abi.ln_backward(dy, x, mean, rstd, w)
    leaves = [t.clone().requires_grad_() for t in (x, w, b)]
    torch.cuda.synchronize()
    stream = torch.cuda.Stream()
    with torch.cuda.stream(stream):
        out = rie.nn.layer_norm(leaves[0].view(3, 100, 96), leaves[1], leaves[2])
        out.backward(dy.view(3, 100, 96))
    stream.synchronize()
    assert out.shape == (3, 100, 96) and torch.equal(out.reshape(300, 96), y)
    for leaf, r in zip(leaves, refs):
        assert torch.equal(leaf.grad, r)
    with torch.no_grad():
        assert torch.equal(rie.nn.layer_norm(x, w, b), y)
    # without parameters, and some gradients only
    ones = torch.ones(96, device=DEV)
    assert torch.equal(rie.nn.layer_norm(x), rie.nn.layer_norm(x, ones, torch.zeros_like(ones)))
    wl = w.clone().requires_grad_()
    rie.nn.layer_norm(x, wl, b).backward(dy)
    assert torch.equal(wl.grad, refs[1])


def test_no_rows():
    x = torch.empty(0, 48, device=DEV, requires_grad=True)
    w, b = (torch.ones(48, device=DEV, requires_grad=True) for _ in range(2))
    y = rie.nn.layer_norm(x, w, b)
    assert y.shape == (0, 48)
    y.sum().backward()
    assert (w.grad == 0).all() and (b.grad == 0).all() and x.grad.shape == (0, 48)


def test_gradients_against_differences():
    """fp32, along a direction: a central difference with step 2^-6 is within
    1e-3 of the norms' product."""
    x, w, b, dy = make(3, 20, 130, F32)
    y, mean, rstd = abi.ln_forward(x, w, b)
    grads = abi.ln_backward(dy, x, mean, rstd, w)
    step = 2.0 ** -6
    for i in range(3):
        ten = [x, w, b]
        d = torch.randn(ten[i].shape, generator=torch.Generator().manual_seed(i)).to(DEV)
        vals = []
        for sign in (1, -1):
            moved = list(ten)
            moved[i] = ten[i] + sign * step * d
            vals.append((abi.ln_forward(*moved)[0].double() * dy.double()).sum().item())
        diff = (vals[0] - vals[1]) / (2 * step)
        got = (grads[i].double() * d.double()).sum().item()
        assert abs(diff - got) <= 1e-3 * (grads[i].double().norm() * d.double().norm()).item()


def test_values_that_are_not_finite_stay_in_their_row():
    x, w, b, _ = make(4, 40, 64, F32)
    ref = rie.nn.layer_norm(x, w, b)
    x[7, 3], x[20, 0] = float("nan"), float("inf")
    y = rie.nn.layer_norm(x, w, b)
    rows = torch.ones(40, dtype=torch.bool, device=DEV)
    rows[7] = rows[20] = False
    assert torch.equal(y[rows], ref[rows]) and not torch.isfinite(y[7]).any()


def test_refusals():
    x = torch.zeros(4, 8, device=DEV)
    for call, msg in [
        (lambda: rie.nn.layer_norm(x.cpu()), "device"),
        (lambda: rie.nn.layer_norm(x.half()), "fp32 or bf16"),
        (lambda: rie.nn.layer_norm(x, torch.ones(7, device=DEV)), "vectors of 8"),
        (lambda: rie.nn.layer_norm(x, torch.ones(8, device=DEV).bfloat16()), "fp32"),
        (lambda: rie.nn.layer_norm(x, eps=0.0), "eps"),
        (lambda: rie.nn.layer_norm(torch.zeros(4, 0, device=DEV)), "channel"),
        (lambda: rie.nn.RiemannLayerNorm(0), "feature"),
    ]:
        with pytest.raises(RuntimeError, match=msg):
            call()
