"""Rotation, gated feed-forward and attention inside a window where element
offsets pass 32 bits: rows at the end of buffers of more than 2^31 elements
give what the same rows give in small ones. And on a stream of the caller's,
behind work that is still under way there."""
import pytest
import torch

from feed_forward_reference import assert_close, reference
from helpers import DEV
from riemannengine_amd import abi

pytestmark = pytest.mark.gpu

BF16 = torch.bfloat16


def ints(values):
    return torch.tensor(values, dtype=torch.int32, device=DEV)


def test_rotation_of_many_rows():
    from riemannengine import nn
    n, heads, kv, dim, few = 420_000, 32, 8, 128, 40
    assert n * (heads + kv) * dim > 2 ** 31 and n * heads * dim < 2 ** 31
    g = torch.Generator(device=DEV).manual_seed(0)
    # one tensor of both, so the keys' rows have the long stride too
    rows = torch.zeros(n, heads + kv, dim, dtype=BF16, device=DEV)
    rows[-few:] = torch.randn(few, heads + kv, dim, generator=g, device=DEV).to(BF16)
    positions = torch.arange(n, device=DEV)[:, None]
    freq = nn.rotary_frequencies([dim // 2])
    w = torch.randn(dim, generator=g, device=DEV)
    print("far rows", flush=True)
    for first, last in ((0, heads + kv), (heads, heads + kv)):
        part = rows[:, first:last]
        far = abi.rotary_forward(part, None, positions, freq, [dim // 2], norm=True,
                                 weights=(w, None))[0]
        near = abi.rotary_forward(part[-few:], None, positions[-few:], freq, [dim // 2],
                                  norm=True, weights=(w, None))[0]
        assert torch.equal(far[-few:], near) and near.abs().max() > 0
        del far
        gx, _, gw, _ = abi.rotary_backward((part, None), part, None, positions, freq,
                                           [dim // 2], norm=True, weights=(w, None))
        rx, _, rw, _ = abi.rotary_backward((part[-few:], None), part[-few:], None,
                                           positions[-few:], freq, [dim // 2], norm=True,
                                           weights=(w, None))
        assert torch.equal(gx[-few:], rx) and (gx[:-few:1000] == 0).all()
        # the other rows add zeros to the weight's gradient, in another order
        size = (part[-few:].float() ** 2).sum((0, 1)).max() * 4
        assert (gw - rw).abs().max() <= 1e-5 * size
        del gx


# wide rows, and wide hidden ones beside what the backward keeps of them
@pytest.mark.parametrize("channels,hidden", [(8192, 24), (24, 8192)])
def test_feed_forward_of_many_rows(channels, hidden):
    n, few, outputs = 263_000, 200, 16
    assert n * max(channels, hidden) > 2 ** 31
    g = torch.Generator(device=DEV).manual_seed(1)

    def normal(*shape, scale=1.0):
        return (torch.randn(shape, generator=g, device=DEV) * scale).to(BF16)

    x = torch.zeros(n, channels, dtype=BF16, device=DEV)
    x[-few:] = normal(few, channels)
    gate, up = (normal(hidden, channels, scale=channels ** -0.5) for _ in range(2))
    down, gy = normal(outputs, hidden, scale=hidden ** -0.5), normal(n, outputs)
    print("far rows", flush=True)
    want = reference(x[-few:], gate, up, down, "silu", gy[-few:])
    y, saved = abi.gated_forward(x, gate, up, down, "silu", True)
    assert_close(y[-few:], want[0], "y")
    assert (y[:-few:1000] == 0).all()
    gx, *weights = abi.gated_backward(gy, x, gate, up, down, saved, "silu")
    assert_close(gx[-few:], want[1], "grad_x")
    # rows of zeros have h, dg x and du x of zero
    for got, ref, name in zip(weights, want[2:], ("grad_gate", "grad_up", "grad_down")):
        assert_close(got, ref, name)


def test_attention_in_a_window_of_a_long_cache():
    heads, dim, far, lk = 8, 128, 2_200_000, 900
    assert far * heads * dim > 2 ** 31
    g = torch.Generator().manual_seed(2)
    q = torch.randn(70, heads, dim, generator=g).to(BF16).to(DEV)
    go = torch.randn(70, heads, dim, generator=g).to(BF16).to(DEV)
    k = torch.zeros(far + lk, heads, dim, dtype=BF16, device=DEV)
    v = torch.zeros(far + lk, heads, dim, dtype=BF16, device=DEV)
    k[far:] = torch.randn(lk, heads, dim, generator=g).to(BF16).to(DEV)
    v[far:] = torch.randn(lk, heads, dim, generator=g).to(BF16).to(DEV)
    print("far keys", flush=True)
    near, nearv = torch.zeros_like(k), torch.zeros_like(v)
    near[:lk], nearv[:lk] = k[far:], v[far:]
    for rows in (1, 70):
        qo_far, ko_far = ints([0, 0, rows]), ints([0, far, far + lk])
        qo, ko = ints([0, rows, rows]), ints([0, lk, far + lk])
        kw = dict(causal=True, window=300, sinks=4)
        a = abi.attn_forward(q[:rows], k, v, qo_far, ko_far, **kw)
        b = abi.attn_forward(q[:rows], near, nearv, qo, ko, **kw)
        assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])
        assert torch.isfinite(a[0]).all() and a[0].abs().max() > 0
        ga = abi.attn_backward(go[:rows], q[:rows], k, v, *a, qo_far, ko_far, **kw)
        gb = abi.attn_backward(go[:rows], q[:rows], near, nearv, *b, qo, ko, **kw)
        assert torch.equal(ga[0], gb[0])
        for x, y in zip(ga[1:], gb[1:]):
            assert torch.equal(x[far:], y[:lk]) and y[:lk].abs().max() > 0
            assert (x[:far:1000] == 0).all() and (y[lk::1000] == 0).all()


def test_on_a_stream_behind_its_own_work():
    from riemannengine import nn
    g = torch.Generator(device=DEV).manual_seed(3)
    n, heads, dim = 3000, 8, 64
    base = torch.randn(n, heads, dim, generator=g, device=DEV)
    gate, up, down = (torch.randn(a, b, generator=g, device=DEV) * 0.05
                      for a, b in ((700, heads * dim), (700, heads * dim), (heads * dim, 700)))
    positions, freq = torch.arange(n, device=DEV)[:, None], nn.rotary_frequencies([dim // 2])
    offsets = ints([0, n // 2, n])

    def work(x):
        x = x.detach().requires_grad_()
        q, k = nn.norm_rotate_heads(x, x, positions, freq, [dim // 2])
        a = nn.packed_attention(q, k, x, offsets, window=200, sinks=3)
        y = nn.gated_feed_forward(a.reshape(n, -1), gate, up, down)
        return y.detach(), torch.autograd.grad(y, x, torch.ones_like(y))[0]

    want = work(base * 2)
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        wide = base.repeat(400, 1, 1)  # some time's work in front of the rows
        x = (wide * 2)[-n:].clone()
        got = work(x)
    torch.cuda.current_stream().wait_stream(stream)
    assert all(torch.equal(a, b) for a, b in zip(want, got))
