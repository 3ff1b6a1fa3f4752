"""The transformer operators where element offsets pass 32 bits: rows at the
end of buffers of more than 2^31 elements give what the same rows give at the
start of small ones, bit for bit (the same kernels on the same values). And
all three in a captured graph, replayed on changing inputs."""
import pytest
import torch

import riemannengine as rie
from riemannengine_amd import abi
from helpers import DEV

pytestmark = pytest.mark.gpu

BF16 = torch.bfloat16


def ints(values):
    return torch.tensor(values, dtype=torch.int32, device=DEV)


def test_attention_over_a_long_cache():
    """2.2 million cached rows of 8 x 128: the second sequence starts past
    2^31 elements."""
    heads, hk, dim, far, lk = 8, 8, 128, 2_200_000, 300
    assert far * hk * dim > 2 ** 31
    g = torch.Generator().manual_seed(0)
    q = torch.randn(70, heads, dim, generator=g).to(BF16).to(DEV)
    go = torch.randn(70, heads, dim, generator=g).to(BF16).to(DEV)
    k = torch.zeros(far + lk, hk, dim, dtype=BF16, device=DEV)
    v = torch.zeros(far + lk, hk, dim, dtype=BF16, device=DEV)
    k[far:] = torch.randn(lk, hk, dim, generator=g).to(BF16).to(DEV)
    v[far:] = torch.randn(lk, hk, dim, generator=g).to(BF16).to(DEV)
    print("far keys", flush=True)
    # as many sequences and keys on both sides, so the same launch shapes
    near = torch.cat([k[far:], torch.zeros_like(k[:far])])
    nearv = torch.cat([v[far:], torch.zeros_like(v[:far])])
    for rows in (1, 70):
        qo_far, ko_far = ints([0, 0, rows]), ints([0, far, far + lk])
        qo, ko = ints([0, rows, rows]), ints([0, lk, far + lk])
        a = abi.attn_forward(q[:rows], k, v, qo_far, ko_far, causal=True)
        b = abi.attn_forward(q[:rows], near, nearv, qo, ko, causal=True)
        assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])
        assert torch.isfinite(a[0]).all() and a[0].abs().max() > 0
        ga = abi.attn_backward(go[:rows], q[:rows], k, v, *a, qo_far, ko_far, causal=True)
        gb = abi.attn_backward(go[:rows], q[:rows], near, nearv, *b, qo, ko, causal=True)
        assert torch.equal(ga[0], gb[0])
        for x, y in zip(ga[1:], gb[1:]):
            assert torch.equal(x[far:], y[:lk]) and y[:lk].abs().max() > 0
            assert (x[:far:1000] == 0).all() and (y[lk::1000] == 0).all()


def test_layer_norm_of_many_wide_rows():
    n, C = 300_000, 8192
    assert n * C > 2 ** 31
    g = torch.Generator().manual_seed(1)
    few = torch.randn(40, C, generator=g).to(BF16).to(DEV)
    w, b = torch.randn(C, generator=g).to(DEV), torch.randn(C, generator=g).to(DEV)
    x = torch.zeros(n, C, dtype=BF16, device=DEV)
    x[-40:] = few
    print("far rows", flush=True)
    y, mean, rstd = abi.ln_forward(x, w, b)
    ref, rm, rr = abi.ln_forward(few, w, b)
    assert torch.equal(y[-40:], ref)
    gx, gw, gb = abi.ln_backward(x, x, mean, rstd, w)
    rx, _, rb = abi.ln_backward(few, few, rm, rr, w)
    assert torch.equal(gx[-40:], rx)
    # the other rows add zeros to the bias gradient, in another order
    assert (gb - rb).abs().max() <= 1e-5 * few.float().abs().sum(0).max()


def test_embedding_of_a_large_table():
    V, C = 530_000, 4096
    assert V * C > 2 ** 31
    g = torch.Generator().manual_seed(2)
    table = torch.zeros(V, C, dtype=BF16, device=DEV)
    table[-50:] = torch.randn(50, C, generator=g).to(BF16).to(DEV)
    small = table[-50:].clone()
    ids = torch.randint(0, 50, (3000,), generator=g).to(DEV)
    dy = torch.randn(3000, C, generator=g).to(BF16).to(DEV)
    print("far table rows", flush=True)
    assert torch.equal(abi.embed_forward(ids + V - 50, table, 2.0),
                       abi.embed_forward(ids, small, 2.0))
    gw = abi.embed_backward(dy, ids + V - 50, V, 2.0)
    assert torch.equal(gw[-50:], abi.embed_backward(dy, ids, 50, 2.0))
    assert (gw[:-50:999] == 0).all()


def test_in_a_graph():
    """Embedding, norm and attention, forward and backward, captured once and
    replayed on new ids and gradients between other work."""
    V, C, heads, n = 37, 64, 4, 333
    torch.manual_seed(3)
    table = torch.randn(V, C, device=DEV, dtype=BF16)
    w, b = torch.rand(C, device=DEV) + 0.5, torch.randn(C, device=DEV)
    offs = ints([0, 100, 100, 333])
    ids = torch.zeros(n, dtype=torch.int64, device=DEV)
    go = torch.zeros(n, heads, C // heads, device=DEV, dtype=BF16)

    def step():
        x = abi.embed_forward(ids, table, 1.5)
        y, mean, rstd = abi.ln_forward(x, w, b)
        q = y.view(n, heads, C // heads)
        out, lse = abi.attn_forward(q, q, q, offs, offs, causal=True)
        gq, gk, gv = abi.attn_backward(go, q, q, q, out, lse, offs, offs, causal=True)
        gx, gw, gb = abi.ln_backward((gq + gk + gv).view(n, C), x, mean, rstd, w)
        return out, gw, gb, abi.embed_backward(gx, ids, V, 1.5)

    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        for _ in range(2):
            step()
    torch.cuda.current_stream().wait_stream(stream)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        outs = step()
    for i in range(4):
        g = torch.Generator().manual_seed(i)
        ids.copy_(torch.randint(-1, V, (n,), generator=g))
        go.copy_(torch.randn(go.shape, generator=g))
        print("replay", i, flush=True)
        graph.replay()
        got = [o.clone() for o in outs]
        want = step()
        torch.cuda.synchronize()
        for x, y in zip(got, want):
            assert torch.equal(x, y)
