"""The transformer operators with more rows, sequences or table rows than the
workgroups of one launch take (HIP keeps the threads along a grid's axis below
2^32: 2^24 workgroups of 256)."""
import pytest
import torch

from riemannengine_amd import abi
from helpers import DEV

pytestmark = pytest.mark.gpu

BF16 = torch.bfloat16
MOST = 2 ** 24  # workgroups of 256 threads


def test_embedding_of_many_ids():
    """Rows of 33 chunks take a wave each, four to a workgroup."""
    n, C = 4 * MOST + 1001, 264
    print("many ids", flush=True)
    table = torch.randn(50, C, device=DEV).to(BF16)
    ids = torch.randint(-1, 50, (n,), device=DEV, dtype=torch.int32)
    y = abi.embed_forward(ids, table, 2.0)
    table = torch.cat([table, torch.zeros(1, C, dtype=BF16, device=DEV)]) * 2
    for at in range(0, n, MOST // 4):  # a slice of every part, and the ends
        rows = slice(at, min(at + 3000, n))
        assert torch.equal(y[rows], table[ids[rows].long()])
    assert torch.equal(y[-3000:], table[ids[-3000:].long()])


def test_embedding_gradient_of_a_large_table():
    """Four table rows to a wave, sixteen to a workgroup: the last table rows
    are in the second launch."""
    V, C, n = 16 * MOST + 4000, 4, 5000
    print("many table rows", flush=True)
    ids = torch.randint(0, 60, (n,), device=DEV) + (V - 60)
    ids[::2] -= V - 60
    dy = torch.randn(n, C, device=DEV).to(BF16)
    gw = abi.embed_backward(dy, ids, V, 1.5)
    small = torch.where(ids < 60, ids, ids - (V - 60) + 60)
    ref = abi.embed_backward(dy, small, 120, 1.5)
    assert torch.equal(gw[:60], ref[:60]) and torch.equal(gw[-60:], ref[60:])
    assert not gw[60:-60].any()


def test_layer_norm_of_many_narrow_rows():
    """Sixty-four rows of up to 16 chunks to a workgroup."""
    n, C = 64 * MOST + 777, 2
    print("many rows", flush=True)
    few = torch.randn(50000, C, device=DEV).to(BF16)
    x = torch.zeros(n, C, dtype=BF16, device=DEV)
    x[-50000:] = few
    x[64 * MOST - 100000:64 * MOST - 50000] = few
    w, b = torch.randn(C, device=DEV), torch.randn(C, device=DEV)
    y, mean, rstd = abi.ln_forward(x, w, b)
    want = abi.ln_forward(few, w, b)
    for got, ref in zip((y, mean, rstd), want):
        assert torch.equal(got[-50000:], ref)
        assert torch.equal(got[64 * MOST - 100000:64 * MOST - 50000], ref)
    assert torch.equal(y[0], b.to(BF16)) and torch.equal(y[n // 2], y[0])


@pytest.mark.parametrize("kv_heads", [8, 3])
def test_attention_of_many_short_sequences(kv_heads):
    """A tile for every sequence and key head. Each row sees one key: its
    result is that key's value, grad_v the row's grad_out, grad_q and grad_k
    nothing but the rounding of a difference of two equal sums."""
    heads, dim = kv_heads, 8
    n = MOST // kv_heads + 5000
    print("many sequences", n, kv_heads, flush=True)
    q, k, v, go = (torch.randn(n, heads, dim, device=DEV).to(BF16) for _ in range(4))
    o = torch.arange(n + 1, dtype=torch.int32, device=DEV)
    out, lse = abi.attn_forward(q, k, v, o, o, causal=True)
    assert torch.equal(out, v)
    scores = (q.float() * k.float()).sum(-1) * dim ** -0.5
    assert (lse.t() - scores).abs().max() <= 1e-5 * (1 + scores.abs().max())
    dq, dk, dv = abi.attn_backward(go, q, k, v, out, lse, o, o, causal=True)
    # its probability is 1 but for lse's and the score's rounding
    assert (dv.float() - go.float()).abs().max() <= 2.0 ** -8 * go.float().abs().max()
    size = (go.float().abs() * v.float().abs()).sum(-1).max() * k.float().abs().max()
    assert dq.float().abs().max() <= 2.0 ** -18 * size
    assert dk.float().abs().max() <= 2.0 ** -18 * size
