"""Attention over packed sequences: rhip_attn_forward / rhip_attn_backward and
riemannengine.nn.packed_attention against the definition in fp64, within the
bounds of attention_reference: lengths from zero to several tiles, tile edges,
rows that see nothing, grouped heads, head widths that fill no tile, strided
and unaligned inputs, caches with room, what lies in masked places,
refusals, other streams, and gradients against differences."""
import math

import numpy as np
import pytest
import torch

import riemannengine as rie
from riemannengine_amd import abi
from attention_reference import assert_within, attention
from helpers import DEV

pytestmark = pytest.mark.gpu

F32, BF16 = torch.float32, torch.bfloat16


def offsets(lens):
    return torch.tensor([0] + list(lens)).cumsum(0).int().to(DEV)


def inputs(seed, n_q, n_k, heads, kv_heads, dim, dtype):
    g = torch.Generator().manual_seed(seed)

    def make(*shape):
        return torch.randn(shape, generator=g).to(dtype).to(DEV)

    return (make(n_q, heads, dim), make(n_k, kv_heads, dim), make(n_k, kv_heads, dim),
            make(n_q, heads, dim))


def check(q, k, v, grad, q_off, k_off, k_len=None, causal=False, scale=None, what=""):
    print(what, tuple(q.shape), tuple(k.shape), q.dtype, "causal" if causal else "", flush=True)
    want = attention(q, k, v, q_off, k_off, k_len, causal, scale, grad)
    out, lse = abi.attn_forward(q, k, v, q_off, k_off, k_len, causal, scale)
    assert_within(out, want["out"], what + " out")
    d = q.shape[2]
    lse = lse.double().cpu().numpy()
    seen = np.isfinite(want["lse"])
    assert (np.isneginf(lse) == ~seen).all(), what + " lse of empty rows"
    assert np.allclose(lse[seen], want["lse"][seen], rtol=2.0 ** -20, atol=2.0 ** -16 * d)
    grads = abi.attn_backward(grad, q, k, v, out, torch.from_numpy(lse).float().to(DEV), q_off,
                              k_off, k_len, causal, scale)
    for name, g in zip(("dq", "dk", "dv"), grads):
        assert_within(g, want[name], f"{what} {name}")
    return out, grads


LENS = [[1], [0], [2, 0, 1], [31, 32, 33, 63, 64, 65], [127, 128, 129], [0, 300, 0, 7], [517]]


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("causal", [False, True])
def test_lengths(dtype, causal):
    for i, lens in enumerate(LENS):
        q, k, v, g = inputs(i, sum(lens), sum(lens), 4, 2, 32, dtype)
        o = offsets(lens)
        check(q, k, v, g, o, o, causal=causal, what=f"lens {lens}")


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("dim", [1, 5, 8, 16, 24, 32, 40, 64, 72, 96, 127, 128])
def test_head_widths(dtype, dim):
    lens = [70, 1, 150]
    q, k, v, g = inputs(dim, sum(lens), sum(lens), 3, 1, dim, dtype)
    o = offsets(lens)
    check(q, k, v, g, o, o, causal=True, what=f"dim {dim}")


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("heads,kv_heads", [(1, 1), (8, 8), (8, 1), (6, 2), (5, 5)])
def test_grouped_heads(dtype, heads, kv_heads):
    lens = [100, 33, 161]
    q, k, v, g = inputs(heads, sum(lens), sum(lens), heads, kv_heads, 64, dtype)
    o = offsets(lens)
    check(q, k, v, g, o, o, causal=True, what=f"heads {heads}/{kv_heads}")


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize("dim", [64, 128])
def test_other_key_lengths(dtype, causal, dim):
    """More keys than rows, fewer (causal: the first rows see nothing), none."""
    q_lens, k_lens = [5, 0, 200, 130, 1, 40, 1], [200, 3, 7, 0, 700, 41, 1]
    q, k, v, g = inputs(1, sum(q_lens), sum(k_lens), 4, 2, dim, dtype)
    out, _ = check(q, k, v, g, offsets(q_lens), offsets(k_lens), causal=causal, what="q != k")
    o = out[205:335]  # 130 rows without keys
    assert (o == 0).all()


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("heads,kv_heads,dim", [(8, 2, 128), (4, 4, 64), (32, 1, 32), (3, 1, 40)])
@pytest.mark.parametrize("rows", [1, 3])
def test_few_rows_over_a_cache(dtype, heads, kv_heads, dim, rows):
    """Single tokens (and three) against caches whose regions have room."""
    fills, room = [1, 700, 64, 0, 2049, 33, 5], 19
    q, k, v, g = inputs(2, rows * len(fills), sum(fills) + room * len(fills), heads, kv_heads,
                        dim, dtype)
    k_off = offsets([f + room for f in fills])
    k_len = torch.tensor(fills, dtype=torch.int32, device=DEV)
    for s, f in enumerate(fills):  # what the room holds reaches nothing
        k[int(k_off[s]) + f:int(k_off[s + 1])] = math.nan
        v[int(k_off[s]) + f:int(k_off[s + 1])] = math.inf
    out, (_, gk, gv) = check(q, k, v, g, offsets([rows] * len(fills)), k_off, k_len, causal=True,
                             what="cache")
    for s, f in enumerate(fills):
        assert (gk[int(k_off[s]) + f:int(k_off[s + 1])] == 0).all()
        assert (gv[int(k_off[s]) + f:int(k_off[s + 1])] == 0).all()


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_one_long_sequence_for_one_row(dtype):
    q, k, v, g = inputs(3, 1, 40001, 4, 1, 64, dtype)
    check(q, k, v, g, offsets([1]), offsets([40001]), causal=True, what="one row")


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("dim", [32, 40])
@pytest.mark.parametrize("shift", [0, 1, 4])
def test_strides(dtype, dim, shift):
    """Views of one projection [rows, (heads + 2 key heads) dim + 3], heads
    and rows strided, from an unaligned start; grad_out of one value."""
    lens, h, hk = [90, 41], 4, 2
    n, width = sum(lens), (h + 2 * hk) * dim
    g = torch.Generator().manual_seed(shift)
    flat = torch.randn(n * (width + 4) + 8, generator=g).to(dtype).to(DEV)
    rows = torch.as_strided(flat, (n, h + 2 * hk, dim), (width + 4, dim, 1), shift)
    q, k, v = rows[:, :h], rows[:, h:h + hk], rows[:, h + hk:]
    grad = torch.full((1, 1, 1), 0.5, dtype=dtype, device=DEV).expand(n, h, dim)
    o = offsets(lens)
    check(q, k, v, grad, o, o, causal=True, what=f"stride +{shift}")
    # heads before rows, keys shared by expansion
    qt = q.transpose(0, 1).contiguous().transpose(0, 1)
    ke = k[:, :1].expand(n, h, dim)
    check(qt, ke, v[:, :1].expand(n, h, dim), grad, o, o, what="heads first, expanded keys")


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_rows_outside_every_sequence(dtype):
    q, k, v, g = inputs(4, 300, 280, 2, 1, 64, dtype)
    q_off, k_off = offsets([50, 60]), offsets([45, 70])
    out, (gq, gk, gv) = check(q, k, v, g, q_off, k_off, what="unowned rows")
    assert (out[110:] == 0).all() and (gq[110:] == 0).all()
    assert (gk[115:] == 0).all() and (gv[115:] == 0).all()


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("bad", [math.nan, math.inf, -math.inf])
def test_masked_places_do_not_reach_a_row(dtype, bad):
    """Keys and values that are not finite reach the rows that see them and
    none else: not earlier rows of a causal sequence, not other sequences."""
    lens, at = [40, 170, 90], 40 + 77
    q, k, v, _ = inputs(5, sum(lens), sum(lens), 4, 2, 64, dtype)
    o = offsets(lens)
    clean, _ = abi.attn_forward(q, k, v, o, o, causal=True)
    for t in ("k", "v"):
        kk, vv = k.clone(), v.clone()
        (kk if t == "k" else vv)[at] = bad
        out, _ = abi.attn_forward(q, kk, vv, o, o, causal=True)
        want = attention(q, k, v, o, o, causal=True)["out"]
        rows = torch.ones(sum(lens), dtype=torch.bool)
        rows[at:40 + 170] = False  # rows that see it
        np_rows = rows.numpy()
        assert_within(out[rows.to(DEV)], (want[0][np_rows], want[1][np_rows]), f"{t} {bad}")
        if t == "v" or math.isnan(bad):
            assert not torch.isfinite(out[at:40 + 170]).any()
    # a first row that is not finite, and an empty row beside it
    q2, k2, v2, _ = inputs(6, 50, 20, 1, 1, 32, dtype)
    v2[0] = bad
    out, lse = abi.attn_forward(q2, k2, v2, offsets([50]), offsets([20]), causal=True)
    assert (out[:30] == 0).all() and torch.isneginf(lse[0, :30]).all()
    assert not torch.isfinite(out[30:]).any()


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("rows", [170, 9000])
def test_masked_places_do_not_reach_a_gradient(dtype, dim, rows):
    """Causal: a grad_out row that is not finite reaches the gradients of the
    keys it sees (and its own), keys and values that are not finite those of
    the rows that see them; the others keep their values. Both launch shapes
    (9000 rows on 4 heads fill the chip with whole tiles)."""
    lens = [40, rows, 90]
    n = sum(lens)
    q, k, v, g = inputs(11, n, n, 4, 4 if rows > 1000 else 2, dim, dtype)
    o = offsets(lens)
    at = 40 + 77
    print("masked gradients", dtype, dim, rows, flush=True)
    out, lse = abi.attn_forward(q, k, v, o, o, causal=True)
    clean = abi.attn_backward(g, q, k, v, out, lse, o, o, causal=True)
    tol = [16 * torch.finfo(dtype).eps * c.abs().max() for c in clean]
    g2 = g.clone()
    g2[at] = math.nan
    gq, gk, gv = abi.attn_backward(g2, q, k, v, out, lse, o, o, causal=True)
    others = torch.arange(n, device=DEV) != at
    assert (gq[others] - clean[0][others]).abs().max() <= tol[0]
    unseen = torch.ones(n, dtype=torch.bool, device=DEV)
    unseen[40:at + 1] = False
    assert (gk[unseen] - clean[1][unseen]).abs().max() <= tol[1]
    assert (gv[unseen] - clean[2][unseen]).abs().max() <= tol[2]
    assert not torch.isfinite(gv[40:at + 1]).any() and not torch.isfinite(gq[at]).any()
    k2, v2 = k.clone(), v.clone()
    k2[at], v2[at] = math.inf, math.nan
    out, lse = abi.attn_forward(q, k2, v2, o, o, causal=True)
    gq, gk, gv = abi.attn_backward(g, q, k2, v2, out, lse, o, o, causal=True)
    rows_ok = torch.ones(n, dtype=torch.bool, device=DEV)
    rows_ok[at:40 + rows] = False
    assert (gq[rows_ok] - clean[0][rows_ok]).abs().max() <= tol[0]
    assert (gk[:40] - clean[1][:40]).abs().max() <= tol[1]


def test_rounding_error_of_out():
    """bf16: out + rest is the fp32 result to about twice 8 bits, and with it
    rows that see one key have no query gradient but fp32 noise."""
    lens = [1, 60, 1, 2000]
    n = sum(lens)
    q, k, v, g = inputs(12, n, n, 8, 2, 64, BF16)
    o = offsets(lens)
    print("rest", flush=True)
    rest = torch.full_like(q, math.nan)
    out, lse = abi.attn_forward(q, k, v, o, o, causal=True, rest=rest)
    want = attention(q, k, v, o, o, causal=True)["out"]
    u = torch.finfo(BF16).eps / 2
    # P is rounded; the result is not: the bound's other half is u^2 |out|
    assert_within(out.double() + rest.double(), (want[0], want[1] / 2 + u * u * abs(want[0])),
                  "out + rest")
    gq, _, _ = abi.attn_backward(g, q, k, v, out, lse, o, o, causal=True, rest=rest)
    want = attention(q, k, v, o, o, None, True, None, g)["dq"]
    assert_within(gq, want, "dq")
    size = (g.double().abs() * v.double().abs().amax()).sum(-1).amax().item()
    first = gq[[0, 1, 61, 62]].double().abs().max().item()
    assert first <= 64 * 2.0 ** -24 * 8 * size, first


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("heads,kv_heads,dim", [(8, 8, 32), (4, 4, 64), (8, 4, 128), (9, 3, 40),
                                                (4, 2, 80), (8, 8, 96)])
@pytest.mark.parametrize("total", [12000, 24000, 40000])
def test_shared_tiles(dtype, heads, kv_heads, dim, total):
    """Enough rows for tiles of 32, 64 and 128 rows on every CU (both sides)."""
    lens = [total // kv_heads // 3 + 77, 1, 0, 130, total // 14]
    n = sum(lens)
    if heads == 9 and dtype == BF16:
        lens = [n, 0, 63]
        n = sum(lens)
    q, k, v, g = inputs(13, n, n, heads, kv_heads, dim, dtype)
    o = offsets(lens)
    print("shared tiles", n, heads, kv_heads, dim, dtype, flush=True)
    out, lse = abi.attn_forward(q, k, v, o, o, causal=True)
    grads = abi.attn_backward(g, q, k, v, out, lse, o, o, causal=True)
    for s in range(len(lens)):  # fp64 by the sequence, on the device
        sl = slice(int(o[s]), int(o[s + 1]))
        if lens[s] == 0:
            continue
        for h in range(0, heads, max(1, heads // 2)):
            b = h // (heads // kv_heads)
            Q, K, V, G = (t.double() for t in (q[sl, h], k[sl, b], v[sl, b], g[sl, h]))
            S = (Q @ K.t()) * dim ** -0.5
            S.masked_fill_(torch.ones_like(S, dtype=torch.bool).triu(1), -math.inf)
            P = S.softmax(-1)
            del S
            O = P @ V
            u = torch.finfo(BF16).eps / 2 if dtype == BF16 else 0.0
            e = 2.0 ** -24 * (dim + lens[s] + 16) * 8
            err = (out[sl, h].double() - O).abs() - 1.01 * (2 * u + e) * (P @ V.abs())
            assert err.max() <= 0, (s, h, "out")
            big = (G.abs() * O.abs()).sum(1, keepdim=True)
            dS = P * (G @ V.t() - (G * O).sum(1, keepdim=True))
            bound = u * (dS.abs() + P * big) + 3 * e * P * (G.abs() @ V.abs().t() + big)
            want = dim ** -0.5 * (dS @ K)
            err = ((grads[0][sl, h].double() - want).abs()
                   - 1.01 * (dim ** -0.5 * (bound @ K.abs()) + u * want.abs()))
            assert err.max() <= 0, (s, h, "dq")
    # the keys' gradients against the same in smaller pieces: each head of a
    # group by itself, added in fp64
    h0 = heads // kv_heads
    parts = []
    for h in range(h0):
        o1, l1 = abi.attn_forward(q[:, h:h + 1], k[:, :1], v[:, :1], o, o, causal=True)
        parts.append(abi.attn_backward(g[:, h:h + 1], q[:, h:h + 1], k[:, :1], v[:, :1], o1, l1,
                                       o, o, causal=True))
    for i, name in ((1, "dk"), (2, "dv")):
        want = sum(p[i][:, 0].double() for p in parts)
        # each side rounds its results and the operands of its sums
        tol = (h0 + 1) * 4 * torch.finfo(dtype).eps * want.abs().max()
        if dtype == F32:
            tol = 1e-4 * want.abs().max()
        assert (grads[i][:, 0].double() - want).abs().max() <= tol, name


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_large_scores(dtype):
    """Scores of a few thousand: the maximum is taken off before the exponential."""
    q, k, v, g = inputs(7, 200, 200, 2, 2, 64, F32)
    q, k, v, g = (t.to(dtype) for t in (q * 30, k * 30, v, g))
    o = offsets([200])
    print("large scores", dtype, flush=True)
    out, lse = abi.attn_forward(q, k, v, o, o, causal=True)
    want = attention(q, k, v, o, o, None, True, None, g)
    assert_within(out, want["out"], "large scores")
    assert torch.isfinite(lse).all()
    # the type's lowest value as a key: a score so low that its weight is 0
    k2 = k.clone()
    k2[5] = 0
    q2 = q.clone()
    q2[:, :, 0], k2[:, :, 0] = 1, 0
    k2[5, :, 0] = torch.finfo(dtype).min / 4
    out, _ = abi.attn_forward(q2, k2, v, o, o)
    keep = torch.arange(200, device=DEV) != 5
    ref, _ = abi.attn_forward(q2, k2[keep], v[keep], o, offsets([199]))
    tol = 2.0 ** -7 if dtype == BF16 else 1e-4
    assert (out - ref).abs().max() <= tol * v.abs().max()


@pytest.mark.parametrize("causal", [False, True])
def test_gradients_against_differences(causal):
    """fp32: the gradient along a direction against a central difference of
    <out, g>; step 2^-6, error below step^2 times the third derivative (of the
    order of the value here) plus 2^-23 value / step: 1e-3 of the norms."""
    lens = [45, 20]
    q, k, v, g = inputs(8, 65, 65, 4, 2, 40, F32)
    o = offsets(lens)
    out, lse = abi.attn_forward(q, k, v, o, o, causal=causal)
    grads = abi.attn_backward(g, q, k, v, out, lse, o, o, causal=causal)
    step = 2.0 ** -6
    for i, name in enumerate("qkv"):
        ten = [q, k, v]
        direction = torch.randn(ten[i].shape, generator=torch.Generator().manual_seed(i)).to(DEV)
        vals = []
        for sign in (1, -1):
            moved = list(ten)
            moved[i] = ten[i] + sign * step * direction
            y, _ = abi.attn_forward(*moved, o, o, causal=causal)
            vals.append((y.double() * g.double()).sum().item())
        diff = (vals[0] - vals[1]) / (2 * step)
        got = (grads[i].double() * direction.double()).sum().item()
        size = (grads[i].double().norm() * direction.double().norm()).item()
        assert abs(diff - got) <= 1e-3 * size, (name, diff, got)


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_autograd_and_streams(dtype):
    """nn.packed_attention: equal to the C ABI's results, gradients of shared
    keys summed by autograd, on another stream, twice the same bits."""
    lens, h, dim = [130, 5, 77], 4, 64
    n = sum(lens)
    q, k, v, g = inputs(9, n, n, h, 1, dim, dtype)
    o = offsets(lens)
    rest = torch.empty_like(q) if dtype == BF16 else None  # as the layer keeps it
    ref, lse = abi.attn_forward(q, k, v, o, o, causal=True, rest=rest)
    refs = abi.attn_backward(g, q, k, v, ref, lse, o, o, causal=True, rest=rest)
    leaves = [t.clone().requires_grad_() for t in (q, k, v)]
    torch.cuda.synchronize()
    stream = torch.cuda.Stream()
    with torch.cuda.stream(stream):
        out = rie.nn.packed_attention(*leaves, o.long(), causal=True)
        out.backward(g)
    stream.synchronize()
    assert torch.equal(out, ref)
    for leaf, r in zip(leaves, refs):
        assert torch.equal(leaf.grad, r)
    # only some gradients wanted
    kl = k.clone().requires_grad_()
    rie.nn.packed_attention(q, kl, v, o, causal=True).backward(g)
    assert torch.equal(kl.grad, refs[1])
    ql = q.clone().requires_grad_()
    rie.nn.packed_attention(ql, k, v, o, o, causal=True).backward(g)
    assert torch.equal(ql.grad, refs[0])
    # keys expanded over the heads: autograd sums them again
    ke = k.clone().requires_grad_()
    rie.nn.packed_attention(q, ke.expand(n, h, dim), v.expand(n, h, dim), o, causal=True,
                            scale=dim ** -0.5).backward(g)
    want = attention(q, k, v, o, o, None, True, None, g)["dk"]
    # h results are rounded to the type each, and their sum again
    u = torch.finfo(dtype).eps / 2
    assert_within(ke.grad, (want[0], 2 * want[1] + (h + 1) * 4 * u * np.abs(want[0]).max()),
                  "expanded keys")
    with torch.no_grad():
        assert torch.equal(rie.nn.packed_attention(*leaves, o, causal=True), ref)


def test_refusals():
    q, k, v, _ = inputs(10, 8, 8, 4, 2, 16, F32)
    o = offsets([8])
    nn = rie.nn
    for call, msg in [
        (lambda: nn.packed_attention(q.cpu(), k, v, o), "one device"),
        (lambda: nn.packed_attention(q, k[:, :, :8], v[:, :, :8], o), "width"),
        (lambda: nn.packed_attention(q, k, v[:4], o), "same shape"),
        (lambda: nn.packed_attention(q[:, :3], k, v, o), "multiple"),
        (lambda: nn.packed_attention(q, k.bfloat16(), v, o), "dtype"),
        (lambda: nn.packed_attention(q.half(), k.half(), v.half(), o), "fp32 or bf16"),
        (lambda: nn.packed_attention(q, k, v, o.float()), "int32 or int64"),
        (lambda: nn.packed_attention(q, k, v, o.cpu()), "device"),
        (lambda: nn.packed_attention(q, k, v, o, offsets([4, 4])), "offsets"),
        (lambda: nn.packed_attention(q, k[:4], v[:4], o), "same rows"),
        (lambda: nn.packed_attention(q, k, v, o, o, offsets([1, 2])), "lengths"),
        (lambda: nn.packed_attention(q, k, v, o, scale=0.0), "scale"),
        (lambda: nn.packed_attention(q, k, v, o, scale=math.inf), "scale"),
        (lambda: nn.packed_attention(*(torch.zeros(8, 2, 136, device=DEV),) * 3, o), "128"),
    ]:
        with pytest.raises(RuntimeError, match=msg):
            call()
    # nothing to do is no error
    e = torch.empty(0, 4, 16, device=DEV)
    assert nn.packed_attention(e, k[:0], v[:0], offsets([])).shape == (0, 4, 16)
    assert nn.packed_attention(e, k, v, offsets([0]), o).shape == (0, 4, 16)
