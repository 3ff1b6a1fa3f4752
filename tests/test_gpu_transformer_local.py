"""The operators of a local transformer stage together, as they are used: the
layers on sparse tensors against the same computed scene by scene in torch, with
gradients; a decoder that reads a prompt and then goes on token by token over its
cache against the whole sequence at once; and the example."""
import os
import sys

import pytest
import torch

import riemannengine as rie
from helpers import DEV

sys.path.insert(0, os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))),
                                "examples"))
pytestmark = pytest.mark.gpu
F = torch.nn.functional


def scene(n=150, batch=3, seed=0):
    """Coordinates with the batches mixed."""
    g = torch.Generator().manual_seed(seed)
    c = torch.stack([torch.randint(0, batch, (4 * n,), generator=g)]
                    + [torch.randint(0, 12, (4 * n,), generator=g) for _ in range(3)], 1)
    c = torch.unique(c, dim=0)
    return c[torch.randperm(len(c), generator=g)][:n].int().to(DEV)


def turned(x, coords, rotary):
    """x [n, heads, width] turned by coords [n, axes], pairs (p, pairs + p)."""
    freq = torch.cat([10000.0 ** (-torch.arange(s, dtype=torch.float64, device=DEV) / s)
                      for s in rotary])
    axis = torch.repeat_interleave(torch.arange(3, device=DEV), torch.tensor(rotary, device=DEV))
    angle = coords.double()[:, axis] * freq
    c, s = torch.cos(angle)[:, None].to(x.dtype), torch.sin(angle)[:, None].to(x.dtype)
    n = len(freq)
    a, b = x[..., :n], x[..., n:2 * n]
    return torch.cat([a * c - b * s, a * s + b * c, x[..., 2 * n:]], -1)


def by_scene(p, x, coords, heads, kv_heads, causal, window, sinks, rotary, head_norm, gated):
    """AttentionBlock's formula with torch's own operations, in x's type."""
    C = x.shape[1]
    d = C // heads
    parts, rows_of = [], []
    for b in coords[:, 0].unique():
        rows = (coords[:, 0] == b).nonzero()[:, 0]
        n = len(rows)
        h = x[rows]
        qkv = F.linear(F.layer_norm(h, (C,), p["norm1.weight"], p["norm1.bias"]),
                       p["attention.projection.weight"],
                       p["attention.projection.bias"]).view(n, heads + 2 * kv_heads, d)
        q, k, v = qkv.split([heads, kv_heads, kv_heads], 1)
        if head_norm:
            q, k = (t * (t.square().mean(-1, keepdim=True) + 1e-6).rsqrt()
                    * p[f"attention.{name}_norm.weight"] for t, name in ((q, "query"), (k, "key")))
        if rotary:
            q, k = (turned(t, coords[rows, 1:], rotary) for t in (q, k))
        k, v = (t.repeat_interleave(heads // kv_heads, 1).transpose(0, 1) for t in (k, v))
        s = q.transpose(0, 1) @ k.transpose(1, 2) * d ** -0.5
        i = torch.arange(n, device=DEV)
        away = i[:, None] - i[None, :]
        sees = torch.ones(n, n, dtype=torch.bool, device=DEV)
        if window is not None:
            sees = (away.abs() < window) | (i[None, :] < sinks)
        if causal:
            sees = sees & (away >= 0)
        s = s.masked_fill(~sees, -torch.inf)
        o = (s.softmax(-1) @ v).transpose(0, 1).reshape(n, C)
        h = h + F.linear(o, p["attention.output.weight"], p["attention.output.bias"])
        m = F.layer_norm(h, (C,), p["norm2.weight"], p["norm2.bias"])
        if gated:
            m = (F.silu(m @ p["feed_forward.gate"].t()) * (m @ p["feed_forward.up"].t())
                 ) @ p["feed_forward.down"].t()
        else:
            m = F.linear(F.gelu(F.linear(m, p["up.weight"], p["up.bias"])), p["down.weight"],
                         p["down.bias"])
        parts.append(h + m)
        rows_of.append(rows)
    back = torch.empty(len(x), dtype=torch.long, device=DEV)
    back[torch.cat(rows_of)] = torch.arange(len(x), device=DEV)
    return torch.cat(parts)[back]


OPTIONS = [dict(), dict(gated=True), dict(rotary=[4, 2, 1]), dict(rotary=[3, 3, 2], head_norm=True),
           dict(window=9, sinks=2), dict(window=20, rotary=[0, 4, 4], gated=True),
           dict(window=7, sinks=3, rotary=[3, 3, 2], head_norm=True, gated=True)]


@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize("options", OPTIONS, ids=lambda o: "-".join(o) or "plain")
def test_block_matches_scene_by_scene(options, causal):
    """fp32 against fp64, outputs and every gradient. An element's path crosses
    about a thousand fp32 roundings (norms over 64, heads of 16 over 50 keys, 256
    hidden, and in the gradients 150 rows): 2^10 half steps of 2^-24 of the largest
    value is 6.1e-5."""
    torch.manual_seed(0)
    coords = scene()
    block = rie.nn.AttentionBlock(64, 4, 2, 4, causal, **options)
    block.to(DEV)
    params = block.named_parameters()
    with torch.no_grad():
        for p in params.values():
            p.add_(torch.randn_like(p) * 0.05)
    x = torch.randn(150, 64, device=DEV, requires_grad=True)
    out = block(rie.SparseTensor(x, coords)).F
    go = torch.randn_like(out)
    leaves = [x, *params.values()]
    grads = torch.autograd.grad(out, leaves, go)
    wide = [t.detach().double().requires_grad_() for t in leaves]
    want = by_scene(dict(zip(params, wide[1:])), wide[0], coords, 4, 2, causal,
                    options.get("window"), options.get("sinks", 0), options.get("rotary"),
                    options.get("head_norm", False), options.get("gated", False))
    for got, ref, name in zip([out, *grads], [want, *torch.autograd.grad(want, wide, go.double())],
                              ["out", "x", *params]):
        assert got.shape == ref.shape
        assert (got.double() - ref).abs().max() <= 6.1e-5 * ref.abs().max(), name


def test_norm_weights_stay_fp32():
    block = rie.nn.AttentionBlock(64, 4, rotary=[3, 3, 2], head_norm=True, gated=True)
    block.to(DEV)
    block.to(torch.bfloat16)
    types = {n: p.dtype for n, p in block.named_parameters().items()}
    assert {n for n, t in types.items() if t == torch.float32} == {
        "norm1.weight", "norm1.bias", "norm2.weight", "norm2.bias",
        "attention.query_norm.weight", "attention.key_norm.weight"}
    x = torch.randn(150, 64, device=DEV, dtype=torch.bfloat16, requires_grad=True)
    out = block(rie.SparseTensor(x, scene())).F
    assert out.dtype == torch.bfloat16
    grads = torch.autograd.grad(out.float().sum(), [x, *block.named_parameters().values()])
    assert all(g.isfinite().all() for g in grads)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_tokens_over_a_cache_match_the_whole_sequence(dtype):
    """Prompts of three sequences, then five tokens each, in caches with room: the
    tokens' rows equal those of one pass over everything, but for sums in another
    order (fp32: 2^9 half steps of the largest value; bf16: four roundings a row
    passes, of 2^-8 each, twice)."""
    nn = rie.nn
    g = torch.Generator(device=DEV).manual_seed(0)
    C, heads, kv, d, window, sinks = 128, 8, 2, 16, 12, 3
    lens, new, room = [30, 1, 17], 5, 64
    freq = nn.rotary_frequencies([8])

    def normal(*shape, scale=1.0):
        return (torch.randn(*shape, generator=g, device=DEV) * scale).to(dtype)

    wqkv, wo = normal((heads + 2 * kv) * d, C, scale=C ** -0.5), normal(C, C, scale=C ** -0.5)
    gate, up = normal(300, C, scale=C ** -0.5), normal(300, C, scale=C ** -0.5)
    down = normal(C, 300, scale=300 ** -0.5)
    wq, wk = (torch.rand(d, generator=g, device=DEV) + 0.5 for _ in range(2))
    norm = torch.rand(C, generator=g, device=DEV) + 0.5
    rows = [normal(n + new, C) for n in lens]

    def offsets(v):
        return torch.tensor([0, *v]).cumsum(0).int().to(DEV)

    def heads_of(x, places):
        qkv = F.linear(nn.layer_norm(x, norm), wqkv).view(len(x), heads + 2 * kv, d)
        q, k = nn.norm_rotate_heads(qkv[:, :heads], qkv[:, heads:heads + kv], places, freq, [8],
                                    wq, wk)
        return q, k, qkv[:, heads + kv:]

    def rest(x, mixed):
        x = x + F.linear(mixed.reshape(len(x), C), wo)
        return x + nn.gated_feed_forward(nn.layer_norm(x, norm), gate, up, down)

    with torch.no_grad():
        x = torch.cat(rows)
        o = offsets([n + new for n in lens])
        q, k, v = heads_of(x, torch.cat([torch.arange(n + new, device=DEV) for n in lens]))
        whole = rest(x, nn.packed_attention(q, k, v, o, causal=True, window=window, sinks=sinks))

        cache_k = torch.full((3 * room, kv, d), float("nan"), device=DEV, dtype=dtype)
        cache_v = cache_k.clone()
        regions = offsets([room] * 3)
        x = torch.cat([r[:n] for r, n in zip(rows, lens)])
        q, k, v = heads_of(x, torch.cat([torch.arange(n, device=DEV) for n in lens]))
        at = torch.cat([torch.arange(n, device=DEV) + i * room for i, n in enumerate(lens)])
        cache_k[at], cache_v[at] = k, v
        fill = torch.tensor(lens, dtype=torch.int32, device=DEV)
        prompts = rest(x, nn.packed_attention(q, cache_k, cache_v, offsets(lens), regions, fill,
                                              True, window=window, sinks=sinks))
        got = [[p] for p in prompts.split(lens)]
        for t in range(new):
            x = torch.stack([r[n + t] for r, n in zip(rows, lens)])
            q, k, v = heads_of(x, fill.long())
            at = fill.long() + torch.arange(3, device=DEV) * room
            cache_k[at], cache_v[at] = k, v
            fill += 1
            y = rest(x, nn.packed_attention(q, cache_k, cache_v, offsets([1] * 3), regions, fill,
                                            True, window=window, sinks=sinks))
            for i in range(3):
                got[i].append(y[i:i + 1])
    got = torch.cat([torch.cat(r) for r in got])
    limit = 2.0 ** -15 if dtype == torch.float32 else 2.0 ** -5
    assert got.isfinite().all()
    assert (got.double() - whole.double()).abs().max() <= limit * whole.double().abs().max()


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_example_runs(dtype):
    import voxel_transformer
    losses = voxel_transformer.train(steps=3, n_scenes=2, voxels=300, dtype=dtype, local=True,
                                     log=lambda *_: None)
    assert len(losses) == 3 and all(l == l and abs(l) != float("inf") for l in losses)


def test_refusals():
    nn = rie.nn
    for kw, match in [(dict(window=0), "window"), (dict(sinks=2), "window"),
                      (dict(rotary=[20, 20, 20]), "pairs"), (dict(rotary=[3, -1, 2]), "pairs"),
                      (dict(head_norm=True), "rotary")]:
        with pytest.raises(RuntimeError, match=match):
            nn.RiemannAttention(64, 4, **kw)
    with pytest.raises(RuntimeError, match="silu"):
        nn.RiemannGatedFeedForward(64, 100, "relu")
    block = nn.RiemannAttention(64, 4, rotary=[4, 4])
    block.to(DEV)
    with pytest.raises(RuntimeError, match="axes"):
        block(rie.SparseTensor(torch.randn(150, 64, device=DEV), scene()))
    layer = nn.RiemannGatedFeedForward(64, 100)
    layer.to(DEV)
    with pytest.raises(RuntimeError, match="features"):
        layer(rie.SparseTensor(torch.randn(150, 32, device=DEV), scene()))
    x = torch.randn(150, 64, device=DEV)
    assert torch.equal(layer(rie.SparseTensor(x, scene())).F,
                       nn.gated_feed_forward(x, layer.gate, layer.up, layer.down))
    assert torch.equal(layer(x), nn.gated_feed_forward(x, layer.gate, layer.up, layer.down))
