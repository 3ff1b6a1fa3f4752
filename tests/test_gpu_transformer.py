"""The transformer layers on sparse tensors (RiemannEmbedding,
RiemannLayerNorm, RiemannAttention, AttentionBlock) together: a stage from
voxel classes to logits against the same computed scene by scene in torch,
batches out of order, dtype casts, a few training steps that lower the loss."""
import pytest
import torch

import riemannengine as rie
from helpers import DEV

pytestmark = pytest.mark.gpu


def scene(n=150, batch=3, seed=0):
    """Coordinates with the batches mixed, and a class per voxel (some none)."""
    g = torch.Generator().manual_seed(seed)
    c = torch.stack([torch.randint(0, batch, (4 * n,), generator=g)]
                    + [torch.randint(0, 12, (4 * n,), generator=g) for _ in range(3)], 1)
    c = torch.unique(c, dim=0)
    c = c[torch.randperm(len(c), generator=g)][:n].int().to(DEV)
    ids = torch.randint(-1, 5, (n,), generator=g).to(DEV)
    return c, ids


def by_scene(block, x, coords, heads, kv_heads, causal):
    """AttentionBlock's formula with torch's own operations, scene by scene."""
    p = block.named_parameters()
    F = torch.nn.functional
    C = x.shape[1]
    d = C // heads
    out = torch.empty_like(x)
    for b in coords[:, 0].unique():
        rows = (coords[:, 0] == b).nonzero()[:, 0]
        h = x[rows]
        n = F.layer_norm(h, (C,), p["norm1.weight"], p["norm1.bias"])
        qkv = (F.linear(n, p["attention.projection.weight"], p["attention.projection.bias"])
               .view(len(rows), heads + 2 * kv_heads, d).transpose(0, 1))
        q, k, v = qkv.split([heads, kv_heads, kv_heads])
        k, v = (t.repeat_interleave(heads // kv_heads, 0) for t in (k, v))
        s = torch.matmul(q, k.transpose(1, 2).contiguous()) * d ** -0.5
        if causal:
            s = s.masked_fill(torch.ones(len(rows), len(rows), dtype=torch.bool,
                                         device=s.device).triu(1), -torch.inf)
        o = torch.matmul(s.softmax(-1), v.contiguous()).transpose(0, 1).reshape(len(rows), C)
        h = h + F.linear(o, p["attention.output.weight"], p["attention.output.bias"])
        n = F.layer_norm(h, (C,), p["norm2.weight"], p["norm2.bias"])
        h = h + F.linear(F.gelu(F.linear(n, p["up.weight"], p["up.bias"])), p["down.weight"],
                         p["down.bias"])
        out[rows] = h
    return out


@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize("heads,kv_heads", [(4, 0), (4, 2)])
def test_block_matches_scene_by_scene(causal, heads, kv_heads):
    """fp32: two sums of the same terms in other orders; 2e-5 of the largest
    value is 2^-24 times the ~300 roundings along one output's path."""
    torch.manual_seed(0)
    coords, ids = scene()
    emb = rie.nn.RiemannEmbedding(5, 64, scale=8.0)
    block = rie.nn.AttentionBlock(64, heads, kv_heads, causal=causal)
    emb.to(DEV), block.to(DEV)
    base = rie.SparseTensor(torch.zeros(len(ids), 1, device=DEV), coords)
    x = emb(ids, base)
    assert (x.F[ids < 0] == 0).all()
    # columns a norm cannot tell apart would leave an all-zero row at 0 / eps
    x = rie.SparseTensor(x.F + 0.01 * torch.randn(x.F.shape, device=DEV), x.coordinate_map_key,
                         x.coordinate_manager)
    y = block(x)
    want = by_scene(block, x.F, coords, heads, kv_heads or heads, causal)
    assert y.coordinate_map_key == x.coordinate_map_key
    assert (y.F - want).abs().max() <= 2e-5 * want.abs().max()
    seed = torch.randn(want.shape, device=DEV)
    params = list(block.parameters()) + [emb.weight]
    got = torch.autograd.grad(y.F, params, seed, retain_graph=True)  # x is shared
    ref = torch.autograd.grad(want, params, seed)
    for g, r in zip(got, ref):
        assert (g - r).abs().max() <= 1e-4 * r.abs().max()


def test_layer_norm_layer():
    coords, _ = scene()
    norm = rie.nn.RiemannLayerNorm(32)
    norm.to(DEV)
    norm.to(torch.bfloat16)  # parameters stay fp32
    assert all(p.dtype == torch.float32 for p in norm.parameters())
    x = rie.SparseTensor(torch.randn(len(coords), 32, device=DEV).bfloat16(), coords)
    y = norm(x)
    assert y.F.dtype == torch.bfloat16
    assert torch.equal(y.F, rie.nn.layer_norm(x.F, *norm.parameters()))
    with pytest.raises(RuntimeError, match="features"):
        rie.nn.RiemannLayerNorm(16)(x)
    assert not list(rie.nn.RiemannLayerNorm(16, affine=False).parameters())


def test_refusals():
    for call, msg in [(lambda: rie.nn.RiemannAttention(64, 5), "multiple"),
                      (lambda: rie.nn.RiemannAttention(64, 4, 3), "multiple"),
                      (lambda: rie.nn.AttentionBlock(64, 4, expansion=0), "expansion")]:
        with pytest.raises(RuntimeError, match=msg):
            call()


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_training_lowers_the_loss(dtype):
    """Classes of masked voxels from the others: twenty steps, as a program
    trains the stage."""
    torch.manual_seed(1)
    coords, ids = scene(n=400, batch=2, seed=1)
    ids = (coords[:, 1] // 3).long()  # a class that the position decides
    emb = rie.nn.RiemannEmbedding(5, 64, scale=8.0)
    block = rie.nn.AttentionBlock(64, 4, 2)
    norm = rie.nn.RiemannLayerNorm(64)
    head = torch.nn.Linear(64, 4).to(DEV)
    for m in (emb, block, norm):
        m.to(DEV)
    if dtype == torch.bfloat16:
        emb.to(dtype), block.to(dtype)
    where = torch.nn.Linear(3, 64).to(DEV)
    params = [*emb.parameters(), *block.parameters(), *norm.parameters(), *head.parameters(),
              *where.parameters()]
    optimizer = torch.optim.Adam(params, lr=2e-3)
    hidden = torch.rand(len(ids), device=DEV) < 0.3
    seen = torch.where(hidden, 4, ids)
    base = rie.SparseTensor(torch.zeros(len(ids), 1, device=DEV), coords)
    losses = []
    for _ in range(20):
        x = emb(seen, base)
        f = x.F + where(coords[:, 1:].float() / 12).to(x.F.dtype)
        x = rie.SparseTensor(f, x.coordinate_map_key, x.coordinate_manager)
        logits = head(norm(block(x)).F.float())
        loss = torch.nn.functional.cross_entropy(logits[hidden], ids[hidden])
        optimizer.zero_grad()
        loss.backward()
        optimizer.step()
        losses.append(loss.item())
    print(dtype, losses[0], losses[-1], flush=True)
    assert losses[-1] < 0.7 * losses[0]


def test_example_trains():
    """The example's training loop, a few steps in each type."""
    import importlib.util
    import os
    path = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "examples",
                        "voxel_transformer.py")
    spec = importlib.util.spec_from_file_location("voxel_transformer", path)
    example = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(example)
    for dtype in (torch.float32, torch.bfloat16):
        losses = example.train(steps=25, n_scenes=2, voxels=600, channels=64, blocks=1,
                               dtype=dtype, log=lambda text: print(text, flush=True))
        assert losses[-1] < 0.9 * losses[0]
