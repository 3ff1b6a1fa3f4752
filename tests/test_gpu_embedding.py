"""rhip_embed_forward / rhip_embed_backward and riemannengine.nn.embedding
against the definition: tables from one row to many, ids used never, once and
thousands of times (runs of the 64-position segments and their edges), ids
outside the table, odd widths, strides, int32 and int64 ids, refusals.

The forward is one fp32 product rounded once: exact in fp64 and rounded, the
same bits. The gradient of a row with m positions may be off by 2^-24 (m + 2)
times the sum of |dy|, and by the type's unit roundoff."""
import numpy as np
import pytest
import torch

import riemannengine as rie
from riemannengine_amd import abi
from helpers import DEV

pytestmark = pytest.mark.gpu

F32, BF16 = torch.float32, torch.bfloat16
U = {dt: torch.finfo(dt).eps / 2 for dt in (F32, BF16)}


def check(ids, weight, dy, scale, what):
    print(what, len(ids), tuple(weight.shape), weight.dtype, ids.dtype, flush=True)
    V, C = weight.shape
    known = ((ids >= 0) & (ids < V)).cpu()
    host = ids.cpu().long()
    y = abi.embed_forward(ids, weight, scale)
    want = torch.zeros(len(ids), C)
    want[known] = weight.float().cpu()[host[known]] * torch.tensor(scale, dtype=F32)
    assert torch.equal(y.cpu(), want.to(weight.dtype)), what
    gw = abi.embed_backward(dy, ids, V, scale)
    d = dy.double().cpu()[known]
    ref = torch.zeros(V, C, dtype=torch.float64).index_add_(0, host[known], d) * scale
    size = torch.zeros(V, C, dtype=torch.float64).index_add_(0, host[known], d.abs()) * abs(scale)
    count = torch.bincount(host[known], minlength=V)[:, None]
    err = (gw.double().cpu() - ref).abs()
    bound = 2.0 ** -24 * (count + 2) * size + U[weight.dtype] * ref.abs()
    assert bool((err <= 1.01 * bound).all()), (what, float((err - bound).max()))
    assert bool((gw.cpu()[count[:, 0] == 0] == 0).all())
    assert torch.equal(gw, abi.embed_backward(dy, ids, V, scale))  # the same bits again


def make(seed, n, V, C, dtype, ids=None, is32=False):
    g = torch.Generator().manual_seed(seed)
    if ids is None:
        ids = torch.randint(-1, V + 1, (n,), generator=g)  # -1 and V: outside
    ids = ids.int() if is32 else ids.long()
    return (ids.to(DEV), torch.randn(V, C, generator=g).to(dtype).to(DEV),
            torch.randn(n, C, generator=g).to(dtype).to(DEV))


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("n,V,C", [(1, 1, 1), (1, 5000, 64), (5, 3, 7), (64, 1, 32), (65, 1, 33),
                                   (1000, 20, 64), (20000, 7, 129), (3000, 2000, 255),
                                   (4097, 511, 512), (500, 70000, 40), (300, 100, 1100),
                                   (2048, 65536, 16), (40, 10, 4099), (2, 9, 8),
                                   (2047, 300, 24), (2049, 300, 24), (9000, 300000, 8)])
def test_sizes(dtype, n, V, C):
    check(*make(n, n, V, C, dtype, is32=n % 2 == 0), 3.5, f"n {n} V {V} C {C}")


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("runs", [[63, 64, 65], [64, 64, 64], [1, 128, 1, 127, 129], [200, 0, 3, 64],
                                  [0, 0, 1000], [32, 96, 640, 65]])
def test_runs_around_the_segments(dtype, runs):
    """Given numbers of uses per row, in a shuffled order."""
    ids = torch.repeat_interleave(torch.arange(len(runs)), torch.tensor(runs))
    ids = ids[torch.randperm(len(ids), generator=torch.Generator().manual_seed(0))]
    check(*make(1, len(ids), len(runs), 48, dtype, ids), 1.0, f"runs {runs}")


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("C", [4, 13, 32, 64, 100, 256, 520])
def test_every_count(dtype, C):
    """Rows used 0 to 66 times, and 67 to 200: every number of positions a
    wave or a chunk's part can hold, for every number of lanes per row."""
    for lo, hi in ((0, 67), (67, 201)):
        runs = torch.arange(lo, hi)
        ids = torch.repeat_interleave(torch.arange(len(runs)), runs)
        ids = ids[torch.randperm(len(ids), generator=torch.Generator().manual_seed(C))]
        check(*make(C, len(ids), len(runs), C, dtype, ids), 1.5, f"counts {lo}..{hi - 1} C {C}")


@pytest.mark.parametrize("shift", [0, 1])
@pytest.mark.parametrize("dtype", [F32, BF16])
def test_strides(dtype, shift):
    n, V, C = 200, 30, 50
    g = torch.Generator().manual_seed(shift)
    table = torch.randn(V * 61 + 8, generator=g).to(dtype).to(DEV)
    weight = torch.as_strided(table, (V, C), (61, 1), shift)
    ids = torch.randint(0, V, (n,), generator=g).to(DEV)
    dy = torch.randn(1, C, generator=g).to(dtype).to(DEV).expand(n, C)
    check(ids, weight, dy, 1.0, f"stride +{shift}")


def test_extreme_ids():
    big = torch.tensor([0, 2 ** 31, -2 ** 31, 2 ** 32, 2 ** 62, -2 ** 63, 4, 5])
    check(*make(2, 8, 5, 24, F32, big), 2.0, "extreme ids")


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_autograd_and_streams(dtype):
    ids, weight, dy = make(3, 600, 50, 96, dtype)
    y = abi.embed_forward(ids, weight, 2.0)
    gw = abi.embed_backward(dy, ids, 50, 2.0)
    leaf = weight.clone().requires_grad_()
    torch.cuda.synchronize()
    stream = torch.cuda.Stream()
    with torch.cuda.stream(stream):
        out = rie.nn.embedding(ids.view(20, 30), leaf, 2.0)
        out.backward(dy.view(20, 30, 96))
    stream.synchronize()
    assert out.shape == (20, 30, 96) and torch.equal(out.reshape(600, 96), y)
    assert torch.equal(leaf.grad, gw)
    emb = rie.nn.RiemannEmbedding(50, 96, scale=2.0)
    emb.to(torch.device(DEV))
    assert torch.equal(emb(ids.int()), abi.embed_forward(ids, emb.weight, 2.0))


def test_nothing_to_look_up():
    w = torch.ones(6, 8, device=DEV, requires_grad=True)
    y = rie.nn.embedding(torch.empty(0, dtype=torch.int64, device=DEV), w)
    assert y.shape == (0, 8)
    y.sum().backward()
    assert (w.grad == 0).all()


def test_refusals():
    ids, w = torch.zeros(4, dtype=torch.int64, device=DEV), torch.zeros(3, 8, device=DEV)
    for call, msg in [
        (lambda: rie.nn.embedding(ids.cpu(), w), "device"),
        (lambda: rie.nn.embedding(ids.float(), w), "int32 or int64"),
        (lambda: rie.nn.embedding(ids, w.half()), "fp32 or bf16"),
        (lambda: rie.nn.embedding(ids, w[0]), "rows, channels"),
        (lambda: rie.nn.embedding(ids, w, float("inf")), "finite"),
        (lambda: rie.nn.RiemannEmbedding(0, 8), "rows"),
    ]:
        with pytest.raises(RuntimeError, match=msg):
            call()
