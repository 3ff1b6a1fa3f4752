"""riemannengine.nn.rotate_heads and norm_rotate_heads against their definition
in fp64: widths that fill 16-byte chunks and that do not, several axes, parts
that stay, far positions, views.

Tolerances: a result's rounding is half a step of its type; in front of it
stand fp32 sums and products of a pair (of a head, with the norm), counted as
some steps of 2^-24 of the pair's (the head's) magnitude, and the angle's
cosine and sine, each off by at most 2^-22."""
import pytest
import torch

pytestmark = pytest.mark.gpu
DTYPES = [torch.float32, torch.bfloat16]
STEP = 2.0 ** -24
ANGLE = 2.0 ** -22


def frequencies(sections):
    from riemannengine import nn
    return nn.rotary_frequencies(sections)


def turned(x, positions, freq, sections, interleaved, back=False):
    axis = torch.repeat_interleave(torch.arange(len(sections)), torch.tensor(sections)).to(x.device)
    angle = positions.double()[:, axis] * freq * (-1 if back else 1)
    c, s = torch.cos(angle)[:, None], torch.sin(angle)[:, None]
    pairs = sum(sections)
    y = x.clone()
    first, second = ((slice(0, 2 * pairs, 2), slice(1, 2 * pairs, 2)) if interleaved
                     else (slice(0, pairs), slice(pairs, 2 * pairs)))
    a, b = x[..., first], x[..., second]
    y[..., first], y[..., second] = a * c - b * s, a * s + b * c
    return y


def reach(x, sections, interleaved):
    """The magnitude that a turned element's errors scale with."""
    pairs = sum(sections)
    m = x.abs().clone()
    first, second = ((slice(0, 2 * pairs, 2), slice(1, 2 * pairs, 2)) if interleaved
                     else (slice(0, pairs), slice(pairs, 2 * pairs)))
    m[..., first] = m[..., second] = x.abs()[..., first] + x.abs()[..., second]
    return m


def close(got, value, off, name):
    half = torch.finfo(got.dtype).eps / 2
    assert got.shape == value.shape and torch.isfinite(got).all(), name
    over = (got.double() - value).abs() - half * value.abs() - off - 1e-37
    assert over.numel() == 0 or over.max() <= 0, (name, float(over.max()), int(over.argmax()))


def place(n, sections, kind, generator):
    axes = len(sections)
    if kind == "int32":  # a sparse tensor's coordinates, the batch in front
        return torch.randint(-300, 300, (n, axes + 1), generator=generator, device="cuda",
                             dtype=torch.int32)[:, 1:]
    if kind == "int64":
        return torch.randint(0, 1000000, (n, axes), generator=generator, device="cuda")
    return torch.rand((n, axes), generator=generator, device="cuda") * 200 - 100


def case(n, heads, kv_heads, dim, dtype, sections, kind, seed=0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    rows = torch.randn((n, heads + 2 * kv_heads, dim), generator=g, device="cuda").to(dtype)
    q, k = rows[:, :heads], rows[:, heads:heads + kv_heads]
    grads = [torch.randn(t.shape, generator=g, device="cuda").to(dtype) for t in (q, k)]
    weights = [torch.randn(dim, generator=g, device="cuda") * 0.2 + 1 for _ in range(2)]
    return q, k, place(n, sections, kind, g), grads, weights


def check_alone(x, positions, sections, interleaved, grad):
    from riemannengine import nn
    freq = frequencies(sections)
    leaf = x.detach().requires_grad_()
    y = nn.rotate_heads(leaf, positions, freq, sections, interleaved)
    gx, = torch.autograd.grad(y, leaf, grad)
    for got, v, back in ((y.detach(), x, False), (gx, grad, True)):
        v = v.double()
        close(got, turned(v, positions, freq, sections, interleaved, back),
              (ANGLE + 3 * STEP) * reach(v, sections, interleaved), "turned back" if back else "y")
    with torch.no_grad():
        assert torch.equal(nn.rotate_heads(x, positions, freq, sections, interleaved), y)


def check_normed(q, k, positions, sections, interleaved, grads, weights, eps=1e-6):
    from riemannengine import nn
    freq = frequencies(sections)
    leaves = [t.detach().requires_grad_() for t in (q, k, *weights)]
    ys = nn.norm_rotate_heads(*leaves[:2], positions, freq, sections, *leaves[2:], eps,
                              interleaved)
    got = [t.detach() for t in ys] + list(torch.autograd.grad(ys, leaves, grads))
    dim = q.shape[2]
    # mean of squares, root, reciprocal and the products with it and the weight
    norm = (dim / 2 + 8) * STEP
    for i, (x, w, gy) in enumerate(zip((q, k), weights, grads)):
        x, w, gy = x.double(), w.double(), gy.double()
        r = ((x ** 2).mean(-1, keepdim=True) + eps) ** -0.5
        z = x * r * w
        close(got[i], turned(z, positions, freq, sections, interleaved),
              (ANGLE + 3 * STEP + norm) * reach(z, sections, interleaved), "y")
        d = turned(gy, positions, freq, sections, interleaved, True)
        ed = (ANGLE + 3 * STEP) * reach(gy, sections, interleaved)
        t = d * w * x * r  # the mean's terms
        gx = r * (d * w - x * r * t.mean(-1, keepdim=True))
        et = ((ed * (w * x).abs() * r).mean(-1, keepdim=True)
              + 2 * norm * t.abs().mean(-1, keepdim=True))
        off = r * (ed * w.abs() + (norm + 4 * STEP) * (d * w).abs() + (x * r).abs()
                   * (et + (2 * norm + 4 * STEP) * t.abs().mean(-1, keepdim=True)))
        close(got[2 + i], gx, off, "grad_x")
        rows = (d * x * r).abs().sum((0, 1))
        # fp32 sums within a workgroup, at most 2^12 terms a lane, then fp64
        close(got[4 + i], (d * x * r).sum((0, 1)),
              (ed * x.abs() * r).sum((0, 1)) + (norm + 2.0 ** -12) * 0.5 * rows, "grad_weight")


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("n,heads,dim,sections,kind", [
    (1, 1, 2, [1], "int32"), (5, 3, 3, [1], "int64"), (1, 4, 64, [32], "int64"),
    (37, 8, 32, [6, 5, 5], "int32"), (100, 2, 40, [20], "float"), (33, 5, 40, [4, 3, 2], "int32"),
    (64, 1, 128, [64], "int64"), (19, 6, 96, [16, 16, 16], "float"), (9, 3, 250, [125], "int64"),
    (7, 2, 256, [128], "int64"), (12, 2, 255, [100, 3], "int32"), (6, 2, 80, [1, 2, 3, 0, 4, 5, 6, 7],
                                                                  "int32"),
    (1027, 8, 32, [6, 5, 5], "int32"), (2500, 1, 16, [8], "int64"),
])
def test_alone(n, heads, dim, sections, kind, interleaved, dtype):
    q, _, positions, grads, _ = case(n, heads, 1, dim, dtype, sections, kind)
    check_alone(q, positions, sections, interleaved, grads[0])


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("n,heads,kv_heads,dim,sections,kind", [
    (1, 1, 1, 2, [1], "int32"), (3, 4, 2, 5, [2], "int64"), (32, 32, 8, 128, [64], "int64"),
    (41, 8, 8, 32, [6, 5, 5], "int32"), (100, 6, 2, 40, [20], "float"),
    (77, 3, 1, 80, [8, 8, 8], "int32"), (5, 2, 2, 256, [128], "int64"),
    (6, 3, 1, 253, [60, 60], "float"), (1500, 16, 4, 64, [32], "int64"), (900, 1, 1, 8, [2], "int32"),
])
def test_normed(n, heads, kv_heads, dim, sections, kind, interleaved, dtype):
    q, k, positions, grads, weights = case(n, heads, kv_heads, dim, dtype, sections, kind)
    check_normed(q, k, positions, sections, interleaved, grads, weights)


@pytest.mark.parametrize("dtype", DTYPES)
def test_many_rows(dtype):
    """More tiles than workgroups, and more rows of sums than lanes that add them."""
    q, k, positions, grads, weights = case(30011, 8, 2, 64, dtype, [11, 11, 10], "int32")
    check_normed(q, k, positions, [11, 11, 10], False, grads, weights)
    check_alone(q, positions, [11, 11, 10], True, grads[0])


@pytest.mark.parametrize("dtype", DTYPES)
def test_without_weights_and_partial_gradients(dtype):
    from riemannengine import nn
    q, k, positions, grads, _ = case(50, 4, 2, 48, dtype, [24], "int64")
    freq, ones = frequencies([24]), [torch.ones(48, device="cuda")] * 2
    with_ones = nn.norm_rotate_heads(q, k, positions, freq, [24], *ones)
    for a, b in zip(nn.norm_rotate_heads(q, k, positions, freq, [24]), with_ones):
        assert torch.equal(a, b)
    leaf, w = k.detach().requires_grad_(), ones[1].clone().requires_grad_()
    yq, yk = nn.norm_rotate_heads(q, leaf, positions, freq, [24], ones[0], w)
    first = torch.autograd.grad(yk, [leaf, w], grads[1], retain_graph=True)
    both = torch.autograd.grad([yq, yk], [leaf, w], [torch.zeros_like(grads[0]), grads[1]])
    assert all(torch.equal(a, b) for a, b in zip(first, both))


def test_one_axis_positions_and_far_ones():
    """Positions up to 2^31 turn as exactly as near ones."""
    from riemannengine import nn
    x = torch.randn(64, 2, 32, device="cuda")
    far = torch.randint(2 ** 30, 2 ** 31 - 1, (64,), device="cuda", dtype=torch.int32)
    freq = frequencies([16])
    y = nn.rotate_heads(x, far, freq, [16])
    assert torch.equal(y, nn.rotate_heads(x, far[:, None].long(), freq, [16]))
    close(y, turned(x.double(), far[:, None], freq, [16], False),
          (ANGLE + 3 * STEP) * reach(x.double(), [16], False), "far")


def test_no_rows():
    from riemannengine import nn
    q, k, positions, _, weights = case(0, 4, 2, 16, torch.float32, [8], "int64")
    leaves = [w.requires_grad_() for w in weights]
    ys = nn.norm_rotate_heads(q, k, positions, frequencies([8]), [8], *leaves)
    assert ys[0].shape == (0, 4, 16) and ys[1].shape == (0, 2, 16)
    for g in torch.autograd.grad([y.sum() for y in ys], leaves):
        assert not g.any()


def test_what_is_not_finite_stays_in_its_pair():
    from riemannengine import nn
    x = torch.randn(6, 3, 40, device="cuda")
    positions = torch.randint(1, 50, (6, 1), device="cuda")
    clean = nn.rotate_heads(x, positions, frequencies([10]), [10])
    x[2, 1, 3], x[4, 0, 30] = float("nan"), float("inf")
    y = nn.rotate_heads(x, positions, frequencies([10]), [10])
    touched = torch.zeros(x.shape, dtype=torch.bool, device="cuda")
    touched[2, 1, 3] = touched[2, 1, 13] = touched[4, 0, 30] = True
    assert torch.equal(y[~touched], clean[~touched])
    assert y[2, 1, 3].isnan() and y[2, 1, 13].isnan() and y[4, 0, 30] == float("inf")


@pytest.mark.parametrize("dtype", DTYPES)
def test_views(dtype):
    """Rows that start between 16-byte chunks, heads that overlap, gradients of
    one value everywhere and transposed ones."""
    g = torch.Generator(device="cuda").manual_seed(3)
    base = torch.randn((60, 700), generator=g, device="cuda").to(dtype)
    x = base.as_strided((60, 5, 48), (700, 50, 1), 3)
    positions = place(60, [8, 8], "int32", g)
    check_alone(x, positions, [8, 8], False, torch.ones((), dtype=dtype, device="cuda")
                .expand(60, 5, 48))
    gy = torch.randn((5, 60, 48), generator=g, device="cuda").to(dtype).transpose(0, 1)
    k = base.as_strided((60, 2, 48), (700, 0, 1), 400)
    check_normed(x, k, positions, [8, 8], True, [gy, gy[:, :2]],
                 [torch.rand(48, generator=g, device="cuda") + 0.5 for _ in range(2)])


def test_captured_and_repeated():
    from riemannengine import nn
    q, k, positions, grads, weights = case(700, 8, 2, 64, torch.bfloat16, [32], "int64")
    freq = frequencies([32])
    leaves = [t.detach().clone().requires_grad_() for t in (q, k, *weights)]

    def step():
        ys = nn.norm_rotate_heads(*leaves[:2], positions, freq, [32], *leaves[2:])
        return [*(y.detach() for y in ys), *torch.autograd.grad(ys, leaves, grads)]

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = step()
    for seed in (1, 2, 3):
        oq, ok, op, og, ow = case(700, 8, 2, 64, torch.bfloat16, [32], "int64", seed)
        with torch.no_grad():
            for a, b in zip((*leaves, positions, *grads), (oq, ok, *ow, op, *og)):
                a.copy_(b)
        graph.replay()
        torch.cuda.synchronize()
        for a, b in zip(held, step()):
            assert torch.equal(a, b)


def test_frequencies():
    from riemannengine import nn
    f = nn.rotary_frequencies([4, 2], 100.0, "cpu")
    want = [1, 100 ** -0.25, 100 ** -0.5, 100 ** -0.75, 1, 0.1]
    assert f.dtype == torch.float64 and torch.allclose(f, torch.tensor(want, dtype=torch.float64))
    assert nn.rotary_frequencies([3], device=torch.device("cuda")).is_cuda


def test_refusals():
    from riemannengine import nn
    q, k, positions, grads, weights = case(8, 4, 2, 16, torch.float32, [8], "int64")
    f = frequencies([8])
    for args, match in [
            ((q.cpu(), positions, f, [8]), "device tensors"),
            ((q.half(), positions, f, [8]), "fp32 or bf16"),
            ((q[0], positions, f, [8]), "rows, heads, width"),
            ((q, positions[:-1], f, [8]), "positions"),
            ((q, positions.double(), f, [8]), "positions"),
            ((q, positions.cpu(), f, [8]), "positions"),
            ((q, positions, f.float(), [8]), "fp64"),
            ((q, positions, f[:-1], [8]), "fp64"),
            ((q, positions, f, [4, 4]), "positions"),
            ((q, positions, f, [9]), "pairs"),
            ((q, positions, f, [9, -1]), "sections"),
            ((q, positions, f, []), "sections"),
            ((q, positions, f, [1] * 9), "sections"),
            ((torch.zeros(8, 1, 300, device="cuda"), positions, f, [8]), "256"),
            ((q, positions, f.clone().requires_grad_(), [8]), "no gradients")]:
        with pytest.raises(RuntimeError, match=match):
            nn.rotate_heads(*args)
    for args, match in [
            ((q, k[:-1], positions, f, [8]), "keys"), ((q, k.bfloat16(), positions, f, [8]), "keys"),
            ((q, k[..., :-1], positions, f, [8]), "keys"),
            ((q, k, positions, f, [8], weights[0][:-1]), "norm weights"),
            ((q, k, positions, f, [8], weights[0].bfloat16()), "norm weights"),
            ((q, k, positions, f, [8], None, None, 0.0), "eps")]:
        with pytest.raises(RuntimeError, match=match):
            nn.norm_rotate_heads(*args)
    leaf = q.detach().clone().requires_grad_()
    y = nn.rotate_heads(leaf, positions, f, [8])
    with pytest.raises(RuntimeError, match="second derivatives"):
        torch.autograd.grad(y, leaf, grads[0], create_graph=True)
