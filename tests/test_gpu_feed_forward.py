"""riemannengine.nn.gated_feed_forward against its definition in fp64: sizes from
one row and one channel to several tiles, views, both types and activations."""
import pytest
import torch

from feed_forward_reference import assert_close, reference

pytestmark = pytest.mark.gpu
NAMES = ("y", "grad_x", "grad_gate", "grad_up", "grad_down")
DTYPES = [torch.float32, torch.bfloat16]


def make(n, channels, hidden, outputs, dtype, seed=0):
    g = torch.Generator(device="cuda").manual_seed(seed)

    def normal(*shape, scale=1.0):
        return (torch.randn(shape, generator=g, device="cuda") * scale).to(dtype)

    return (normal(n, channels), normal(hidden, channels, scale=channels ** -0.5),
            normal(hidden, channels, scale=channels ** -0.5),
            normal(outputs, hidden, scale=hidden ** -0.5), normal(n, outputs))


def train(x, gate, up, down, grad_y, kind):
    from riemannengine import nn
    leaves = [t.detach().requires_grad_() for t in (x, gate, up, down)]
    y = nn.gated_feed_forward(*leaves, kind)
    return [y.detach(), *torch.autograd.grad(y, leaves, grad_y)]


def check(x, gate, up, down, grad_y, kind):
    from riemannengine import nn
    want = reference(x, gate, up, down, kind, grad_y)
    for got, ref, name in zip(train(x, gate, up, down, grad_y, kind), want, NAMES):
        assert got.dtype == x.dtype
        assert_close(got, ref, name)
    with torch.no_grad():
        assert_close(nn.gated_feed_forward(x, gate, up, down, kind), want[0], "inference")


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("kind", ["silu", "gelu"])
@pytest.mark.parametrize("n,channels,hidden,outputs", [
    (1, 1, 1, 1), (1, 64, 96, 64), (3, 7, 5, 9), (16, 33, 47, 12), (17, 128, 200, 64),
    (33, 256, 100, 256), (64, 40, 1000, 40), (65, 40, 1000, 41), (128, 128, 128, 128),
    (129, 63, 130, 65), (300, 96, 257, 96), (257, 520, 300, 136), (1000, 32, 17, 32),
    (200, 33, 47, 12), (256, 96, 200, 96), (193, 600, 700, 600),  # few rows in several parts
])
def test_sizes(n, channels, hidden, outputs, kind, dtype):
    check(*make(n, channels, hidden, outputs, dtype), kind)


# tiles of 256 rows and columns, and sums over k split or not
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("n,channels,hidden", [
    (4096, 1024, 2048), (4000, 1000, 2100), (70, 2048, 4099), (8300, 64, 96), (513, 4096, 512), (180, 2048, 4099),
    (3200, 1024, 1536),  # fp32: parts that hold whole tiles and share their ends
])
def test_large(n, channels, hidden, dtype):
    check(*make(n, channels, hidden, channels, dtype, seed=1), "silu")


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("n", [5, 200])
def test_views(n, dtype):
    """Row strides, starts between 16-byte chunks, weights that are parts of one
    matrix, a transposed gradient and one that is a single value everywhere."""
    x, gate, up, down, gy = make(n, 67, 90, 50, dtype, seed=2)
    x = torch.cat([x, x], 1)[:, 5:5 + 64]
    both = torch.cat([gate, up], 0)
    gate, up = both[:90, 1:65], both[90:, 3:67]
    down = torch.cat([down, down], 1)[:, 7:97]
    check(x, gate, up, down, gy.t().contiguous().t(), "silu")
    check(x, gate, up, down, torch.ones(1, 1, dtype=dtype, device="cuda").expand(n, 50), "gelu")


def test_far_activations():
    """Projections far from zero: the activation and its slope keep their limits."""
    for kind in ("silu", "gelu"):
        for dtype in DTYPES:
            x, gate, up, down, gy = make(96, 64, 80, 48, dtype, seed=3)
            check(x * 4, gate * 2, up, down, gy, kind)


@pytest.mark.parametrize("dtype", DTYPES)
def test_no_rows(dtype):
    x, gate, up, down, gy = make(0, 24, 40, 16, dtype)
    y, gx, *weights = train(x, gate, up, down, gy, "silu")
    assert y.shape == (0, 16) and gx.shape == (0, 24)
    assert all(not w.any() for w in weights)


def test_leading_axes_and_single_gradients():
    from riemannengine import nn
    x, gate, up, down, _ = make(30, 24, 40, 16, torch.float32)
    flat = nn.gated_feed_forward(x, gate, up, down)
    assert torch.equal(nn.gated_feed_forward(x.view(5, 6, 24), gate, up, down),
                       flat.view(5, 6, 16))
    assert torch.equal(nn.gated_feed_forward(x[0], gate, up, down), flat[0])
    whole = train(x, gate, up, down, torch.ones_like(flat), "silu")[1:]
    for i in range(4):
        leaves = [t.detach().requires_grad_(j == i) for j, t in enumerate((x, gate, up, down))]
        y = nn.gated_feed_forward(*leaves)
        grad, = torch.autograd.grad(y, [leaves[i]], torch.ones_like(y))
        assert torch.equal(grad, whole[i])


@pytest.mark.parametrize("dtype", DTYPES)
def test_gradients_by_differences(dtype):
    """A step along random directions: the change of sum(y * w) is what the
    gradients say, up to the second order of a step of 2^-6 and the roundings."""
    x, gate, up, down, w = make(70, 24, 40, 16, torch.float32, seed=4)
    grads = train(*(t.to(dtype) for t in (x, gate, up, down, w)), "silu")[1:]
    g = torch.Generator(device="cuda").manual_seed(5)
    h = 2.0 ** -6
    for i, grad in enumerate(grads):
        args = [t.to(dtype).double() for t in (x, gate, up, down)]
        turn = torch.randn(grad.shape, generator=g, device="cuda", dtype=torch.float64)
        turn /= turn.norm()

        def value(step):
            moved = [t + step * turn if j == i else t for j, t in enumerate(args)]
            a = torch.nn.functional.silu(moved[0] @ moved[1].t()) * (moved[0] @ moved[2].t())
            return ((a @ moved[3].t()) * w.to(dtype).double()).sum()

        # the fourth-order difference quotient: its error is below 1e-6 here
        slope = (8 * (value(h) - value(-h)) - (value(2 * h) - value(-2 * h))) / (12 * h)
        said = (grad.double() * turn).sum()
        # roundings of dg, du, h and the result, all in the same direction at most
        bound = (4 * torch.finfo(dtype).eps + 1e-6) * grad.double().norm()
        assert abs(slope - said) <= bound


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("n", [9, 150])
def test_what_is_not_finite_stays_in_its_rows(n, dtype):
    """Odd widths fill up to whole chunks beside NaN and infinities."""
    from riemannengine import nn
    x, gate, up, down, _ = make(n, 37, 45, 23, dtype, seed=6)
    clean = nn.gated_feed_forward(x, gate, up, down)
    x[3, 5], x[7, 0] = float("nan"), float("inf")
    y = nn.gated_feed_forward(x, gate, up, down)
    others = [i for i in range(n) if i not in (3, 7)]
    assert torch.equal(y[others], clean[others])
    assert y[3].isnan().all() and not y[7].isfinite().any()


def test_runs_repeat_and_match_another_stream():
    x, gate, up, down, gy = make(900, 512, 700, 512, torch.bfloat16, seed=7)
    first = train(x, gate, up, down, gy, "silu")
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        second = train(x, gate, up, down, gy, "silu")
    torch.cuda.current_stream().wait_stream(stream)
    assert all(torch.equal(a, b) for a, b in zip(first, second))


@pytest.mark.parametrize("n", [4, 300])
def test_captured(n):
    """A training step in a graph, replayed with other rows."""
    from riemannengine import nn
    x, gate, up, down, gy = make(n, 64, 100, 64, torch.bfloat16, seed=8)
    leaves = [t.detach().requires_grad_() for t in (x, gate, up, down)]

    def step():
        y = nn.gated_feed_forward(*leaves)
        return [y.detach(), *torch.autograd.grad(y, leaves, gy)]

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = step()
    for seed in (9, 10, 11):
        other = make(n, 64, 100, 64, torch.bfloat16, seed=seed)
        with torch.no_grad():
            for a, b in zip((*leaves, gy), other):
                a.copy_(b)
        graph.replay()
        torch.cuda.synchronize()
        for a, b in zip(held, train(*other, "silu")):
            assert torch.equal(a, b)


def test_refusals():
    from riemannengine import nn
    x, gate, up, down, gy = make(8, 24, 40, 16, torch.float32)
    call = nn.gated_feed_forward
    for args, match in [
            ((x.cpu(), gate, up, down), "device tensor"),
            ((x.half(), gate, up, down), "fp32 or bf16"),
            ((x, gate.bfloat16(), up, down), "dtype and device"),
            ((x, gate[:, :-1], up, down), "hidden"),
            ((x, gate, up[:-1], down), "hidden"),
            ((x, gate, up, down[:, :-1]), "outputs"),
            ((x, gate, up, down.cpu()), "dtype and device"),
            ((x, gate, up, down, "relu"), "silu"),
            ((x[:, :0], gate[:, :0], up[:, :0], down), "channel"),
            ((x, gate[:0], up[:0], down[:, :0]), "hidden")]:
        with pytest.raises(RuntimeError, match=match):
            call(*args)
    leaf = x.clone().requires_grad_()
    y = call(leaf, gate, up, down)
    with pytest.raises(RuntimeError, match="second derivatives"):
        torch.autograd.grad(y, leaf, gy, create_graph=True)
    import torch.autograd.forward_ad as fwd
    with fwd.dual_level():
        with pytest.raises(RuntimeError):
            call(fwd.make_dual(x, torch.ones_like(x)), gate, up, down)
