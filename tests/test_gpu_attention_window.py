"""riemannengine.nn.packed_attention inside a window, with sinks and without,
against the definition in fp64, in every shape of launch: windows of one key to
more than there are, on both sides and under a causal mask, caches with spare
room, rows that see nothing, values that are not finite in masked places."""
import pytest
import torch

from riemannengine_amd import abi
from attention_device import assert_within
from attention_window_device import attention, sees
from helpers import DEV

F32, BF16 = torch.float32, torch.bfloat16
# query rows, keys (None: the same), heads, key heads
SHAPES = {
    "a few rows": ([40, 170, 0, 90], None, 4, 2),
    "more short ones": ([130] * 64, None, 8, 8),
    "many short ones": ([40] * 200, None, 8, 8),
    "medium": ([600, 601, 595], None, 16, 2),
    "medium, two": ([1500, 1473], None, 16, 2),
    "long": ([2400, 2337, 2431], None, 16, 4),
    "long, few heads": ([2400, 2337, 2431], None, 4, 2),
    "single tokens": ([1, 1, 3, 1], [3000, 1, 700, 129], 8, 2),
    "rows over more keys": ([70, 200, 33], [1100, 900, 33], 8, 2),
    "rows over fewer keys": ([200, 70, 300], [90, 64, 0], 4, 4),
}
# window, sinks, causal
WINDOWS = [(1, 0, True), (1, 3, False), (33, 0, False), (100, 4, True), (64, 32, False),
           (700, 40, True), (5000, 2, True), (300, 5000, False)]


def offsets(lens):
    return torch.tensor([0] + list(lens)).cumsum(0).int().to(DEV)


def make(shape, dim, dtype, seed=0):
    q, k, heads, kv_heads = SHAPES[shape]
    g = torch.Generator(device=DEV).manual_seed(seed)

    def normal(n, h):
        return torch.randn(n, h, dim, generator=g, device=DEV).to(dtype)

    k = k or q
    return (normal(sum(q), heads), normal(sum(k), kv_heads), normal(sum(k), kv_heads),
            offsets(q), offsets(k), normal(sum(q), heads))


def train(q, k, v, qo, ko, go, causal, window, sinks, k_len=None):
    from riemannengine import nn
    leaves = [t.detach().requires_grad_() for t in (q, k, v)]
    out = nn.packed_attention(*leaves, qo, ko, k_len, causal, window=window, sinks=sinks)
    return [out.detach(), *torch.autograd.grad(out, leaves, go)]


def check(q, k, v, qo, ko, go, causal, window, sinks, k_len=None):
    from riemannengine import nn
    want = attention(q, k, v, qo, ko, k_len, causal, go, window, sinks)
    for got, name in zip(train(q, k, v, qo, ko, go, causal, window, sinks, k_len),
                         ("out", "dq", "dk", "dv")):
        assert_within(got, want[name], name)
    with torch.no_grad():
        assert_within(nn.packed_attention(q, k, v, qo, ko, k_len, causal, window=window,
                                          sinks=sinks), want["out"], "inference")


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_the_shapes_reach_every_launch(dtype):
    got = {w: set() for w in abi.ATTN_WINDOW_PASSES}
    for q, k, heads, kv_heads in SHAPES.values():
        for window, sinks, causal in WINDOWS:
            for which in got:
                blocks, splits = abi.attn_plan(which, dtype, sum(q), sum(k or q), len(q), heads,
                                               kv_heads, 64, causal, window, sinks)
                got[which].add((blocks, splits > 1))
    assert {b for b, _ in got["forward"]} == {1, 2, 4} and (1, True) in got["forward"]
    assert {b for b, _ in got["queries"]} == {1, 2, 4}
    assert {b for b, _ in got["keys"]} == {1, 2, 4}
    assert got["apart"] == {(0, False), (1, False), (1, True)}


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("dim", [20, 32, 64, 96, 128])
@pytest.mark.parametrize("shape", list(SHAPES))
def test_every_launch(shape, dim, dtype):
    args = make(shape, dim, dtype)
    for i, (window, sinks, causal) in enumerate(WINDOWS):
        if dim in (32, 128) or (i + dim // 4) % 2:
            print(shape, dim, dtype, window, sinks, causal, flush=True)
            check(*args, causal, window, sinks)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("causal", [False, True])
def test_around_the_tiles(causal, dtype):
    """Windows and sinks a key less and more than the kernels' tiles."""
    g = torch.Generator(device=DEV).manual_seed(1)
    lens = [255, 64, 1, 130]
    q, go = (torch.randn(450, 4, 32, generator=g, device=DEV).to(dtype) for _ in range(2))
    k, v = (torch.randn(450, 2, 32, generator=g, device=DEV).to(dtype) for _ in range(2))
    o = offsets(lens)
    for window in (2, 31, 32, 33, 63, 64, 65, 127, 128, 129):
        for sinks in (0, 1, 31, 32, 33, 65):
            check(q, k, v, o, o, go, causal, window, sinks)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [F32, BF16])
def test_a_wide_window_is_no_window(dtype):
    from riemannengine import nn
    q, k, v, qo, ko, _ = make("medium", 64, dtype)
    for causal in (False, True):
        want = nn.packed_attention(q, k, v, qo, ko, causal=causal)
        for window in (601, 2 ** 31 - 1, 2 ** 40):
            got = nn.packed_attention(q, k, v, qo, ko, causal=causal, window=window)
            # the same launch, the same products in the same order
            assert torch.equal(got, want)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("causal", [False, True])
def test_caches_with_room(causal, dtype):
    """Keys in use of larger regions: those behind them, NaN here, are not read
    and get zero gradients; rows behind the last sequence get zeros."""
    g = torch.Generator(device=DEV).manual_seed(2)
    q_lens, used, room = [1, 40, 1, 7], [500, 300, 1, 0], [700, 300, 64, 5]
    q, go = (torch.randn(sum(q_lens) + 9, 8, 64, generator=g, device=DEV).to(dtype)
             for _ in range(2))
    k, v = (torch.randn(sum(room) + 40, 2, 64, generator=g, device=DEV).to(dtype)
            for _ in range(2))
    ko = offsets(room)
    free = torch.ones(k.shape[0], dtype=torch.bool, device=DEV)
    for at, n in zip(ko.tolist(), used):
        free[at:at + n] = False
    k[free], v[free] = float("nan"), float("inf")
    k_len = torch.tensor(used, dtype=torch.int32, device=DEV)
    for window, sinks in ((1, 0), (100, 4), (64, 200), (10 ** 6, 0)):
        clean_k, clean_v = k.masked_fill(free[:, None, None], 0), v.masked_fill(free[:, None, None], 0)
        want = attention(q, clean_k, clean_v, offsets(q_lens), ko, k_len, causal, go, window,
                         sinks)
        got = train(q, k, v, offsets(q_lens), ko, go, causal, window, sinks, k_len)
        for t, name in zip(got, ("out", "dq", "dk", "dv")):
            assert_within(t, want[name], name)
        assert not got[0][sum(q_lens):].any() and not got[1][sum(q_lens):].any()
        assert not got[2][free].any() and not got[3][free].any()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("shape,dim", [("a few rows", 64), ("more short ones", 32), ("medium", 128),
                                       ("medium, two", 64), ("long", 64), ("long", 128),
                                       ("rows over more keys", 20)])
def test_what_is_not_finite_reaches_only_what_sees_it(shape, dim, dtype):
    """What does not see such a value keeps its result. (Not bit for bit: the rows
    of a wave take a step of their running maximum together, and one whose
    maximum m stays is then scaled by exp2(m c - round(m c)), as near to 1 as
    the products' rounding, 2^-24 |m c|, allows; the bounds' e has it.)"""
    q, k, v, qo, ko, go = make(shape, dim, dtype, seed=3)
    heads, kv_heads = q.shape[1], k.shape[1]
    s = 1
    q0, lq = int(qo[s]), int(qo[s + 1] - qo[s])
    k0, lk = int(ko[s]), int(ko[s + 1] - ko[s])
    names = ("out", "dq", "dk", "dv")

    def hold(got, want, rows, keys, what):
        """All but the marked rows and keys are within their bounds."""
        for t, name, marked in zip(got, names, (rows, rows, keys, keys)):
            value, bound = want[name]
            assert_within(t[~marked], (value[~marked], bound[~marked]), (name, *what))

    for window, sinks, causal in ((20, 0, False), (50, 3, True), (1, 40, False)):
        seen = sees(lq, lk, causal, window, sinks, DEV)
        want = attention(q, k, v, qo, ko, None, causal, go, window, sinks)
        for key in (1, lk // 2 + 5, lk - 21):  # a sink, and keys inside and at the end
            for what, value in (("k", float("nan")), ("v", float("nan")), ("v", float("inf"))):
                bad_k, bad_v = k.clone(), v.clone()
                (bad_k if what == "k" else bad_v)[k0 + key, 0, dim // 3] = value
                got = train(q, bad_k, bad_v, qo, ko, go, causal, window, sinks)
                rows = torch.zeros(q.shape[:2], dtype=torch.bool, device=DEV)
                rows[q0:q0 + lq, :heads // kv_heads] = seen[:, key, None]
                keys = torch.zeros(k.shape[:2], dtype=torch.bool, device=DEV)
                # keys that share a row with it
                keys[k0:k0 + lk, 0] = (seen[seen[:, key]].any(0) if seen[:, key].any()
                                       else torch.zeros(lk, dtype=torch.bool, device=DEV))
                keys[k0 + key, 0] = True
                hold(got, want, rows, keys, (window, sinks, key, what))
                assert not got[0][rows][:, dim // 3].isfinite().any()
        for row in (2, lq // 2, lq - 1):
            for what, value in (("q", float("nan")), ("go", float("inf"))):
                bad_q, bad_go = q.clone(), go.clone()
                (bad_q if what == "q" else bad_go)[q0 + row, 0, dim // 3] = value
                got = train(bad_q, k, v, qo, ko, bad_go, causal, window, sinks)
                rows = torch.zeros(q.shape[:2], dtype=torch.bool, device=DEV)
                rows[q0 + row, 0] = True
                keys = torch.zeros(k.shape[:2], dtype=torch.bool, device=DEV)
                keys[k0:k0 + lk, 0] = seen[row]
                hold(got, want, rows, keys, (window, sinks, row, what))
                if seen[row].any():
                    assert not got[3][keys][:, dim // 3].isfinite().any()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [F32, BF16])
def test_captured_and_repeated(dtype):
    from riemannengine import nn
    q, k, v, qo, ko, go = make("medium", 64, dtype)
    leaves = [t.detach().clone().requires_grad_() for t in (q, k, v)]

    def step():
        out = nn.packed_attention(*leaves, qo, ko, causal=True, window=90, sinks=5)
        return [out.detach(), *torch.autograd.grad(out, leaves, go)]

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = step()
    for seed in (1, 2, 3):
        other = make("medium", 64, dtype, seed)
        with torch.no_grad():
            for a, b in zip((*leaves, go), (*other[:3], other[5])):
                a.copy_(b)
        graph.replay()
        torch.cuda.synchronize()
        for a, b in zip(held, step()):
            assert torch.equal(a, b)


@pytest.mark.gpu
def test_strides_and_scale():
    from riemannengine import nn
    g = torch.Generator(device=DEV).manual_seed(4)
    rows = torch.randn(300, 12, 40, generator=g, device=DEV)
    q, k, v = rows[:, :6], rows[:, 6:9], rows[:, 9:]
    o = offsets([120, 180])
    for scale in (0.05, 2.0):
        want = attention(q, k, v, o, o, None, True, None, 37, 2, scale)
        got = nn.packed_attention(q, k, v, o, None, None, True, scale, 37, 2)
        assert_within(got, want["out"], "out")


@pytest.mark.gpu
def test_refusals():
    from riemannengine import nn
    q, k, v, qo, ko, _ = make("a few rows", 32, F32)
    for kw, match in [({"window": 0}, "at least one key"), ({"window": -3}, "at least one key"),
                      ({"window": 4, "sinks": -1}, "sinks"), ({"sinks": 2}, "beside a window"),
                      ({"window": 4, "sinks": 2 ** 31}, "sinks")]:
        with pytest.raises(RuntimeError, match=match):
            nn.packed_attention(q, k, v, qo, ko, **kw)


def test_plan_refuses():
    for args, match in [(("keys", F32, 8, 8, 1, 2, 2, 32, False, 0), "window"),
                        (("keys", F32, 8, 8, 1, 2, 2, 32, False, 3, -1), "sinks"),
                        (("apart", F32, 8, 8, 1, 2, 2, 32, False), "apart")]:
        with pytest.raises(RuntimeError, match=match):
            abi.attn_plan(*args)
