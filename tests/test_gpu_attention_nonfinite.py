"""Infinities and NaN in causal attention: element by element, a result is not
finite where the definition makes it so (a row, or a key, that sees such a
value) and within the bounds of attention_reference everywhere else, in every
shape of launch; and such inputs, as of a step that diverges, cost no more
than a few times a clean call."""
import math

import pytest
import torch

from riemannengine_amd import abi
from attention_device import attention
from helpers import DEV

pytestmark = pytest.mark.gpu

F32, BF16 = torch.float32, torch.bfloat16
INF, NAN = math.inf, math.nan

# sequences' lengths, heads, key heads: one, two and four 32-row blocks per
# workgroup of rows and of keys, with and without split keys' kernels
SHAPES = [([40, 170, 90], 4, 2), ([130] * 32, 8, 8), ([130] * 64, 8, 8),
          ([2400] * 3, 16, 4), ([2400] * 4, 8, 4), ([1500] * 2, 16, 2)]
KINDS = ["values", "grad_out", "key", "low_key", "query", "queries"]


def offsets(lens):
    return torch.tensor([0] + list(lens)).cumsum(0).int().to(DEV)


def matches(got, want, special, what):
    """got within its bound of want but where `special` (NaN: not finite, an
    infinity: that infinity, else 0) is set."""
    val, err = want
    got = got.double()
    plain = special == 0
    diff = (got - val).abs()
    bad = plain & ~(diff <= 1.01 * err + 1e-30)
    assert not bad.any(), (what, int(bad.sum()), bad.nonzero()[0].tolist())
    assert not torch.isfinite(got[special.isnan()]).any(), what
    signed = special.isinf()
    assert torch.equal(got[signed], special[signed]), what


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("shape,dim", [(0, 32), (0, 64), (0, 96), (0, 128), (0, 20), (1, 32),
                                       (1, 64), (1, 96), (1, 128), (2, 20), (2, 32), (2, 64),
                                       (2, 96), (2, 128), (3, 32), (3, 64), (3, 128), (4, 64),
                                       (4, 128), (5, 64), (5, 128)])
def test_only_what_sees_it(shape, dim, dtype, kind):
    lens, heads, kv_heads = SHAPES[shape]
    n = sum(lens)
    g = torch.Generator(device=DEV).manual_seed(shape * 1000 + dim)
    q, go = (torch.randn(n, heads, dim, generator=g, device=DEV).to(dtype) for _ in range(2))
    k, v = (torch.randn(n, kv_heads, dim, generator=g, device=DEV).to(dtype) for _ in range(2))
    o = offsets(lens)
    s = 1  # the sequence they lie in: rows a .. b - 1
    a, b = int(o[s]), int(o[s + 1])
    first, second = a + (b - a) // 2 + 5, a + (b - a) - 21
    d1, d2 = dim // 3, dim - 1
    print(kind, lens[:3], len(lens), heads, kv_heads, dim, dtype, flush=True)
    nothing = {"out": q, "dq": q, "dk": k, "dv": k}
    special = {m: torch.zeros(t.shape, dtype=torch.float64, device=DEV)
               for m, t in nothing.items()}
    inputs = {"q": q, "k": k, "v": v, "go": go}
    clean = dict(inputs)
    k_off = o

    def put(name, row, d, value):
        if inputs[name] is clean[name]:
            inputs[name], clean[name] = inputs[name].clone(), clean[name].clone()
        inputs[name][row, :, d] = value
        clean[name][row, :, d] = 0.0

    if kind == "values":
        put("v", first, d1, INF)
        put("v", second, d2, NAN)
        special["out"][first:b, :, d1] = INF
        special["out"][second:b, :, d2] = NAN
        special["dq"][first:b] = NAN  # their grad_out . out is not finite
        special["dk"][a:b] = NAN
    elif kind == "grad_out":
        put("go", first, d1, -INF)
        put("go", second, d2, NAN)
        special["dv"][a:first + 1, :, d1] = -INF
        special["dv"][a:second + 1, :, d2] = NAN
        special["dq"][first] = special["dq"][second] = NAN
        special["dk"][a:second + 1] = NAN
    elif kind == "key":
        put("k", first, d1, NAN)
        special["out"][first:b] = special["dq"][first:b] = NAN
        special["dk"][a:b] = special["dv"][a:b] = NAN
    elif kind == "low_key":
        # the sequence's first key has a score of -inf in every row: no weight,
        # and 0 * -inf in the gradient of q. The others as without that key.
        q[:, :, d1] = 1
        put("k", a, d1, -INF)
        special["dq"][a:b, :, d1] = NAN
    else:
        put("q", first, d1, NAN if kind == "query" else INF)
        special["out"][first] = special["dq"][first] = NAN
        special["dk"][a:first + 1] = special["dv"][a:first + 1] = NAN
        if kind == "queries":  # two rows, the later one of NaN throughout
            put("q", second, slice(None), NAN)
            special["out"][second] = special["dq"][second] = NAN
            special["dk"][a:second + 1] = special["dv"][a:second + 1] = NAN
    if kind == "low_key":
        keep = torch.arange(n, device=DEV) != a
        k_off = o - (o > a).int()  # row i sees one key less: the first is gone
        want = attention(q, k[keep], v[keep], o, k_off, causal=True, grad=go)
        for m in ("dk", "dv"):
            want[m] = tuple(torch.cat([t[:a], torch.zeros_like(t[:1]), t[a:]]) for t in want[m])
        # row a of the sequence now sees nothing but that key: probability 1 of
        # a score of -inf is no number; what the kernels give is not checked
        special["out"][a], special["dq"][a] = 0.0, 0.0
        rows = torch.arange(n, device=DEV) != a
    else:
        want = attention(clean["q"], clean["k"], clean["v"], o, o, causal=True, grad=clean["go"])
        rows = torch.ones(n, dtype=torch.bool, device=DEV)
    q, k, v, go = (inputs[m] for m in ("q", "k", "v", "go"))
    out, lse = abi.attn_forward(q, k, v, o, o, causal=True)

    def check(name, got, pick=slice(None)):
        matches(got[pick], tuple(t[pick] for t in want[name]), special[name][pick], name)

    check("out", out, rows)
    if kind == "low_key":
        go = go.clone()
        go[a] = 0  # of the row that is not checked
        lse[:, a] = 0
        want2 = attention(q, k[keep], v[keep], o, k_off, causal=True, grad=go)
        for m in ("dq", "dk", "dv"):
            want[m] = want2[m]
        for m in ("dk", "dv"):
            want[m] = tuple(torch.cat([t[:a], torch.zeros_like(t[:1]), t[a:]]) for t in want[m])
    dq, dk, dv = abi.attn_backward(go, q, k, v, out, lse, o, o, causal=True)
    check("dq", dq, rows)
    check("dk", dk)
    check("dv", dv)


@pytest.mark.parametrize("what", ["first value", "all queries", "all values", "all gradients"])
@pytest.mark.parametrize("dtype", [F32, BF16])
def test_time(dtype, what):
    """Two causal sequences of 2000: at most 4 times a clean call and 100 us."""
    heads, dim, lens = 4, 64, [2000, 2000]
    n = sum(lens)
    g = torch.Generator(device=DEV).manual_seed(0)
    q, k, v, go = (torch.randn(n, heads, dim, generator=g, device=DEV).to(dtype)
                   for _ in range(4))
    o = offsets(lens)

    def step(q, v, go):
        out, lse = abi.attn_forward(q, k, v, o, o, causal=True)
        abi.attn_backward(go, q, k, v, out, lse, o, o, causal=True)

    def best(*args):
        times = []
        for _ in range(5):
            start, end = (torch.cuda.Event(enable_timing=True) for _ in range(2))
            start.record()
            step(*args)
            end.record()
            end.synchronize()
            times.append(start.elapsed_time(end))
        return min(times[1:])

    clean = best(q, v, go)
    if what == "first value":
        v = v.clone()
        v[0] = NAN
    elif what == "all queries":
        q = torch.full_like(q, NAN)
    elif what == "all values":
        v = torch.full_like(v, NAN)
    else:
        go = torch.full_like(go, NAN)
    bad = best(q, v, go)
    print(what, dtype, clean, bad, flush=True)
    assert bad <= 4 * clean + 0.1
