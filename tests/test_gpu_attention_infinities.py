"""Values of attention that are infinite: a row that sees one has that infinity in
its place, whichever of a workgroup's waves and splits found it, and the others keep
what they have without it. Under a causal mask, inside windows, in every shape of
launch."""
import math

import pytest
import torch

from attention_window_device import attention, sees
from helpers import DEV
from riemannengine_amd import abi
from test_gpu_attention_window import SHAPES, make, offsets
from test_gpu_attention_nonfinite import matches

F32, BF16 = torch.float32, torch.bfloat16
DIM = 24
# window, sinks, causal; a window of 10000 is none
CALLS = [(10000, 0, True), (20, 0, True), (20, 0, False), (50, 3, True), (7, 70, False)]


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("window,sinks,causal", CALLS)
@pytest.mark.parametrize("shape", SHAPES)
def test_infinities(shape, window, sinks, causal, dtype):
    q, k, v, qo, ko, _ = make(shape, DIM, dtype, seed=4)
    bad, clean = v.clone(), v.clone()
    special = torch.zeros(q.shape, dtype=torch.float64, device=DEV)
    for s in range(len(qo) - 1):
        q0, k0 = int(qo[s]), int(ko[s])
        lq, lk = int(qo[s + 1]) - q0, int(ko[s + 1]) - k0
        if not lq or not lk:
            continue
        seen = sees(lq, lk, causal, window, sinks, DEV)
        # every 41st key from the third on has +inf in element 5, -inf in 11 or NaN in 23
        for i, (d, value) in enumerate(((5, math.inf), (11, -math.inf), (23, math.nan))):
            keys = torch.arange(lk, device=DEV)[3 + 41 * i::123]
            bad[k0 + keys, :, d] = value
            clean[k0 + keys, :, d] = 0.0
            rows = seen[:, keys].any(1)
            special[q0:q0 + lq, :, d][rows] = value
    window_of = dict(window=None if window == 10000 else window, sinks=sinks)
    out, _ = abi.attn_forward(q, k, bad, qo, ko, causal=causal, **window_of)
    want = attention(q, k, clean, qo, ko, None, causal, None, window, sinks)["out"]
    matches(out, want, special, (shape, window, sinks, causal))


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("window,sinks,causal", CALLS)
@pytest.mark.parametrize("shape", SHAPES)
def test_infinite_gradients(shape, window, sinks, causal, dtype):
    """Of rows' gradients: that infinity in the same place of every key that such a row
    sees; no number in those rows' dq and those keys' dk."""
    q, k, v, qo, ko, go = make(shape, DIM, dtype, seed=5)
    bad, clean = go.clone(), go.clone()
    special = {n: torch.zeros(t.shape, dtype=torch.float64, device=DEV)
               for n, t in (("dq", q), ("dk", k), ("dv", v))}
    for s in range(len(qo) - 1):
        q0, k0 = int(qo[s]), int(ko[s])
        lq, lk = int(qo[s + 1]) - q0, int(ko[s + 1]) - k0
        if not lq or not lk:
            continue
        seen = sees(lq, lk, causal, window, sinks, DEV)
        for i, (d, value) in enumerate(((5, math.inf), (11, -math.inf), (23, math.nan))):
            rows = torch.arange(lq, device=DEV)[3 + 97 * i::291]
            bad[q0 + rows, :, d] = value
            clean[q0 + rows, :, d] = 0.0
            keys = seen[rows].any(0)
            special["dv"][k0:k0 + lk, :, d][keys] = value
            special["dk"][k0:k0 + lk][keys] = math.nan
            special["dq"][q0 + rows[seen[rows].any(1)]] = math.nan
    window_of = dict(window=None if window == 10000 else window, sinks=sinks)
    out, lse = abi.attn_forward(q, k, v, qo, ko, causal=causal, **window_of)
    grads = abi.attn_backward(bad, q, k, v, out, lse, qo, ko, causal=causal, **window_of)
    want = attention(q, k, v, qo, ko, None, causal, clean, window, sinks)
    for name, got in zip(("dq", "dk", "dv"), grads):
        matches(got, want[name], special[name], (name, shape, window, sinks, causal))


@pytest.mark.gpu
@pytest.mark.parametrize("window", [None, 40])
def test_an_infinity_before_a_masked_one(window):
    """32 rows at keys 10 to 41: key 12's infinity lies in one wave's tile, key 40's,
    which rows up to 29 do not see, in another's that has nothing for the first 22."""
    q = torch.randn(32, 1, 16, device=DEV)
    k, v = (torch.randn(42, 1, 16, device=DEV) for _ in range(2))
    v[12, 0, 3], v[40, 0, 7] = math.inf, math.nan
    out, _ = abi.attn_forward(q, k, v, offsets([32]), offsets([42]), causal=True, window=window)
    assert (out[2:, 0, 3] == math.inf).all()
    assert out[:30, 0, 7].isfinite().all() and out[30:, 0, 7].isnan().all()
    rest = [d for d in range(16) if d not in (3, 7)]
    assert out[:, :, rest].isfinite().all() and out[:2, 0, 3].isfinite().all()
