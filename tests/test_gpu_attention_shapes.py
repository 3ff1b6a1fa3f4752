"""Every launch shape of the attention kernels (one, two and four 32-row blocks
per workgroup of query rows and of keys, whole and split, rows loaded in
16-byte chunks and element by element) against the definition in fp64, every
element of every head within the bounds of attention_reference. That the
shapes are reached is asserted from rhip_attn_plan, without a GPU."""
import pytest
import torch

from riemannengine_amd import abi
from attention_device import assert_within, attention
from helpers import DEV

F32, BF16 = torch.float32, torch.bfloat16

# query rows, keys (None: the same), heads, key heads
SHAPES = {
    "a few rows": ([40, 170, 90], None, 4, 2),
    "short, 8 heads": ([130] * 32, None, 8, 8),
    "more short ones": ([130] * 64, None, 8, 8),
    "many short ones": ([40] * 200, None, 8, 8),
    "one head": ([45] * 64, None, 1, 1),
    "medium": ([600, 601, 595], None, 16, 2),
    "medium, two": ([1500, 1473], None, 16, 2),
    "long": ([2400, 2337, 2431], None, 16, 4),
    "long, four": ([2400, 2300, 2500, 2399], None, 8, 4),
    "long, few heads": ([2400, 2337, 2431], None, 4, 2),
    "single tokens": ([1, 1, 3, 1], [3000, 1, 700, 129], 8, 2),
    "rows over more keys": ([70, 200, 33], [1100, 900, 33], 8, 2),
}
DIMS = [20, 32, 64, 96, 128]  # 20: no whole 16-byte chunks in bf16


def plan(which, shape, dtype, dim, causal):
    q, k, heads, kv_heads = SHAPES[shape]
    return abi.attn_plan(which, dtype, sum(q), sum(k or q), len(q), heads, kv_heads, dim, causal)


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("dim", DIMS)
def test_the_shapes_reach_every_launch(dtype, dim):
    for causal in (False, True):
        got = {plan("forward", s, dtype, dim, causal) for s in SHAPES}
        assert {b for b, _ in got} == {1, 2, 4} and any(n > 1 for b, n in got)
        assert {plan("queries", s, dtype, dim, causal) for s in SHAPES} == {(1, 1), (2, 1), (4, 1)}
        got = {(b, n > 1) for b, n in (plan("keys", s, dtype, dim, causal) for s in SHAPES)}
        assert got >= {(1, False), (4, False), (4, True)}
    both = {(b, n > 1) for causal in (False, True)
            for b, n in (plan("keys", s, dtype, dim, causal) for s in SHAPES)}
    assert both == {(b, split) for b in (1, 2, 4) for split in (False, True)}


def test_plan_refuses():
    for call, msg in [
        (lambda: abi.attn_plan("forward", F32, 8, 8, 1, 3, 2, 32, False), "multiple"),
        (lambda: abi.attn_plan("keys", F32, 8, 8, 1, 2, 2, 200, False), "128"),
        (lambda: abi.attn_plan("keys", F32, -1, 8, 1, 2, 2, 20, False), "count"),
    ]:
        with pytest.raises(RuntimeError, match=msg):
            call()
    lib, d = abi.lib(), abi.RhipAttn(n_q=1, n_k=1, n_seq=1, heads=1, kv_heads=1, dim=8, scale=1.0)
    import ctypes
    n = ctypes.c_int32()
    assert lib.rhip_attn_plan(ctypes.byref(d), 3, ctypes.byref(n), ctypes.byref(n)) != 0
    assert lib.rhip_attn_plan(ctypes.byref(d), 0, None, ctypes.byref(n)) != 0


@pytest.mark.gpu
@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("dim", DIMS)
@pytest.mark.parametrize("shape", SHAPES)
def test_against_the_definition(shape, dim, dtype, causal):
    q_lens, k_lens, heads, kv_heads = SHAPES[shape]
    k_lens = k_lens or q_lens
    plans = {w: plan(w, shape, dtype, dim, causal) for w in abi.ATTN_PASSES}
    print(shape, dim, dtype, causal, plans, flush=True)
    g = torch.Generator(device=DEV).manual_seed(dim)

    def make(n, h):
        if dim != 20:
            return torch.randn(n, h, dim, generator=g, device=DEV).to(dtype)
        # rows of 23 elements from an odd element on: no 16-byte chunks in fp32 either
        flat = torch.randn(n * h * 23 + 1, generator=g, device=DEV).to(dtype)
        return flat[1:].view(n, h, 23)[:, :, :20]

    q, go = make(sum(q_lens), heads), make(sum(q_lens), heads)
    k, v = make(sum(k_lens), kv_heads), make(sum(k_lens), kv_heads)
    q_off, k_off = (torch.tensor([0] + list(t)).cumsum(0).int().to(DEV) for t in (q_lens, k_lens))
    want = attention(q, k, v, q_off, k_off, causal=causal, grad=go)
    out, lse = abi.attn_forward(q, k, v, q_off, k_off, causal=causal)
    assert_within(out, want["out"], "out")
    grads = abi.attn_backward(go, q, k, v, out, lse, q_off, k_off, causal=causal)
    for name, got in zip(("dq", "dk", "dv"), grads):
        assert_within(got, want[name], name)
