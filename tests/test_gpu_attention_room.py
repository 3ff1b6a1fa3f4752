"""Keys behind those in use (key_lengths) without a causal mask: their
gradients are exactly zero and what lies there reaches nothing, for fills at
and around the edges of blocks and tiles, in every shape of launch of the
keys' kernel (one, two and four 32-key blocks to a workgroup, the query rows
whole and split over workgroups); the keys in use against the definition in
fp64, within the bounds of attention_reference."""
import math

import pytest
import torch

import riemannengine as rie
from riemannengine_amd import abi
from attention_device import assert_within, attention
from helpers import DEV

pytestmark = pytest.mark.gpu

F32, BF16 = torch.float32, torch.bfloat16


def offsets(lens):
    return torch.tensor([0] + list(lens)).cumsum(0).int().to(DEV)


def cache(seed, q_lens, fills, rooms, heads, kv_heads, dim, dtype):
    """q, k, v, grad, offsets and lengths; the room holds NaN and infinity."""
    g = torch.Generator().manual_seed(seed)
    regions = [f + r for f, r in zip(fills, rooms)]

    def make(*shape):
        return torch.randn(shape, generator=g).to(dtype).to(DEV)

    q, grad = make(sum(q_lens), heads, dim), make(sum(q_lens), heads, dim)
    k, v = make(sum(regions), kv_heads, dim), make(sum(regions), kv_heads, dim)
    k_off = offsets(regions)
    k_len = torch.tensor(fills, dtype=torch.int32, device=DEV)
    spare = torch.zeros(sum(regions), dtype=torch.bool, device=DEV)
    for at, f, n in zip(k_off.tolist(), fills, regions):
        spare[at + f:at + n] = True
    k[spare], v[spare] = math.nan, math.inf
    return q, k, v, grad, offsets(q_lens), k_off, k_len, spare


# query rows, fills, room, heads, key heads, width: what the keys' kernel takes
# in bf16 and fp32 (blocks per workgroup x splits)
CASES = [
    # a few rows over every fill around a block and a tile
    ([7, 40, 1, 33, 64, 5, 130, 9], [20, 31, 32, 33, 63, 65, 127, 129], 45, 4, 2, 32),
    # the smallest score sums: one key in use, many rows
    ([300, 300], [1, 2], 62, 2, 1, 64),
    ([300], [20], 300, 16, 2, 32),                # split over four workgroups
    ([40] * 8, [40, 33, 32, 31, 64, 1, 0, 45], 30, 8, 2, 40),
    ([40] * 64, [33, 40, 64, 17] * 16, 30, 8, 8, 64),
    ([40] * 200, [33, 40, 100, 17] * 50, 40, 8, 8, 96),
    ([40] * 200, [33, 40, 130, 127] * 50, 40, 8, 8, 128),
    ([600] * 3, [567, 601, 640], 130, 16, 2, 128),
    ([2400] * 3, [2400, 2337, 2225], 70, 4, 2, 128),
    ([2400] * 3, [2400, 2337, 2225], 70, 4, 4, 32),
    ([45, 100], [50, 77], 20, 3, 1, 20),          # loaded element by element
]


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("case", range(len(CASES)))
def test_spare_keys_have_no_gradient(dtype, case):
    q_lens, fills, room, heads, kv_heads, dim = CASES[case]
    rooms = [room + 3 * (i % 3) for i in range(len(fills))]
    q, k, v, g, q_off, k_off, k_len, spare = cache(case, q_lens, fills, rooms, heads, kv_heads,
                                                   dim, dtype)
    print("spare keys", q_lens[:4], fills[:8], heads, kv_heads, dim, dtype, flush=True)
    want = attention(q, k, v, q_off, k_off, k_len, grad=g)
    out, lse = abi.attn_forward(q, k, v, q_off, k_off, k_len)
    assert_within(out, want["out"], "out")
    grads = abi.attn_backward(g, q, k, v, out, lse, q_off, k_off, k_len)
    for name, got in zip(("dq", "dk", "dv"), grads):
        assert_within(got, want[name], name)
    assert (grads[1][spare] == 0).all() and (grads[2][spare] == 0).all()


def test_spare_keys_through_autograd():
    q, k, v, g, q_off, k_off, k_len, spare = cache(1, [50, 9], [40, 33], [24, 31], 4, 2, 32, F32)
    k, v = torch.nan_to_num(k), torch.nan_to_num(v)
    leaves = [t.clone().requires_grad_() for t in (q, k, v)]
    rie.nn.packed_attention(*leaves, q_off, k_off, k_len).backward(g)
    want = attention(q, k, v, q_off, k_off, k_len, grad=g)
    for leaf, name in zip(leaves, ("dq", "dk", "dv")):
        assert_within(leaf.grad, want[name], name)
    assert (leaves[1].grad[spare] == 0).all() and (leaves[2].grad[spare] == 0).all()
