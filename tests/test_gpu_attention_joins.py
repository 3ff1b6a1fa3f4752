"""Gradients of few keys that many rows see: the rows are split over workgroups, whose
partial sums a join adds up. Every number of splits, in the keys' launch and in that
of the sinks' blocks, heads up to 64 wide and wider, against the definition in
fp64."""
import pytest
import torch

import attention_device
import attention_window_device
from attention_device import assert_within
from helpers import DEV
from riemannengine_amd import abi

F32, BF16 = torch.float32, torch.bfloat16
KEYS, HEADS = 45, 4  # over one key head
ROWS = {2: 300, 3: 450, 4: 600, 6: 900, 8: 1200, 12: 1700, 16: 2500, 24: 3500, 32: 5000}
APART = {2: 100, 4: 200, 8: 400, 16: 800, 32: 1600, 64: 3200}
WINDOW, SINKS = 30, 3
DIMS = [33, 40, 64, 65, 80, 128]


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("dim", DIMS)
def test_the_rows_reach_every_number_of_splits(dim, dtype):
    for splits, rows in ROWS.items():
        args = ("keys", dtype, rows, KEYS, 1, HEADS, 1, dim, False)
        assert abi.attn_plan(*args)[1] == splits
    for splits, rows in APART.items():
        args = ("apart", dtype, rows, KEYS, 1, HEADS, 1, dim, False, WINDOW, SINKS)
        assert abi.attn_plan(*args)[1] == splits


def tensors(rows, dim, dtype):
    g = torch.Generator(device=DEV).manual_seed(rows + dim)
    q, go = (torch.randn(rows, HEADS, dim, generator=g, device=DEV).to(dtype) for _ in range(2))
    k, v = (torch.randn(KEYS, 1, dim, generator=g, device=DEV).to(dtype) for _ in range(2))
    q_off, k_off = (torch.tensor([0, n], dtype=torch.int32, device=DEV) for n in (rows, KEYS))
    return go, q, k, v, q_off, k_off


def check(definition, rows, dim, dtype, **window):
    go, q, k, v, q_off, k_off = tensors(rows, dim, dtype)
    want = definition.attention(q, k, v, q_off, k_off, grad=go, **window)
    out, lse = abi.attn_forward(q, k, v, q_off, k_off, **window)
    grads = abi.attn_backward(go, q, k, v, out, lse, q_off, k_off, **window)
    for name, got in zip(("dq", "dk", "dv"), grads):
        assert_within(got, want[name], name)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("dim", DIMS)
@pytest.mark.parametrize("splits", ROWS)
def test_keys(splits, dim, dtype):
    check(attention_device, ROWS[splits], dim, dtype)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("dim", DIMS)
@pytest.mark.parametrize("splits", APART)
def test_sinks(splits, dim, dtype):
    check(attention_window_device, APART[splits], dim, dtype, window=WINDOW, sinks=SINKS)
