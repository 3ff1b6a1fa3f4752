"""Sizes past 32 bits, which a C call's int32 would take for others, are refused by
the ctypes callers, without a GPU."""
import pytest
import torch

from riemannengine_amd import abi

BIG = 2 ** 32 + 8  # as an int32: 8


@pytest.fixture
def no_library(monkeypatch):
    monkeypatch.setattr(abi, "_require_cuda", lambda t, name: None)
    monkeypatch.setattr(abi, "lib", lambda: pytest.fail("the library was called"))


def there(*shape, dtype=torch.bfloat16):
    return torch.empty(shape, dtype=dtype, device="meta")


@pytest.mark.parametrize("x,gate,down", [
    (there(1, BIG), there(24, BIG), there(8, 24)),
    (there(1, 16), there(BIG, 16), there(8, BIG)),
    (there(1, 16), there(24, 16), there(BIG, 24)),
])
def test_gated(no_library, x, gate, down):
    with pytest.raises(RuntimeError, match="32 bits"):
        abi.gated_forward(x, gate, gate, down)
    with pytest.raises(RuntimeError, match="32 bits"):
        abi.gated_backward(there(1, down.shape[0]), x, gate, gate, down,
                           there(8, dtype=torch.uint8))


@pytest.mark.parametrize("sizes", [(1, BIG, 8, 8), (1, 8, BIG, 8), (1, 8, 8, BIG)])
def test_gated_plan(no_library, sizes):
    with pytest.raises(RuntimeError, match="32 bits"):
        abi.gated_plan("output", torch.float32, *sizes)


@pytest.mark.parametrize("q,k", [
    (there(1, BIG, 16), None), (there(1, 2, BIG), None), (there(1, 2, 16), there(1, BIG, 16)),
])
def test_rotary(no_library, q, k):
    args = (q, k, there(1, 1, dtype=torch.int32), there(4, dtype=torch.float64), [4])
    with pytest.raises(RuntimeError, match="32 bits"):
        abi.rotary_forward(*args)
    with pytest.raises(RuntimeError, match="32 bits"):
        abi.rotary_backward((q, k), *args)


@pytest.mark.parametrize("q,k", [
    (there(1, BIG, 16), there(1, 8, 16)), (there(1, 8, 16), there(1, BIG, 16)),
    (there(1, 1, BIG), there(1, 1, BIG)),
])
def test_attention_inside_a_window(no_library, q, k):
    offsets = there(2, dtype=torch.int32)
    with pytest.raises(RuntimeError, match="32 bits"):
        abi.attn_forward(q, k, k, offsets, offsets, window=4)
    with pytest.raises(RuntimeError, match="32 bits"):
        abi.attn_backward(q, q, k, k, q, there(q.shape[1], 1, dtype=torch.float32), offsets,
                          offsets, window=4)


@pytest.mark.parametrize("at", range(4))
def test_attention_plan(no_library, at):
    sizes = [1, 8, 8, 16]
    sizes[at] = BIG
    with pytest.raises(RuntimeError, match="32 bits"):
        abi.attn_plan("forward", torch.float32, 8, 8, *sizes, False)
