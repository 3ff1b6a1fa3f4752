"""Heads and widths past 32 bits, of tensors that repeat one value, are refused before
a result of that size is asked for."""
import pytest
import torch

from helpers import DEV

pytestmark = pytest.mark.gpu
BIG = 2 ** 32 + 8  # as an int32: 8


def test_refusals():
    from riemannengine import nn
    few, wide = (torch.ones(1, 1, 1, device=DEV).expand(s) for s in ((1, BIG, 8), (1, 1, BIG)))
    x = torch.ones(1, 8, 8, device=DEV)
    places = torch.zeros(1, 1, dtype=torch.int32, device=DEV)
    freq = nn.rotary_frequencies([4])
    offsets = torch.tensor([0, 1], dtype=torch.int32, device=DEV)
    for call, match in [
            (lambda: nn.rotate_heads(few, places, freq, [4]), "heads"),
            (lambda: nn.rotate_heads(wide, places, freq, [4]), "widths up to 256"),
            (lambda: nn.norm_rotate_heads(few, x, places, freq, [4]), "heads"),
            (lambda: nn.norm_rotate_heads(x, few, places, freq, [4]), "heads"),
            (lambda: nn.packed_attention(few, x, x, offsets), "32 bits"),
            (lambda: nn.packed_attention(few, few, few, offsets, window=3), "32 bits"),
            (lambda: nn.packed_attention(wide, wide, wide, offsets, window=3), "32 bits")]:
        with pytest.raises(RuntimeError, match=match):
            call()
