"""The launches of the gated feed-forward block's products, without a GPU: the tests'
sizes reach all of them, and parts of shared tiles add up to the whole."""
import ctypes
import math
import random

import pytest
import torch

from feed_forward_launches import SIZES, reached, shares
from riemannengine_amd import abi

DTYPES = [torch.float32, torch.bfloat16]


def some_sizes(count, seed):
    rng = random.Random(seed)

    def log(lo, hi):
        return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))

    return [(log(1, 16384), log(1, 4096), log(1, 11008), log(1, 4096)) for _ in range(count)]


@pytest.mark.parametrize("dtype", DTYPES)
def test_sizes_reach_every_launch(dtype):
    every = set().union(*(reached(dtype, s) for s in some_sizes(8000, 0)))
    tested = set().union(*(reached(dtype, s) for s in SIZES[dtype]))
    assert not every - tested, sorted(every - tested)


@pytest.mark.parametrize("dtype", DTYPES)
def test_parts_add_up(dtype):
    """Part w has units [units w / parts, units (w + 1) / parts) of the line of all tiles
    of k. Every part has some, none has parts of more than two tiles, and where it has
    parts of two the first is the one that it begins with."""
    for sizes in SIZES[dtype] + some_sizes(60, 1):
        for product in abi.GATED_PRODUCTS:
            launch = abi.gated_plan(product, dtype, *sizes)
            if launch.parts == 0:
                continue
            per, units = launch.k_tiles, launch.tiles * launch.k_tiles
            cuts = [units * w // launch.parts for w in range(launch.parts + 1)]
            assert cuts[0] == 0 and cuts[-1] == units
            for a, b in zip(cuts, cuts[1:]):
                assert a < b
                first, last = a // per, (b - 1) // per
                partial = [t for t in sorted({first, last})
                           if not (a <= t * per and (t + 1) * per <= b)]
                assert last - first <= 1 or not set(range(first + 1, last)) & set(partial)
            if launch.tiles > launch.parts:  # two parts at most share a tile
                assert min(b - a for a, b in zip(cuts, cuts[1:])) >= per
            if shares(launch) == "even":
                assert all(t * per in set(cuts) for t in range(launch.tiles))


def test_no_launches():
    for product in abi.GATED_PRODUCTS:
        rows = abi.gated_plan(product, torch.float32, 0, 24, 40, 16)
        assert (rows.side == 0) == (product not in ("grad_gates", "grad_down"))
        few = abi.gated_plan(product, torch.bfloat16, 64, 24, 40, 16)
        assert (few.side == 0) == (product in ("hidden", "output"))


@pytest.mark.parametrize("kw,product,match", [
    (dict(dtype=2), 0, "dtype"), (dict(n=-1), 0, "sizes"), (dict(hidden=2 ** 20 + 1), 0, "2^20"),
    (dict(), -1, "RHIP_GATED_"), (dict(), 6, "RHIP_GATED_"),
])
def test_refusals(kw, product, match):
    d = abi.RhipGated(**{**dict(n=8, channels=4, hidden=4, outputs=4, dtype=abi.F32), **kw})
    launch = abi.RhipGatedLaunch()
    assert abi.lib().rhip_gated_plan(ctypes.byref(d), product, ctypes.byref(launch)) != 0
    assert match in abi.lib().rhip_last_error().decode()
    good = abi.RhipGated(n=8, channels=4, hidden=4, outputs=4, dtype=abi.F32)
    assert abi.lib().rhip_gated_plan(ctypes.byref(good), 0, None) != 0
    assert "launch is null" in abi.lib().rhip_last_error().decode()


@pytest.mark.parametrize("sizes", [(1000, 4096, 11008, 4096), *SIZES[torch.bfloat16][:6]])
def test_bf16_parts_hold_one_tile_each(sizes):
    """bf16 cuts tiles evenly, so a part never has parts of two."""
    n, channels, hidden, outputs = (s // 8 * 8 for s in sizes)  # nothing is laid out anew
    d = abi.RhipGated(n=n, x=4096, gate=4096, up=4096, down=4096, grad_y=4096, x_row=channels,
                      gate_row=channels, up_row=channels, down_row=hidden, grad_y_row=outputs,
                      channels=channels, hidden=hidden, outputs=outputs, dtype=abi.BF16)
    for which, products, hiddens in ((abi.GATED_FORWARD, ("hidden", "output"), 0),
                                     (abi.GATED_BACKWARD, abi.GATED_PRODUCTS[2:], 2)):
        sums = 0
        for product in products:
            launch = abi.gated_plan(product, torch.bfloat16, n, channels, hidden, outputs)
            both = 2 if product == "hidden" and launch.side == 64 else 1
            sums = max(sums, launch.parts * launch.side ** 2 * both * 4)
        got = abi._sizeq(abi.lib().rhip_gated_workspace_bytes, ctypes.byref(d), which)
        assert sums + hiddens * n * hidden * 2 <= got <= sums + hiddens * n * hidden * 2 + 2048
