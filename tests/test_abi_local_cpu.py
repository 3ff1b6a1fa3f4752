"""The entry points of the rotation, the gated feed-forward block and attention
inside a window without a GPU: bad descriptors and operands are refused with a
status and a message, and the ctypes callers refuse what the kernels would read
or write past before the library is called."""
import ctypes

import pytest
import torch

from riemannengine_amd import abi

F32, BF16 = torch.float32, torch.bfloat16
SOME = ctypes.c_void_p(4096)  # an address no call here reads


def rotary(**kw):
    d = dict(n=4, positions=4096, position_row=1, frequencies=4096, position_type=0, axes=1,
             sections=(ctypes.c_int32 * 8)(4), dim=8, interleaved=0, norm=0, dtype=abi.F32, eps=1e-6)
    return abi.RhipRotary(**{**d, **kw})


def heads(**kw):
    return abi.RhipRotaryHeads(**{**dict(x=4096, x_row=8, x_head=8, grad_y=4096, grad_y_row=8,
                                         grad_y_head=8, y=4096, heads=1), **kw})


def refused(status, match):
    assert status != 0
    assert match in abi.lib().rhip_last_error().decode(), abi.lib().rhip_last_error().decode()


@pytest.mark.parametrize("kw,match", [
    (dict(dtype=7), "dtype"), (dict(n=-1), "row count"), (dict(n=2 ** 31), "too many rows"),
    (dict(dim=0), "width"), (dict(dim=257), "256"), (dict(axes=0), "axes"), (dict(axes=9), "axes"),
    (dict(sections=(ctypes.c_int32 * 8)(5)), "sections"),
    (dict(sections=(ctypes.c_int32 * 8)(0)), "sections"),
    (dict(sections=(ctypes.c_int32 * 8)(-1)), "sections"), (dict(position_type=3), "position_type"),
    (dict(norm=1, eps=0.0), "eps"), (dict(norm=1, eps=1e-60), "eps"), (dict(positions=None), "positions"),
    (dict(frequencies=None), "frequencies"),
])
def test_rotary_descriptors(kw, match):
    L, r, h = abi.lib(), rotary(**kw), heads()
    refused(L.rhip_rotary_forward(ctypes.byref(r), ctypes.byref(h), None, None), match)
    refused(L.rhip_rotary_backward(ctypes.byref(r), ctypes.byref(h), None, SOME, 1 << 30, None),
            match)


def test_rotary_operands():
    L, r = abi.lib(), rotary()
    normed = rotary(norm=1)
    for d, q, k, backward, match in [
            (r, None, None, False, "first tensor"), (r, heads(x=None), None, False, "operands"),
            (r, heads(y=None), None, False, "operands"), (r, heads(heads=0), None, False, "head"),
            (r, heads(heads=2 ** 21), None, False, "2^20"),
            (r, heads(), heads(x=None), False, "operands"),
            (r, heads(grad_y=None, grad_x=4096), None, True, "operands"),
            (normed, heads(x=None, grad_x=4096), None, True, "operands")]:
        q, k = (None if t is None else ctypes.byref(t) for t in (q, k))
        if backward:
            refused(L.rhip_rotary_backward(ctypes.byref(d), q, k, SOME, 1 << 30, None), match)
        else:
            refused(L.rhip_rotary_forward(ctypes.byref(d), q, k, None), match)
    h = heads(grad_weight=4096)
    refused(L.rhip_rotary_backward(ctypes.byref(normed), ctypes.byref(h), None, None, 0, None),
            "workspace")
    refused(L.rhip_rotary_backward(ctypes.byref(normed), ctypes.byref(h), None, SOME, 64, None),
            "workspace too small")
    assert abi._sizeq(L.rhip_rotary_workspace_bytes, ctypes.byref(normed)) > 8 * 2 * 4
    empty = rotary(n=0, positions=None, frequencies=None)
    assert L.rhip_rotary_forward(ctypes.byref(empty), ctypes.byref(heads()), None, None) == 0


def gated(**kw):
    d = dict(n=100, x=4096, gate=4096, up=4096, down=4096, grad_y=4096, x_row=16, gate_row=16,
             up_row=16, down_row=24, grad_y_row=8, channels=16, hidden=24, outputs=8, activation=0,
             dtype=abi.F32)
    return abi.RhipGated(**{**d, **kw})


@pytest.mark.parametrize("kw,match", [
    (dict(dtype=2), "dtype"), (dict(n=-1), "sizes"), (dict(channels=0), "sizes"),
    (dict(hidden=0), "sizes"), (dict(outputs=0), "sizes"), (dict(hidden=2 ** 20 + 1), "2^20"),
    (dict(n=2 ** 31), "2^31"), (dict(activation=2), "activation"), (dict(x=None), "required"),
    (dict(gate=None), "required"), (dict(up=None), "required"), (dict(down=None), "required"),
])
def test_gated_descriptors(kw, match):
    L, d = abi.lib(), gated(**kw)
    out = ctypes.c_size_t()
    refused(L.rhip_gated_saved_bytes(ctypes.byref(d), ctypes.byref(out)), match)
    for which in range(3):
        refused(L.rhip_gated_workspace_bytes(ctypes.byref(d), which, ctypes.byref(out)), match)
    refused(L.rhip_gated_forward(ctypes.byref(d), SOME, None, 0, SOME, 1 << 30, None), match)
    refused(L.rhip_gated_backward(ctypes.byref(d), SOME, 1 << 30, SOME, SOME, SOME, SOME, SOME,
                                  1 << 30, None), match)


def test_gated_operands():
    L, d = abi.lib(), gated()
    by = ctypes.byref(d)
    refused(L.rhip_gated_workspace_bytes(by, 3, ctypes.byref(ctypes.c_size_t())), "RHIP_GATED_")
    refused(L.rhip_gated_forward(by, None, None, 0, SOME, 1 << 30, None), "y is required")
    refused(L.rhip_gated_forward(by, SOME, None, 0, None, 0, None), "workspace")
    refused(L.rhip_gated_forward(by, SOME, None, 0, SOME, 64, None), "workspace too small")
    refused(L.rhip_gated_forward(by, SOME, SOME, 64, SOME, 1 << 30, None), "workspace too small")
    refused(L.rhip_gated_forward(by, SOME, ctypes.c_void_p(4100), 1 << 30, SOME, 1 << 30, None),
            "aligned")
    refused(L.rhip_gated_backward(by, SOME, 1 << 30, SOME, SOME, None, SOME, SOME, 1 << 30, None),
            "go together")
    refused(L.rhip_gated_backward(by, None, 0, SOME, SOME, SOME, SOME, SOME, 1 << 30, None),
            "saved")
    other = gated(grad_y=None)
    refused(L.rhip_gated_backward(ctypes.byref(other), SOME, 1 << 30, SOME, SOME, SOME, SOME, SOME,
                                  1 << 30, None), "grad_y")
    assert L.rhip_gated_backward(by, None, 0, None, None, None, None, None, 0, None) == 0
    # h, g and u of 100 rows of 24, fp32
    assert abi._sizeq(L.rhip_gated_saved_bytes, by) >= 3 * 100 * 24 * 4


def test_gated_workspace_holds_what_is_laid_out_anew():
    """Aligned matrices stay where they are; odd widths, unaligned starts and row
    strides between chunks go to the workspace."""
    L = abi.lib()

    def size(which=abi.GATED_INFERENCE, **kw):
        return abi._sizeq(L.rhip_gated_workspace_bytes, ctypes.byref(gated(**kw)), which)

    n = 300
    plain = size(n=n)
    assert size(n=n, x=4100) >= plain + n * 16 * 4
    assert size(n=n, x_row=18) >= plain + n * 16 * 4
    assert size(n=n, gate_row=20) >= plain + 2 * 24 * 16 * 4  # unlike strides: both
    for few in (64, 100, 256):  # read as they lie
        assert size(n=few, x=4100, gate_row=20) == size(n=few) < plain
    assert size(n=n, channels=15, x_row=16, gate_row=16, up_row=16) >= plain + n * 16 * 4


def test_window_descriptors():
    L = abi.lib()
    d = abi.RhipAttn(n_q=8, n_k=8, q_offsets=4096, k_offsets=4096, n_seq=1, heads=1, kv_heads=1,
                     dim=8, dtype=abi.F32, scale=1.0)
    out = ctypes.c_size_t()
    for w, match in [(None, "window is null"), (abi.RhipAttnWindow(0, 0), "at least one key"),
                     (abi.RhipAttnWindow(-2, 0), "at least one key"),
                     (abi.RhipAttnWindow(3, -1), "sinks")]:
        by = None if w is None else ctypes.byref(w)
        refused(L.rhip_attn_window_workspace_bytes(ctypes.byref(d), by, 0, ctypes.byref(out)),
                match)
        refused(L.rhip_attn_window_forward(ctypes.byref(d), by, *[SOME] * 7, 1 << 30, None), match)
        refused(L.rhip_attn_window_backward(ctypes.byref(d), by, SOME, 8, 8, *[SOME] * 10, 1 << 30,
                                            None), match)
    # sinks that are most of every sequence have no launch of their own
    args = (F32, 10 ** 7, 10 ** 7, 10 ** 4, 4, 4, 64, True)
    assert abi.attn_plan("apart", *args, 16, 10 ** 9) == (0, 0)
    assert abi.attn_plan("apart", *args, 16, 40)[0] == 1


@pytest.fixture
def no_library(monkeypatch):
    monkeypatch.setattr(abi, "_require_cuda", lambda t, name: None)
    monkeypatch.setattr(abi, "lib", lambda: pytest.fail("the library was called"))


def elsewhere(t):
    return torch.empty(t.shape, dtype=t.dtype, device="meta")


ROTARY = dict(q=torch.zeros(6, 2, 16), k=torch.zeros(6, 1, 16),
              positions=torch.zeros(6, 2, dtype=torch.int32),
              frequencies=torch.zeros(8, dtype=torch.float64), sections=[5, 3], norm=True,
              weights=(torch.zeros(16), None))


@pytest.mark.parametrize("name,value,match", [
    ("q", torch.zeros(6, 32), "q and k"), ("k", torch.zeros(5, 1, 16), "q and k"),
    ("k", torch.zeros(6, 1, 8), "q and k"), ("k", torch.zeros(6, 1, 16, dtype=BF16), "q and k"),
    ("k", elsewhere(ROTARY["k"]), "q and k"), ("positions", torch.zeros(5, 2), "positions"),
    ("positions", torch.zeros(6, 2, dtype=torch.float64), "positions"),
    ("positions", torch.zeros(2, 6).t(), "positions"),
    ("positions", elsewhere(ROTARY["positions"]), "positions"),
    ("frequencies", torch.zeros(8), "frequencies"),
    ("frequencies", torch.zeros(7, dtype=torch.float64), "frequencies"),
    ("frequencies", elsewhere(ROTARY["frequencies"]), "frequencies"), ("sections", [1] * 9, "axes"),
    ("weights", (torch.zeros(15), None), "weight"),
    ("weights", (torch.zeros(16, dtype=BF16), None), "weight"),
    ("weights", (elsewhere(torch.zeros(16)), None), "weight"), ("norm", False, "normed"),
])
def test_rotary_callers(no_library, name, value, match):
    args = {**ROTARY, name: value}
    with pytest.raises(RuntimeError, match=match):
        abi.rotary_forward(**args)
    with pytest.raises(RuntimeError, match=match):
        abi.rotary_backward((args["q"], args["k"]), **args)


def test_rotary_gradients(no_library):
    for bad in (torch.zeros(6, 2, 8), elsewhere(ROTARY["q"])):
        with pytest.raises(RuntimeError, match="gradient"):
            abi.rotary_backward((bad, ROTARY["k"]), **ROTARY)


GATED = dict(x=torch.zeros(6, 16), gate=torch.zeros(24, 16), up=torch.zeros(24, 16),
             down=torch.zeros(8, 24), activation="silu")


@pytest.mark.parametrize("name,value,match", [
    ("x", torch.zeros(6, 15), "channels"), ("gate", torch.zeros(24, 15), "channels"),
    ("up", torch.zeros(23, 16), "channels"), ("down", torch.zeros(8, 23), "channels"),
    ("x", torch.zeros(96), "channels"), ("gate", torch.zeros(24, 16, dtype=BF16), "gate"),
    ("up", elsewhere(GATED["up"]), "up"), ("down", elsewhere(GATED["down"]), "down"),
    ("activation", "relu", "silu"),
])
def test_gated_callers(no_library, name, value, match):
    args = {**GATED, name: value}
    with pytest.raises(RuntimeError, match=match):
        abi.gated_forward(**args)
    with pytest.raises(RuntimeError, match=match):
        abi.gated_backward(torch.zeros(6, 8), args["x"], args["gate"], args["up"], args["down"],
                           torch.zeros(10, dtype=torch.uint8), args["activation"])


@pytest.mark.parametrize("grad_y,saved,match", [
    (torch.zeros(5, 8), torch.zeros(10, dtype=torch.uint8), "grad_y"),
    (torch.zeros(6, 8), torch.zeros(10), "saved"),
    (torch.zeros(6, 8), torch.zeros(10, dtype=torch.uint8, device="meta"), "saved"),
    (torch.zeros(6, 8), torch.zeros(20, dtype=torch.uint8)[::2], "saved"),
])
def test_gated_gradients(no_library, grad_y, saved, match):
    with pytest.raises(RuntimeError, match=match):
        abi.gated_backward(grad_y, GATED["x"], GATED["gate"], GATED["up"], GATED["down"], saved)


def test_sinks_without_a_window(no_library):
    q = torch.zeros(10, 4, 16)
    offs = torch.tensor([0, 10], dtype=torch.int32)
    with pytest.raises(RuntimeError, match="beside a window"):
        abi.attn_forward(q, q, q, offs, offs, sinks=2)


@pytest.mark.parametrize("window,sinks", [(2 ** 32 + 5, 0), (5, 2 ** 32), (2 ** 31, 1)])
def test_windows_past_32_bits(window, sinks):
    with pytest.raises(RuntimeError, match="32 bits"):
        abi.attn_plan("forward", F32, 10, 10, 1, 4, 4, 16, False, window, sinks)


def test_sections_past_32_bits(no_library):
    with pytest.raises(RuntimeError, match="32 bits"):
        abi.rotary_forward(**{**ROTARY, "sections": [5, 2 ** 32 + 3]})
