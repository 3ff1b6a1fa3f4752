"""The ctypes callers of the transformer operators refuse every operand whose
memory the kernels would read or write past, before the library is called.
Host tensors stand in for device ones (the device check is switched off and
the library is never reached), meta tensors for those of another device."""
import pytest
import torch

from riemannengine_amd import abi

F32, BF16 = torch.float32, torch.bfloat16


@pytest.fixture
def no_library(monkeypatch):
    monkeypatch.setattr(abi, "_require_cuda", lambda t, name: None)
    monkeypatch.setattr(abi, "lib", lambda: pytest.fail("the library was called"))


def elsewhere(t):
    return torch.empty(t.shape, dtype=t.dtype, device="meta")


def attention_operands(dtype=BF16):
    q = torch.zeros(10, 4, 16, dtype=dtype)
    k = torch.zeros(12, 2, 16, dtype=dtype)
    offs = torch.tensor([0, 10], dtype=torch.int32)
    return dict(q=q, k=k, v=k, q_offsets=offs, k_offsets=offs,
                k_lengths=torch.tensor([9], dtype=torch.int32), rest=torch.zeros_like(q))


@pytest.mark.parametrize("name", ["k", "v", "q_offsets", "k_offsets", "k_lengths", "rest"])
def test_attention_operands_of_another_device(no_library, name):
    args = attention_operands()
    args[name] = elsewhere(args[name])
    with pytest.raises(RuntimeError, match=name):
        abi.attn_forward(**args)


@pytest.mark.parametrize("rest", [torch.zeros(10, 4, 8, dtype=BF16), torch.zeros(10, 4, 16),
                                  torch.zeros(10, 16, 4, dtype=BF16).transpose(1, 2)])
def test_attention_rest(no_library, rest):
    with pytest.raises(RuntimeError, match="rest"):
        abi.attn_forward(**{**attention_operands(), "rest": rest})


@pytest.mark.parametrize("name,value", [
    ("grad_out", torch.zeros(9, 4, 16, dtype=BF16)),
    ("grad_out", torch.zeros(10, 4, 16, dtype=BF16, device="meta")),
    ("out", torch.zeros(10, 2, 16, dtype=BF16)), ("out", torch.zeros(10, 4, 16)),
    ("out", torch.zeros(4, 10, 16, dtype=BF16).transpose(0, 1)),
    ("lse", torch.zeros(4, 9)), ("lse", torch.zeros(4, 10, dtype=BF16)),
    ("lse", torch.zeros(10, 4).t()), ("lse", torch.zeros(4, 10, device="meta")),
    ("rest", torch.zeros(10, 4, 15, dtype=BF16)),
    ("k_lengths", torch.zeros(1, dtype=torch.int32, device="meta")),
])
def test_attention_backward_operands(no_library, name, value):
    args = attention_operands()
    args.update(grad_out=args["q"], out=torch.zeros_like(args["q"]), lse=torch.zeros(4, 10))
    args[name] = value
    with pytest.raises(RuntimeError, match=name):
        abi.attn_backward(**args)


@pytest.mark.parametrize("name,value", [
    ("x", torch.zeros(48)), ("weight", torch.ones(7)), ("weight", torch.ones(8, dtype=BF16)),
    ("weight", torch.ones(16)[::2]), ("bias", torch.ones(8, 1)),
    ("bias", torch.ones(8, device="meta")),
])
def test_layer_norm_operands(no_library, name, value):
    args = dict(x=torch.zeros(6, 8), weight=torch.ones(8), bias=torch.ones(8))
    args[name] = value
    with pytest.raises(RuntimeError, match=name):
        abi.ln_forward(**args)


@pytest.mark.parametrize("name,value", [
    ("grad_y", torch.zeros(5, 8)), ("grad_y", torch.zeros(6, 7)),
    ("grad_y", torch.zeros(6, 8, device="meta")), ("mean", torch.zeros(5)),
    ("mean", torch.zeros(6, dtype=torch.float64)), ("rstd", torch.zeros(6, device="meta")),
    ("rstd", torch.zeros(12)[::2]), ("weight", torch.ones(9)),
])
def test_layer_norm_backward_operands(no_library, name, value):
    args = dict(grad_y=torch.zeros(6, 8), x=torch.zeros(6, 8), mean=torch.zeros(6),
                rstd=torch.zeros(6), weight=torch.ones(8))
    args[name] = value
    with pytest.raises(RuntimeError, match=name):
        abi.ln_backward(**args)


def test_embedding_operands(no_library):
    ids, table = torch.zeros(5, dtype=torch.int64), torch.zeros(3, 8)
    for call, name in [
        (lambda: abi.embed_forward(ids, elsewhere(table)), "weight"),
        (lambda: abi.embed_forward(ids, table[0]), "weight"),
        (lambda: abi.embed_forward(ids.float(), table), "ids"),
        (lambda: abi.embed_backward(torch.zeros(6, 8), ids, 3), "grad_y"),
        (lambda: abi.embed_backward(torch.zeros(5), ids, 3), "grad_y"),
        (lambda: abi.embed_backward(elsewhere(torch.zeros(5, 8)), ids, 3), "grad_y"),
    ]:
        with pytest.raises(RuntimeError, match=name):
            call()


@pytest.mark.parametrize("call,msg", [
    (lambda L: L.rhip_ln_forward(1, 8, 1, 2 ** 30 + 1, None, None, 1e-5, 1, None, None, abi.F32,
                                 None), "2\\^30"),
    (lambda L: L.rhip_ln_forward(1, 8, 1, 8, None, None, 1e-46, 1, None, None, abi.F32, None),
     "eps"),
    (lambda L: L.rhip_ln_backward(1, 8, 1, 8, 1, 2 ** 25, 1, 1, None, None, 1, 1, abi.F32, 1,
                                  2 ** 40, None), "2\\^25"),
    (lambda L: L.rhip_embed_forward(1, 0, 1, 1, 8, 1, 65535 * 256 + 1, 1.0, 1, abi.F32, None),
     "chunks"),
    (lambda L: L.rhip_embed_backward(1, 8, 1, 0, 1, 1, 65535 * 512 + 1, 1.0, 1, abi.BF16, 1,
                                     2 ** 40, None), "chunks"),
])
def test_widths_that_no_launch_takes(call, msg):
    """Refused on the host: no pointer is looked at."""
    import re
    lib = abi.lib()
    assert call(lib) != 0
    assert re.search(msg, lib.rhip_last_error().decode())
