"""More operators of a transformer stage over packed rows, as a program that
trains or runs one calls them: attention inside a window with a few first keys
that stay visible, the rotation of queries and keys by positions of several
axes (with the heads' norm before it, or alone), and a gated feed-forward
block.

A case is a dict of plain values. `op` names the operator and `mode` the
pass: "forward" (inference), "train" (forward and all gradients) or, for
attention, "token" (one query per sequence over a cache whose regions have
spare room). Lengths are texts, "37,0,129".

`run` takes the operators in their plain form, elementary torch operations
in fp32 rounded once at the end (angles in fp64), unless `own` is set: then
through the `riemannengine` API. `exact` has them from their definitions in
fp64.
"""
from __future__ import annotations

import math

import torch

own = False

DTYPES = {"f32": torch.float32, "bf16": torch.bfloat16}
DEV = "cuda"


# ------------------------------------------------------------------ cases

def _window(mode, dtype, q_lens, k_lens, heads, kv_heads, dim, causal, window, sinks, room=0):
    return {"op": "window", "mode": mode, "dtype": dtype, "q_lens": q_lens, "k_lens": k_lens,
            "heads": heads, "kv_heads": kv_heads, "dim": dim, "causal": causal,
            "window": window, "sinks": sinks, "room": room}


def _rotate(mode, dtype, rows, heads, kv_heads, dim, sections, norm, interleaved, reach):
    """kv_heads 0: one tensor, the rotation alone. reach: positions lie below it."""
    return {"op": "rotate", "mode": mode, "dtype": dtype, "rows": rows, "heads": heads,
            "kv_heads": kv_heads, "dim": dim, "sections": sections, "norm": norm,
            "interleaved": interleaved, "reach": reach}


def _gated(mode, dtype, rows, channels, hidden, activation):
    return {"op": "gated", "mode": mode, "dtype": dtype, "rows": rows, "channels": channels,
            "hidden": hidden, "activation": activation}


def listed():
    scans = "2057,1463,3011,1789"
    texts = "4096,2500,1024,571"
    prompts = "16384,8192,4097,1001"
    rooms = "1501,700,0,1100"
    fills = ("16384,9001,777,12288,1,4096,6543,2048,15001,300,8191,1025,5000,64,11111,3333,"
             "2500,7777,129,10240,600,4500,1800,13000,950,6000,31,8800,2222,14000,480,3700")
    named = {
        # voxels of a batch of scans in the order of a curve through space:
        # each sees those near it on the curve, on both sides
        "window_scans_bf16": _window("train", "bf16", scans, scans, 8, 8, 32, False, 256, 0),
        # the same in full precision: rooms, one of them empty, odd head width
        "window_rooms_f32": _window("train", "f32", rooms, rooms, 6, 2, 40, False, 100, 3),
        # a training batch of packed texts
        "window_texts_bf16": _window("train", "bf16", texts, texts, 16, 4, 128, True, 1024, 4),
        # a batch of long prompts read in before the answers
        "window_prompts_bf16": _window("forward", "bf16", prompts, prompts, 32, 8, 128, True,
                                       2048, 4),
        # one step of 32 answers over their caches
        "window_tokens_bf16": _window("token", "bf16", ",".join(["1"] * 32), fills, 32, 8, 128,
                                      True, 1024, 4, room=64),
        # voxel features of a batch of rooms turned by their coordinates
        "rotate_voxels_bf16": _rotate("train", "bf16", 100003, 8, 0, 32, "6,5,5", False, False,
                                      4096),
        # queries and keys of a training batch of texts
        "norm_rotate_texts_bf16": _rotate("train", "bf16", 16384, 32, 8, 128, "64", True, False,
                                          131072),
        # queries and keys of one step of 32 answers
        "norm_rotate_tokens_bf16": _rotate("forward", "bf16", 32, 32, 8, 128, "64", True, False,
                                           131072),
        # one new token
        "gated_token_bf16": _gated("forward", "bf16", 1, 1024, 2816, "silu"),
        # one step of 32 answers
        "gated_tokens_bf16": _gated("forward", "bf16", 32, 4096, 11008, "silu"),
        # a training batch of texts
        "gated_texts_bf16": _gated("train", "bf16", 8192, 2048, 5504, "silu"),
        # voxel features of a batch of scans in full precision, odd hidden width
        "gated_scans_f32": _gated("train", "f32", 8320, 256, 683, "gelu"),
    }
    return [{"name": name, **c} for name, c in named.items()]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    # the listed cases' largest: a drawn one stays within both
    most = {"bytes": 6.7e8, "flops": 1.6e12}
    while True:
        case = _draw(rng)
        w = work(case)
        if any(w[k] > most[k] for k in most):
            continue
        # fp32 scores of the plain form, and its row blocks
        if case["op"] == "window" and (w["flops"] > 3.5e11 or case["heads"] * sum(
                a * min(b, 2 * case["window"] + 1024)
                for a, b in zip(_lens(case["q_lens"]), _lens(case["k_lens"]))) > 4e9):
            continue
        return case


def _draw(rng):
    op = rng.choice(["window", "window", "rotate", "gated", "gated"])
    dtype = rng.choice(["f32", "bf16", "bf16"])
    if op == "gated":
        mode = rng.choice(["forward", "train"])
        return _gated(mode, dtype, _log(rng, 1, 16384), _log(rng, 16, 4096),
                      _log(rng, 16, 11008), rng.choice(["silu", "silu", "gelu"]))
    kv_heads = rng.choice([1, 2, 3, 4, 8])
    heads = kv_heads * rng.choice([1, 1, 2, 4, 8])
    dim = rng.choice([16, 24, 32, 40, 64, 64, 80, 96, 128, 128])
    if op == "rotate":
        alone = rng.random() < 0.3
        axes = rng.choice([1, 1, 2, 3, 3, 4])
        pairs = dim // 2 if rng.random() < 0.7 else max(axes, dim // 4)
        cuts = sorted(rng.sample(range(1, pairs), axes - 1))
        sections = [b - a for a, b in zip([0] + cuts, cuts + [pairs])]
        return _rotate(rng.choice(["forward", "train", "train"]), dtype, _log(rng, 1, 100000),
                       heads, 0 if alone else kv_heads, dim, ",".join(map(str, sections)),
                       not alone and rng.random() < 0.8, rng.random() < 0.3,
                       _log(rng, 64, 1000000))
    mode = rng.choice(["forward", "train", "train", "token"])
    if mode == "token":
        n = _log(rng, 1, 64)
        k = [_log(rng, 1, 16384) for _ in range(n)]
        q = [1] * n
    else:
        longest = 16384 if mode == "forward" else 4096
        q = [0 if rng.random() < 0.05 else _log(rng, 1, longest)
             for _ in range(_log(rng, 1, 16))]
        # now and then the keys hold an earlier part too, or a part is gone
        k = q
        if rng.random() < 0.2:
            k = [v + _log(rng, 1, 1000) for v in q]
        elif rng.random() < 0.1:
            k = [v // 2 for v in q]
    return _window(mode, dtype, ",".join(map(str, q)), ",".join(map(str, k)), heads, kv_heads,
                   dim, mode == "token" or rng.random() < 0.6, _log(rng, 1, 4096),
                   rng.choice([0, 0, 1, 4, 16, 100]),
                   room=_log(rng, 1, 256) if mode == "token" else 0)


def _lens(text):
    return [int(v) for v in text.split(",")]


def _visible(lq, lk, causal, window, sinks):
    """Pairs (row, key) of a sequence in which the row sees the key."""
    p = torch.arange(lq, dtype=torch.int64) + (lk - lq)
    high = torch.clamp(p + (1 if causal else window), 0, lk)
    low = torch.minimum(torch.clamp(p - window + 1, 0, lk), high)
    first = torch.clamp(p + 1, 0, min(sinks, lk)) if causal else torch.full_like(p, min(sinks, lk))
    return int((high - low + torch.clamp(torch.minimum(first, low), min=0)
                + torch.clamp(first - high, min=0)).sum())


def work(case):
    size = 4 if case["dtype"] == "f32" else 2
    train = case["mode"] == "train"
    if case["op"] == "gated":
        n, c, h = case["rows"], case["channels"], case["hidden"]
        one = 3 * c * h * size + 2 * n * c * size
        return {"bytes": 2 * one if train else one, "flops": n * c * h * (18 if train else 6)}
    if case["op"] == "rotate":
        values = case["rows"] * (case["heads"] + case["kv_heads"]) * case["dim"]
        angles = case["rows"] * len(_lens(case["sections"])) * 4
        # x and y, and in training dy and dx
        return {"bytes": values * size * (4 if train else 2) + angles,
                "flops": values * (20 if train else 8)}
    q, k = _lens(case["q_lens"]), _lens(case["k_lens"])
    h, hk, d = case["heads"], case["kv_heads"], case["dim"]
    pairs = h * sum(_visible(a, b, case["causal"], case["window"], case["sinks"])
                    for a, b in zip(q, k))
    # keys that some row sees
    used = [min(b, a + case["window"] * (1 if case["causal"] else 2) + case["sinks"]) if a else 0
            for a, b in zip(q, k)]
    one = size * d * (2 * h * sum(q) + 2 * hk * sum(used))
    return {"bytes": one * 2 if train else one, "flops": pairs * d * (14 if train else 4)}


# ----------------------------------------------------------------- inputs

def prepare(case, seed):
    g = torch.Generator(device=DEV).manual_seed(seed)
    dt = DTYPES[case["dtype"]]
    train = case["mode"] == "train"

    def normal(*shape, scale=1.0, shift=0.0, dtype=dt):
        return (torch.randn(shape, generator=g, device=DEV) * scale + shift).to(dtype)

    state = {"case": case, "train": train}
    if case["op"] == "gated":
        n, c, h = case["rows"], case["channels"], case["hidden"]
        state["x"] = normal(n, c)
        state["gate"] = normal(h, c, scale=c ** -0.5)
        state["up"] = normal(h, c, scale=c ** -0.5)
        state["down"] = normal(c, h, scale=h ** -0.5)
        leaves = ("x", "gate", "up", "down")
        outputs = [(n, c)]
    elif case["op"] == "rotate":
        n, h, hk, d = case["rows"], case["heads"], case["kv_heads"], case["dim"]
        state["sections"] = _lens(case["sections"])
        axes = len(state["sections"])
        # coordinates with the batch in front, as a sparse tensor has them
        coords = torch.randint(0, case["reach"], (n, axes + 1), generator=g, device=DEV,
                               dtype=torch.int32)
        state["positions"] = coords[:, 1:]
        # each axis has a ladder of its own
        state["frequencies"] = torch.cat([
            10000.0 ** (-torch.arange(s, dtype=torch.float64, device=DEV) / s)
            for s in state["sections"]])
        # the projection's rows: queries, keys (and values) side by side
        rows = normal(n, h + 2 * hk, d)
        state["q"] = rows[:, :h]
        leaves, outputs = ("q",), [(n, h, d)]
        if hk:
            state["k"] = rows[:, h:h + hk]
            leaves, outputs = ("q", "k"), outputs + [(n, hk, d)]
        state["wq"] = state["wk"] = None
        if case["norm"]:
            state["wq"] = normal(d, scale=0.1, shift=1.0, dtype=torch.float32)
            state["wk"] = normal(d, scale=0.1, shift=1.0, dtype=torch.float32)
            leaves += ("wq", "wk")
    else:
        q, k = _lens(case["q_lens"]), _lens(case["k_lens"])
        h, hk, d = case["heads"], case["kv_heads"], case["dim"]
        state["q_lens"], state["k_lens"] = q, k
        rows = [v + case["room"] for v in k]
        state["k_rows"] = rows
        state["q"] = normal(sum(q), h, d)
        state["k"] = normal(sum(rows), hk, d)
        state["v"] = normal(sum(rows), hk, d)

        def offsets(lens):
            return torch.tensor([0] + lens, dtype=torch.int64).cumsum(0).int().to(DEV)

        state["q_offsets"] = offsets(q)
        state["k_offsets"] = state["q_offsets"] if rows == q else offsets(rows)
        state["k_lengths"] = (torch.tensor(k, dtype=torch.int32, device=DEV) if case["room"]
                              else None)
        leaves = ("q", "k", "v")
        outputs = [(sum(q), h, d)]
    if train:
        state["grads"] = [normal(*shape) for shape in outputs]
        for name in leaves:
            state[name] = state[name].detach().requires_grad_()
    state["leaves"] = leaves
    return state


# ------------------------------------------------------------------- runs

def run(state):
    if own:
        return _run_own(state)
    with torch.no_grad():
        return {"window": _plain_window, "rotate": _plain_rotate,
                "gated": _plain_gated}[state["case"]["op"]](state)


def _run_own(state):
    from riemannengine import nn
    case, op = state["case"], state["case"]["op"]

    def call():
        if op == "gated":
            return [nn.gated_feed_forward(state["x"], state["gate"], state["up"], state["down"],
                                          case["activation"])]
        if op == "window":
            return [nn.packed_attention(state["q"], state["k"], state["v"], state["q_offsets"],
                                        state["k_offsets"], state["k_lengths"], case["causal"],
                                        window=case["window"], sinks=case["sinks"])]
        if "k" not in state:
            return [nn.rotate_heads(state["q"], state["positions"], state["frequencies"],
                                    state["sections"], case["interleaved"])]
        if not case["norm"]:
            return [nn.rotate_heads(state[name], state["positions"], state["frequencies"],
                                    state["sections"], case["interleaved"])
                    for name in ("q", "k")]
        return list(nn.norm_rotate_heads(state["q"], state["k"], state["positions"],
                                         state["frequencies"], state["sections"], state["wq"],
                                         state["wk"], 1e-6, case["interleaved"]))

    if not state["train"]:
        with torch.no_grad():
            return call()
    outs = call()
    return [*(out.detach() for out in outs),
            *torch.autograd.grad(outs, [state[name] for name in state["leaves"]],
                                 state["grads"])]


def _activation(g, kind):
    """The activation and its derivative."""
    if kind == "silu":
        s = 1.0 / (1.0 + torch.exp(-g))
        return g * s, s * (1.0 + g * (1.0 - s))
    half = 0.5 * torch.erfc(g * -math.sqrt(0.5))
    return g * half, half + g * torch.exp(-0.5 * g * g) * (1.0 / math.sqrt(2.0 * math.pi))


def _plain_gated(state):
    case, dt = state["case"], state["x"].dtype
    x, wg, wu, wd = (state[n].float() for n in ("x", "gate", "up", "down"))
    g, u = x @ wg.t(), x @ wu.t()
    a, da = _activation(g, case["activation"])
    h = a * u
    y = (h @ wd.t()).to(dt)
    if not state["train"]:
        return [y]
    dy = state["grads"][0].float()
    dh = dy @ wd
    dwd = dy.t() @ h
    dg, du = dh * u * da, dh * a
    dx = dg @ wg + du @ wu
    return [y, dx.to(dt), (dg.t() @ x).to(dt), (du.t() @ x).to(dt), dwd.to(dt)]


def _turns(state):
    """Cosine and sine of every row's pairs, fp32 of fp64 angles."""
    axis = torch.repeat_interleave(torch.arange(len(state["sections"]), device=DEV),
                                   torch.tensor(state["sections"], device=DEV))
    angle = state["positions"].double()[:, axis] * state["frequencies"]
    return torch.cos(angle).float()[:, None], torch.sin(angle).float()[:, None]


def _turned(x, cos, sin, interleaved):
    pairs = cos.shape[-1]
    y = x.clone()
    if interleaved:
        a, b = x[..., 0:2 * pairs:2], x[..., 1:2 * pairs:2]
        y[..., 0:2 * pairs:2], y[..., 1:2 * pairs:2] = a * cos - b * sin, a * sin + b * cos
    else:
        a, b = x[..., :pairs], x[..., pairs:2 * pairs]
        y[..., :pairs], y[..., pairs:2 * pairs] = a * cos - b * sin, a * sin + b * cos
    return y


def _plain_rotate(state):
    case = state["case"]
    cos, sin = _turns(state)
    outs, grads, weight_grads = [], [], []
    for i, name in enumerate(n for n in ("q", "k") if n in state):
        x, dt = state[name].float(), state[name].dtype
        if case["norm"]:
            w = state["w" + name]
            r = 1.0 / torch.sqrt((x * x).mean(-1, keepdim=True) + 1e-6)
            hat = x * r
            outs.append(_turned(hat * w, cos, sin, case["interleaved"]).to(dt))
        else:
            outs.append(_turned(x, cos, sin, case["interleaved"]).to(dt))
        if state["train"]:
            d = _turned(state["grads"][i].float(), cos, -sin, case["interleaved"])
            if case["norm"]:
                weight_grads.append((d * hat).sum((0, 1)))
                d = d * w
                d = r * (d - hat * (d * hat).mean(-1, keepdim=True))
            grads.append(d.to(dt))
    return outs + grads + weight_grads


def _plain_window(state):
    case = state["case"]
    h, hk, d = case["heads"], case["kv_heads"], case["dim"]
    group, window = h // hk, case["window"]
    scale = d ** -0.5
    dt = state["q"].dtype
    out = torch.empty_like(state["q"])
    if state["train"]:
        dq = torch.empty_like(state["q"])
        dk, dv = (torch.zeros(state[n].shape, device=DEV) for n in ("k", "v"))
    q0 = k0 = 0
    for lq, lk, rows in zip(state["q_lens"], state["k_lens"], state["k_rows"]):
        block = max(256, min(window, 1024))
        for r0 in range(0, lq, block):
            r1 = min(r0 + block, lq)
            n = r1 - r0
            shift = lk - lq
            # the keys that the block's rows may see: sinks, then the window
            low = min(max(0, r0 + shift - window + 1), lk)
            high = min(max(low, r1 + shift if case["causal"] else r1 + shift + window - 1), lk)
            first = min(case["sinks"], low)
            keys = torch.cat([torch.arange(first, device=DEV),
                              torch.arange(low, max(high, min(case["sinks"], lk)), device=DEV)])
            # [hk, n * group, d] and [hk, keys, d]
            q = (state["q"][q0 + r0:q0 + r1].float().reshape(n, hk, group, d).permute(1, 2, 0, 3)
                 .reshape(hk, group * n, d))
            k = state["k"][k0 + keys].float().transpose(0, 1).contiguous()
            v = state["v"][k0 + keys].float().transpose(0, 1).contiguous()
            s = torch.bmm(q, k.transpose(1, 2).contiguous()).mul_(scale).view(hk, group, n, -1)
            p = torch.arange(r0, r1, device=DEV)[:, None] + shift
            seen = ((p - keys).abs() < window) | (keys < case["sinks"])
            if case["causal"]:
                seen &= keys <= p
            s.masked_fill_(~seen, -math.inf)
            if len(keys):
                top = s.amax(-1, keepdim=True)
                top = torch.where(top == -math.inf, 0.0, top)
                s = s.sub_(top).exp_()
                total = s.sum(-1, keepdim=True)
                s = s.div_(torch.where(total == 0, 1.0, total))
            s = s.view(hk, group * n, -1)
            o = torch.bmm(s, v)

            def rows_of(t):  # [hk, group * n, d] -> [n, h, d]
                return t.view(hk, group, n, d).permute(2, 0, 1, 3).reshape(n, h, d).to(dt)

            out[q0 + r0:q0 + r1] = rows_of(o)
            if state["train"]:
                do = (state["grads"][0][q0 + r0:q0 + r1].float().reshape(n, hk, group, d)
                      .permute(1, 2, 0, 3).reshape(hk, group * n, d))
                dv.index_add_(0, k0 + keys,
                              torch.bmm(s.transpose(1, 2).contiguous(), do).transpose(0, 1))
                ds = torch.bmm(do, v.transpose(1, 2).contiguous())
                ds = ds.sub_((do * o).sum(-1, keepdim=True)).mul_(s).mul_(scale)
                dq[q0 + r0:q0 + r1] = rows_of(torch.bmm(ds, k))
                dk.index_add_(0, k0 + keys,
                              torch.bmm(ds.transpose(1, 2).contiguous(), q).transpose(0, 1))
        q0, k0 = q0 + lq, k0 + rows
    return [out, dq, dk.to(dt), dv.to(dt)] if state["train"] else [out]


# ------------------------------------------------------------------ exact

def exact(case, seed):
    """The outputs from the definitions in fp64, gradients by autograd over
    them; laid out as `run` returns them."""
    state = prepare(case, seed)
    if case["op"] == "window":
        return _exact_window(case, state)
    leaves = [state[n].detach().double().requires_grad_(state["train"]) for n in state["leaves"]]
    if case["op"] == "gated":
        x, wg, wu, wd = leaves
        act = torch.nn.functional.silu if case["activation"] == "silu" else torch.nn.functional.gelu
        outs = [(act(x @ wg.t()) * (x @ wu.t())) @ wd.t()]
    else:
        outs = [_exact_rotate(case, state, leaf, leaves[2 + i] if case["norm"] else None)
                for i, leaf in enumerate(leaves[:1 if not case["kv_heads"] else 2])]
    if not state["train"]:
        return outs
    grads = torch.autograd.grad(outs, leaves, [t.double() for t in state["grads"]])
    return [*(y.detach() for y in outs), *grads]


def _exact_rotate(case, state, x, weight):
    if weight is not None:
        x = x * ((x ** 2).mean(-1, keepdim=True) + 1e-6) ** -0.5 * weight
    # a pair is a complex number, turned by its axis' coordinate
    pairs, at = sum(state["sections"]), 0
    turned = []
    for axis, size in enumerate(state["sections"]):
        angle = torch.outer(state["positions"][:, axis].double(),
                            state["frequencies"][at:at + size])
        if case["interleaved"]:
            z = torch.complex(x[..., 2 * at:2 * (at + size):2],
                              x[..., 2 * at + 1:2 * (at + size):2])
        else:
            z = torch.complex(x[..., at:at + size], x[..., pairs + at:pairs + at + size])
        turned.append(z * torch.polar(torch.ones_like(angle), angle)[:, None])
        at += size
    z = torch.cat(turned, -1)
    if case["interleaved"]:
        front = torch.view_as_real(z).flatten(-2)
    else:
        front = torch.cat([z.real, z.imag], -1)
    return torch.cat([front, x[..., 2 * pairs:]], -1)


def _exact_window(case, state):
    h, hk, d = case["heads"], case["kv_heads"], case["dim"]
    train, window, sinks = state["train"], case["window"], case["sinks"]
    outs = [torch.zeros(state[n].shape, dtype=torch.float64, device=DEV)
            for n in (("q", "q", "k", "v") if train else ("q",))]
    q0 = k0 = 0
    for lq, lk, rows in zip(state["q_lens"], state["k_lens"], state["k_rows"]):
        step = 512
        for r0 in range(0, lq if lk else 0, step):
            i = torch.arange(r0, min(r0 + step, lq), device=DEV)
            at = (i + (lk - lq))[:, None]
            j = torch.arange(lk, device=DEV)
            sees = (j > at - window) & (j < at + window) | (j < sinks)
            if case["causal"]:
                sees = sees & (j <= at)
            j = j[sees.any(0)]  # of the keys, those that a row of these sees
            if not len(j):
                continue
            some = sees.any(1)  # the rows that see something
            i, bias = i[some], torch.zeros(int(some.sum()), len(j), dtype=torch.float64, device=DEV)
            bias.masked_fill_(~sees[some][:, j], -math.inf)
            pick = [state["q"].detach()[q0 + i].double(), state["k"].detach()[k0 + j].double(),
                    state["v"].detach()[k0 + j].double()]
            pick = [t.requires_grad_(train) for t in pick]
            q, k, v = (t.transpose(0, 1) for t in pick)
            k, v = (t.repeat_interleave(h // hk, 0) for t in (k, v))
            weights = torch.softmax(torch.matmul(q, k.transpose(1, 2).contiguous()) / math.sqrt(d)
                                    + bias, -1)
            y = torch.matmul(weights, v).transpose(0, 1)
            outs[0][q0 + i] = y.detach()
            if train:
                gq, gk, gv = torch.autograd.grad(y, pick, state["grads"][0][q0 + i].double())
                outs[1][q0 + i] = gq
                outs[2][k0 + j] += gk
                outs[3][k0 + j] += gv
        q0, k0 = q0 + lq, k0 + rows
    return outs
