"""Operators of a transformer stage over packed sequences, as a program that
trains or runs one calls them: attention over packed sequences (of scenes,
prompts or single tokens against a cache), layer norm, and embedding lookup
with its gradient.

A case is a dict of plain values. `op` names the operator and `mode` the
pass: "forward" (inference), "train" (forward and all gradients) or, for
attention, "token" (one query per sequence over a cache whose regions have
spare room). Lengths are texts, "37,0,129".

`run` takes the operators in their plain form, elementary torch operations
in fp32 rounded once at the end, unless `own` is set: then through the
`riemannengine` API. `exact` has them from their definitions in fp64.
"""
from __future__ import annotations

import math

import torch

own = False

DTYPES = {"f32": torch.float32, "bf16": torch.bfloat16}
DEV = "cuda"


# ------------------------------------------------------------------ cases

def _attention(mode, dtype, q_lens, k_lens, heads, kv_heads, dim, causal, room=0):
    return {"op": "attention", "mode": mode, "dtype": dtype, "q_lens": q_lens, "k_lens": k_lens,
            "heads": heads, "kv_heads": kv_heads, "dim": dim, "causal": causal, "room": room}


def _norm(mode, dtype, rows, channels):
    return {"op": "norm", "mode": mode, "dtype": dtype, "rows": rows, "channels": channels}


def _embedding(mode, dtype, count, vocabulary, channels, skew):
    return {"op": "embedding", "mode": mode, "dtype": dtype, "count": count,
            "vocabulary": vocabulary, "channels": channels, "skew": skew}


def listed():
    scans = "2057,1463,3011,1789"
    prompts = "8192,4097,2047,1001"
    texts = "4096,2500,1024,571"
    fills = ("16384,9001,777,12288,1,4096,6543,2048,15001,300,8191,1025,5000,64,11111,3333,"
             "2500,7777,129,10240,600,4500,1800,13000,950,6000,31,8800,2222,14000,480,3700")
    named = {
        # a few objects of a small scene, one of them empty: latency counts
        "attention_objects_f32": _attention("train", "f32", "37,0,129", "37,0,129", 4, 2, 32,
                                            False),
        # the coarsest stage of an encoder over a batch of scans: 256 channels
        # in 8 heads, every voxel sees its scan
        "attention_scans_bf16": _attention("train", "bf16", scans, scans, 8, 8, 32, False),
        # the same kind of stage trained in full precision, odd head width
        "attention_rooms_f32": _attention("train", "f32", "1501,700,1100", "1501,700,1100", 6, 2,
                                          40, True),
        # a batch of prompts read in before the answers
        "attention_prompts_bf16": _attention("forward", "bf16", prompts, prompts, 32, 8, 128,
                                             True),
        # a training batch of packed texts
        "attention_texts_bf16": _attention("train", "bf16", texts, texts, 16, 4, 128, True),
        # one step of 32 answers over their caches
        "attention_tokens_bf16": _attention("token", "bf16", ",".join(["1"] * 32), fills, 32, 8,
                                            128, True, room=64),
        # one row: the norm of a single new token
        "norm_token_f32": _norm("forward", "f32", 1, 256),
        # voxel features of a batch of rooms
        "norm_voxels_bf16": _norm("train", "bf16", 100003, 96),
        # wide rows, a training batch of texts
        "norm_texts_bf16": _norm("train", "bf16", 16384, 4096),
        # class embeddings of labelled voxels: few rows, each used thousands
        # of times, some voxels without a label
        "embedding_labels_f32": _embedding("train", "f32", 200003, 20, 64, "labels"),
        # a vocabulary over a training batch of texts: frequent and rare words
        "embedding_words_bf16": _embedding("train", "bf16", 32768, 50021, 1024, "words"),
        # the tokens of one step of 32 answers
        "embedding_tokens_bf16": _embedding("forward", "bf16", 32, 50021, 4096, "words"),
    }
    return [{"name": name, **c} for name, c in named.items()]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    # the listed cases' largest: a drawn one stays within both
    most = {"bytes": 6.1e8, "flops": 7.3e11}
    while True:
        case = _draw(rng)
        w = work(case)
        plain = 4.0 * w["bytes"] if case["op"] != "attention" else _scores(case) * 12.0
        if all(w[k] <= most[k] for k in most) and plain <= 4e10:
            return case


def _draw(rng):
    op = rng.choice(["attention", "attention", "attention", "norm", "embedding"])
    dtype = rng.choice(["f32", "bf16", "bf16"])
    if op == "norm":
        return _norm(rng.choice(["forward", "train", "train"]), dtype, _log(rng, 1, 200000),
                     _log(rng, 16, 8192))
    if op == "embedding":
        skew = rng.choice(["labels", "words"])
        vocabulary = _log(rng, 2, 100) if skew == "labels" else _log(rng, 100, 100000)
        return _embedding(rng.choice(["forward", "train", "train"]), dtype, _log(rng, 1, 200000),
                          vocabulary, _log(rng, 16, 4096), skew)
    kv_heads = rng.choice([1, 2, 3, 4, 8])
    heads = kv_heads * rng.choice([1, 1, 2, 4, 8])
    dim = rng.choice([16, 24, 32, 40, 64, 64, 80, 96, 128, 128])
    mode = rng.choice(["forward", "train", "train", "token"])
    if mode == "token":
        n = _log(rng, 1, 64)
        k = [_log(rng, 1, 16384) for _ in range(n)]
        q = [1] * n
    else:
        longest = 8192 if mode == "forward" else 4096
        q = [0 if rng.random() < 0.05 else _log(rng, 1, longest)
             for _ in range(_log(rng, 1, 16))]
        # now and then the keys hold an earlier part too
        k = [v + _log(rng, 1, 1000) for v in q] if rng.random() < 0.2 else q
    return _attention(mode, dtype, ",".join(map(str, q)), ",".join(map(str, k)), heads, kv_heads,
                      dim, mode == "token" or rng.random() < 0.6,
                      room=_log(rng, 1, 256) if mode == "token" else 0)


def _lens(text):
    return [int(v) for v in text.split(",")]


def _visible(lq, lk, causal):
    """Pairs (row, key) of a sequence in which the row sees the key."""
    if not causal:
        return lq * lk
    first = lk - lq + 1  # keys that row 0 sees (may be negative)
    lo = max(0, -first)  # rows before this one see nothing
    rows = lq - max(lo, 0)
    if rows <= 0:
        return 0
    a, b = max(first, 0) if lo == 0 else first + lo, lk
    return (a + b) * rows // 2


def _scores(case):
    return case["heads"] * sum(a * b for a, b in zip(_lens(case["q_lens"]), _lens(case["k_lens"])))


def work(case):
    size = 4 if case["dtype"] == "f32" else 2
    train = case["mode"] == "train"
    if case["op"] == "norm":
        n, c = case["rows"], case["channels"]
        # x, y, and in training dy and dx (x again belongs to no floor)
        bytes_ = n * c * size * (4 if train else 2) + c * 4 * (4 if train else 2)
        return {"bytes": bytes_, "flops": n * c * (20 if train else 8)}
    if case["op"] == "embedding":
        n, v, c = case["count"], case["vocabulary"], case["channels"]
        rows = min(n, v)
        bytes_ = n * 8 + rows * c * size + n * c * size
        if train:
            bytes_ += n * c * size + v * c * size
        return {"bytes": bytes_, "flops": n * c * (3 if train else 1)}
    q, k = _lens(case["q_lens"]), _lens(case["k_lens"])
    h, hk, d = case["heads"], case["kv_heads"], case["dim"]
    pairs = sum(_visible(a, b, case["causal"]) for a, b in zip(q, k)) * h
    one = size * d * (2 * h * sum(q) + 2 * hk * sum(k))
    # training: q, k, v, o, do read or written once, and the three gradients
    bytes_ = one if not train else one * 2
    return {"bytes": bytes_, "flops": pairs * d * (14 if train else 4)}


# ----------------------------------------------------------------- inputs

def prepare(case, seed):
    g = torch.Generator(device=DEV).manual_seed(seed)
    dt = DTYPES[case["dtype"]]
    train = case["mode"] == "train"

    def normal(*shape, scale=1.0, shift=0.0, dtype=dt):
        return (torch.randn(shape, generator=g, device=DEV) * scale + shift).to(dtype)

    state = {"case": case, "train": train}
    if case["op"] == "norm":
        n, c = case["rows"], case["channels"]
        # rows of different scale around a mean, as after a residual sum
        spread = torch.rand((n, 1), generator=g, device=DEV) * 2 + 0.5
        state["x"] = (torch.randn((n, c), generator=g, device=DEV) * spread + 0.3).to(dt)
        state["weight"] = normal(c, scale=0.1, shift=1.0, dtype=torch.float32)
        state["bias"] = normal(c, scale=0.1, dtype=torch.float32)
        leaves = ("x", "weight", "bias")
        out_shape = (n, c)
    elif case["op"] == "embedding":
        n, v, c = case["count"], case["vocabulary"], case["channels"]
        u = torch.rand(n, generator=g, device=DEV, dtype=torch.float64)
        # "words": probability falls as 1 / rank; "labels": a few classes hold
        # most voxels, and one voxel in ten has none (-1)
        p = 1.0 / torch.arange(1, v + 1, device=DEV, dtype=torch.float64)
        cdf = torch.cumsum(p / p.sum(), 0)
        ids = torch.searchsorted(cdf, u).clamp_(max=v - 1)
        ids = torch.randperm(v, generator=g, device=DEV)[ids]
        if case["skew"] == "labels":
            none = torch.rand(n, generator=g, device=DEV) < 0.1
            ids = torch.where(none, torch.full_like(ids, -1), ids)
        state["ids"] = ids
        state["weight"] = normal(v, c, scale=c ** -0.5)
        state["scale"] = math.sqrt(c)
        leaves = ("weight",)
        out_shape = (n, c)
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
        out_shape = (sum(q), h, d)
    if train:
        state["grad"] = normal(*out_shape)
        for name in leaves:
            state[name].requires_grad_()
    return state


# ------------------------------------------------------------------- runs

def run(state):
    if own:
        return _run_own(state)
    with torch.no_grad():
        return {"attention": _plain_attention, "norm": _plain_norm,
                "embedding": _plain_embedding}[state["case"]["op"]](state)


def _run_own(state):
    from riemannengine import nn
    case, op = state["case"], state["case"]["op"]
    if op == "norm":
        leaves = ("x", "weight", "bias")
        call = lambda: nn.layer_norm(state["x"], state["weight"], state["bias"], 1e-5)
    elif op == "embedding":
        leaves = ("weight",)
        call = lambda: nn.embedding(state["ids"], state["weight"], state["scale"])
    else:
        leaves = ("q", "k", "v")
        call = lambda: nn.packed_attention(state["q"], state["k"], state["v"],
                                           state["q_offsets"], state["k_offsets"],
                                           state["k_lengths"], case["causal"])
    if not state["train"]:
        with torch.no_grad():
            return [call()]
    out = call()
    return [out.detach(),
            *torch.autograd.grad(out, [state[name] for name in leaves], state["grad"])]


def _plain_norm(state):
    x = state["x"].float()
    dt = state["x"].dtype
    mean = x.mean(1, keepdim=True)
    centred = x - mean
    rstd = 1.0 / torch.sqrt((centred * centred).mean(1, keepdim=True) + 1e-5)
    hat = centred * rstd
    y = hat * state["weight"] + state["bias"]
    if not state["train"]:
        return [y.to(dt)]
    dy = state["grad"].float()
    g = dy * state["weight"]
    dx = rstd * (g - g.mean(1, keepdim=True) - hat * (g * hat).mean(1, keepdim=True))
    return [y.to(dt), dx.to(dt), (dy * hat).sum(0), dy.sum(0)]


def _plain_embedding(state):
    ids, w = state["ids"], state["weight"]
    v = w.shape[0]
    known = (ids >= 0) & (ids < v)
    rows = torch.where(known, ids, torch.zeros_like(ids))
    y = torch.where(known[:, None], w[rows].float() * state["scale"], 0.0).to(w.dtype)
    if not state["train"]:
        return [y]
    dy = torch.where(known[:, None], state["grad"].float() * state["scale"], 0.0)
    dw = torch.zeros(w.shape, dtype=torch.float32, device=w.device)
    dw.index_add_(0, rows, dy)
    return [y, dw.to(w.dtype)]


def _plain_attention(state):
    case = state["case"]
    h, hk, d = case["heads"], case["kv_heads"], case["dim"]
    group = h // hk
    scale = d ** -0.5
    dt = state["q"].dtype
    out = torch.empty_like(state["q"])
    if state["train"]:
        dq = torch.empty_like(state["q"])
        dk, dv = torch.empty_like(state["k"]), torch.empty_like(state["v"])
    q0 = k0 = 0
    for lq, lk, rows in zip(state["q_lens"], state["k_lens"], state["k_rows"]):
        # [hk, group * lq, d] and [hk, lk, d]
        q = (state["q"][q0:q0 + lq].float().reshape(lq, hk, group, d).permute(1, 2, 0, 3)
             .reshape(hk, group * lq, d))
        k = state["k"][k0:k0 + lk].float().transpose(0, 1).contiguous()
        v = state["v"][k0:k0 + lk].float().transpose(0, 1).contiguous()
        s = torch.bmm(q, k.transpose(1, 2)).mul_(scale).view(hk, group, lq, lk)
        if case["causal"]:
            i = torch.arange(lq, device=DEV)[:, None]
            j = torch.arange(lk, device=DEV)[None, :]
            s.masked_fill_(j > i + (lk - lq), -math.inf)
        if lk:
            top = s.amax(-1, keepdim=True)
            top = torch.where(top == -math.inf, 0.0, top)
            p = s.sub_(top).exp_()
            total = p.sum(-1, keepdim=True)
            p = p.div_(torch.where(total == 0, 1.0, total)).view(hk, group * lq, lk)
        else:
            p = s.view(hk, group * lq, lk)
        o = torch.bmm(p, v)

        def rows_of(t):  # [hk, group * lq, d] -> [lq, h, d]
            return (t.view(hk, group, lq, d).permute(2, 0, 1, 3).reshape(lq, h, d)).to(dt)

        out[q0:q0 + lq] = rows_of(o)
        if state["train"]:
            do = (state["grad"][q0:q0 + lq].float().reshape(lq, hk, group, d).permute(1, 2, 0, 3)
                  .reshape(hk, group * lq, d))
            dv[k0:k0 + lk] = torch.bmm(p.transpose(1, 2), do).transpose(0, 1).to(dt)
            ds = torch.bmm(do, v.transpose(1, 2))
            ds = ds.sub_((do * o).sum(-1, keepdim=True)).mul_(p).mul_(scale)
            dq[q0:q0 + lq] = rows_of(torch.bmm(ds, k))
            dk[k0:k0 + lk] = torch.bmm(ds.transpose(1, 2), q).transpose(0, 1).to(dt)
        q0, k0 = q0 + lq, k0 + rows
    return [out, dq, dk, dv] if state["train"] else [out]


# ------------------------------------------------------------------ exact

def exact(case, seed):
    """The outputs from the definitions in fp64, gradients by autograd over
    them; laid out as `run` returns them."""
    state = prepare(case, seed)
    names = {"norm": ("x", "weight", "bias"), "embedding": ("weight",),
             "attention": ("q", "k", "v")}[case["op"]]
    if case["op"] == "attention":
        return _exact_attention(case, state)
    leaves = [state[n].detach().double().requires_grad_(state["train"]) for n in names]
    if case["op"] == "norm":
        x, w, b = leaves
        var, mean = torch.var_mean(x, 1, unbiased=False, keepdim=True)
        y = (x - mean) * (var + 1e-5) ** -0.5 * w + b
    else:
        # the table with a zero row behind it for what lies outside
        table = torch.cat([leaves[0] * state["scale"], leaves[0].new_zeros(1, case["channels"])])
        ids, v = state["ids"], case["vocabulary"]
        y = table[torch.where((ids < 0) | (ids >= v), v, ids)]
    if not state["train"]:
        return [y]
    grads = torch.autograd.grad(y, leaves, state["grad"].double())
    return [y.detach(), *grads]


def _exact_attention(case, state):
    h, hk, d = case["heads"], case["kv_heads"], case["dim"]
    outs = [torch.zeros(state[n].shape, dtype=torch.float64, device=DEV)
            for n in (("q", "q", "k", "v") if state["train"] else ("q",))]
    q0 = k0 = 0
    for lq, lk, rows in zip(state["q_lens"], state["k_lens"], state["k_rows"]):
        for head in range(h) if lq and lk else ():
            pick = [state["q"].detach()[q0:q0 + lq, head].double(),
                    state["k"].detach()[k0:k0 + lk, head * hk // h].double(),
                    state["v"].detach()[k0:k0 + lk, head * hk // h].double()]
            pick = [t.requires_grad_(state["train"]) for t in pick]
            bias = torch.zeros(lq, lk, dtype=torch.float64, device=DEV)
            if case["causal"]:
                hidden = torch.ones(lq, lk, dtype=torch.bool, device=DEV).triu(lk - lq + 1)
                bias.masked_fill_(hidden, -math.inf)
            seen = lq if not case["causal"] else min(lq, lk)  # the last rows see something
            weights = torch.softmax(
                (pick[0][lq - seen:] @ pick[1].t()) / math.sqrt(d) + bias[lq - seen:], -1)
            y = weights @ pick[2]
            outs[0][q0 + lq - seen:q0 + lq, head] = y.detach()
            if state["train"]:
                dy = state["grad"][q0 + lq - seen:q0 + lq, head].double()
                gq, gk, gv = torch.autograd.grad(y, pick, dy)
                outs[1][q0:q0 + lq, head] = gq
                outs[2][k0:k0 + lk, head * hk // h] += gk
                outs[3][k0:k0 + lk, head * hk // h] += gv
        q0, k0 = q0 + lq, k0 + rows
    return outs
