"""Attention over packed sequences from its definition in fp64 on the device,
for launches too large for the host, with the bounds of attention_reference
(u, e and the formulas of each result's error are stated there)."""
import math

import torch

from attention_reference import U


def attention(q, k, v, q_off, k_off, k_len=None, causal=False, grad=None):
    """Dict name -> (value, bound), fp64 on the device, of out and, with grad,
    dq, dk, dv."""
    u = U[q.dtype]
    h, d = q.shape[1:]
    group = h // k.shape[1]
    scale = d ** -0.5
    like = {"out": q, "dq": q, "dk": k, "dv": k}
    names = list(like) if grad is not None else ["out"]
    res = {n: tuple(torch.zeros(like[n].shape, dtype=torch.float64, device=q.device)
                    for _ in range(2)) for n in names}
    q_off, k_off = q_off.tolist(), k_off.tolist()
    k_len = None if k_len is None else k_len.tolist()
    for s in range(len(q_off) - 1):
        qs = slice(q_off[s], q_off[s + 1])
        lq = q_off[s + 1] - q_off[s]
        lk = k_off[s + 1] - k_off[s] if k_len is None else k_len[s]
        # the first rows of a causal sequence may see nothing
        none = max(0, lq - lk) if causal else 0
        if lk == 0 or lq == none:
            continue
        qs = slice(qs.start + none, qs.stop)
        ks = slice(k_off[s], k_off[s] + lk)
        hidden = None
        if causal:
            hidden = torch.ones(lq - none, lk, dtype=torch.bool,
                                device=q.device).triu(lk - lq + none + 1)
        for a in range(h):
            b = a // group
            Q, K, V = (t.double() for t in (q[qs, a], k[ks, b], v[ks, b]))
            S = scale * (Q @ K.t().contiguous())
            A = scale * (Q.abs() @ K.abs().t().contiguous())
            if causal:
                S.masked_fill_(hidden, -math.inf)
                A.masked_fill_(hidden, 0.0)
            e = 2.0 ** -24 * (d + lk + 16) * (1 + A.max())
            P = S.softmax(1)
            O = P @ V
            val, err = res["out"]
            val[qs, a] = O
            err[qs, a] = (2 * u + e) * (P @ V.abs())
            if grad is None:
                continue
            G = grad[qs, a].double()
            Pt, Vt = P.t().contiguous(), V.t().contiguous()
            dS = P * (G @ Vt - (G * O).sum(1, keepdim=True))
            big = (G.abs() * O.abs()).sum(1, keepdim=True)
            dS_err = (u * (dS.abs() + P * big)
                      + 3 * e * P * (G.abs() @ Vt.abs() + big))
            val, err = res["dv"]
            val[ks, b] += Pt @ G
            err[ks, b] += (2 * u + 3 * e) * (Pt @ G.abs())
            val, err = res["dq"]
            val[qs, a] = scale * (dS @ K)
            err[qs, a] = scale * (dS_err @ K.abs()) + u * val[qs, a].abs()
            val, err = res["dk"]
            part = scale * (dS.t().contiguous() @ Q)
            val[ks, b] += part
            err[ks, b] += scale * (dS_err.t().contiguous() @ Q.abs()) + u * part.abs()
    return res


def assert_within(got, want, what):
    """got within 1.01 of its bound of want, everywhere; NaN fails."""
    val, err = want
    diff = (got.double() - val).abs()
    bad = ~(diff <= 1.01 * err + 1e-30)
    if bad.any():
        i = tuple(bad.nonzero()[0].tolist())
        raise AssertionError(f"{what}: {int(bad.sum())} of {bad.numel()} off, first at {i}: "
                             f"{float(got[i])} for {float(val[i])}, bound {float(err[i])}")
