"""Attention inside a window from its definition in fp64 on the device, with
the bounds of attention_reference (u, e and each result's formula are stated
there)."""
import math

import torch

from attention_reference import U


def sees(lq, lk, causal, window, sinks, device):
    """[lq, lk]: whether a row sees a key."""
    p = torch.arange(lq, device=device)[:, None] + (lk - lq)
    j = torch.arange(lk, device=device)[None, :]
    m = ((p - j).abs() < window) | (j < sinks)
    return m & (j <= p) if causal else m


def attention(q, k, v, q_off, k_off, k_len=None, causal=False, grad=None, window=1, sinks=0,
              scale=None):
    """Dict name -> (value, bound), fp64 on the device, of out and, with grad,
    dq, dk, dv."""
    u = U[q.dtype]
    h, d = q.shape[1:]
    group = h // k.shape[1]
    scale = d ** -0.5 if scale is None else scale
    like = {"out": q, "dq": q, "dk": k, "dv": k}
    names = list(like) if grad is not None else ["out"]
    res = {n: tuple(torch.zeros(like[n].shape, dtype=torch.float64, device=q.device)
                    for _ in range(2)) for n in names}
    q_off, k_off = q_off.tolist(), k_off.tolist()
    k_len = None if k_len is None else k_len.tolist()
    for s in range(len(q_off) - 1):
        lq = q_off[s + 1] - q_off[s]
        lk = k_off[s + 1] - k_off[s] if k_len is None else k_len[s]
        if not lq or not lk:
            continue
        seen = sees(lq, lk, causal, window, sinks, q.device)
        rows = seen.any(1).nonzero()[:, 0] + q_off[s]
        seen = seen[seen.any(1)]
        if not len(rows):
            continue
        ks = slice(k_off[s], k_off[s] + lk)
        for b in range(k.shape[1]):
            heads = slice(b * group, (b + 1) * group)
            Q = q[rows, heads].double().transpose(0, 1).contiguous()  # [group, rows, d]
            K, V = (t[ks, b].double() for t in (k, v))
            Kt = K.t().contiguous()
            S = (scale * (Q @ Kt)).masked_fill_(~seen, -math.inf)
            A = (scale * (Q.abs() @ Kt.abs())).masked_fill_(~seen, 0.0)
            e = 2.0 ** -24 * (d + int(seen.sum(1).max()) + 16) * (1 + A.amax((1, 2), True))
            P = S.softmax(-1)
            O = P @ V
            val, err = res["out"]
            val[rows, heads] = O.transpose(0, 1)
            err[rows, heads] = ((2 * u + e) * (P @ V.abs())).transpose(0, 1)
            if grad is None:
                continue
            G = grad[rows, heads].double().transpose(0, 1).contiguous()
            Pt, Vt = P.transpose(1, 2).contiguous(), V.t().contiguous()
            dS = P * (G @ Vt - (G * O).sum(-1, keepdim=True))
            big = (G.abs() * O.abs()).sum(-1, keepdim=True)
            dS_err = (u * (dS.abs() + P * big)
                      + 3 * e * P * (G.abs() @ Vt.abs() + big))
            val, err = res["dv"]
            val[ks, b] += (Pt @ G).sum(0)
            err[ks, b] += ((2 * u + 3 * e) * (Pt @ G.abs())).sum(0)
            val, err = res["dq"]
            dQ = scale * (dS @ K)
            val[rows, heads] = dQ.transpose(0, 1)
            err[rows, heads] = (scale * (dS_err @ K.abs()) + u * dQ.abs()).transpose(0, 1)
            val, err = res["dk"]
            part = scale * (dS.transpose(1, 2).contiguous() @ Q)
            val[ks, b] += part.sum(0)
            err[ks, b] += (scale * (dS_err.transpose(1, 2).contiguous() @ Q.abs())
                           + u * part.abs()).sum(0)
    return res
