"""Attention over packed sequences from its definition in fp64 on the CPU,
with the error each result may carry.

Bounds. Let u be the unit roundoff of the result's type (bf16, 8 significant
bits: 2^-8; fp32: 0, its rounding is in e) and e = 2^-24 (D + L + 16) (1 + A), A the largest scale *
sum |q_d k_d|: the fp32 sums over D and L terms, worst case, and a score's
absolute error as its probability's relative one. Then, with |.| elementwise:

  out  u from rounding P, u from the result:  (2 u + e) P |V|
  dV   the same of P^T |dO|
  dS = P o (dP - delta): its rounding u |dS|; delta is summed from the rounded
       out: u P o Delta, Delta = rowsum |dO| |out|; e for dP and delta
  dQ   scale (dS's error) |K| + u |dQ|, dK scale (dS's error)^T |Q| + u |dK|
"""
import numpy as np
import torch

U = {torch.float32: 0.0, torch.bfloat16: torch.finfo(torch.bfloat16).eps / 2}


def attention(q, k, v, q_off, k_off, k_len=None, causal=False, scale=None, grad=None):
    """Dict name -> (value, bound) of out, lse and, with grad, dq, dk, dv.
    Every row sums over the keys it sees and no others."""
    u = U[q.dtype]
    q, k, v = (t.detach().double().cpu().numpy() for t in (q, k, v))
    q_off, k_off = (np.asarray(t.cpu()).astype(int) for t in (q_off, k_off))
    h, d = q.shape[1:]
    group = h // k.shape[1]
    scale = d ** -0.5 if scale is None else scale
    names = ["out"] + (["dq", "dk", "dv"] if grad is not None else [])
    like = {"out": q, "dq": q, "dk": k, "dv": v}
    val = {n: np.zeros(like[n].shape) for n in names}
    err = {n: np.zeros(like[n].shape) for n in names}
    lse = np.full((h, q.shape[0]), -np.inf)
    if grad is not None:
        grad = grad.detach().double().cpu().numpy()
    for s in range(len(q_off) - 1):
        qs = slice(q_off[s], q_off[s + 1])
        lq = q_off[s + 1] - q_off[s]
        lk = k_off[s + 1] - k_off[s] if k_len is None else int(k_len[s])
        ks = slice(k_off[s], k_off[s] + lk)
        for a in range(h):
            b = a // group
            Q, K, V = q[qs, a], k[ks, b], v[ks, b]
            see = np.ones((lq, lk), bool)
            if causal:
                see = np.arange(lk)[None, :] <= np.arange(lq)[:, None] + (lk - lq)
            rows = see.any(1) if lk else np.zeros(lq, bool)
            if not rows.any():
                continue
            sc = np.where(see, scale * (Q @ K.T), -np.inf)[rows]
            see = see[rows]
            top = sc.max(1, keepdims=True)
            w = np.exp(sc - top)
            P = w / w.sum(1, keepdims=True)
            at = np.flatnonzero(rows) + q_off[s]
            lse[a, at] = (top[:, 0] + np.log(w.sum(1)))
            A = (scale * (np.abs(Q[rows]) @ np.abs(K).T))[see].max()
            e = 2.0 ** -24 * (d + lk + 16) * (1 + A)
            O = P @ V
            val["out"][at, a] = O
            err["out"][at, a] = (2 * u + e) * (P @ np.abs(V))
            if grad is None:
                continue
            G = grad[qs, a][rows]
            dP = G @ V.T
            delta = (G * O).sum(1, keepdims=True)
            dS = P * (dP - delta)
            big = (np.abs(G) * np.abs(O)).sum(1, keepdims=True)
            dS_err = u * (np.abs(dS) + P * big) + 3 * e * P * (np.abs(G) @ np.abs(V).T + big)
            val["dv"][ks, b] += P.T @ G
            err["dv"][ks, b] += (2 * u + 3 * e) * (P.T @ np.abs(G))
            val["dq"][at, a] = scale * (dS @ K)
            err["dq"][at, a] = scale * (dS_err @ np.abs(K)) + u * np.abs(val["dq"][at, a])
            val["dk"][ks, b] += scale * (dS.T @ Q[rows])
            err["dk"][ks, b] += (scale * (dS_err.T @ np.abs(Q[rows]))
                                 + u * np.abs(scale * (dS.T @ Q[rows])))
    res = {n: (val[n], err[n]) for n in names}
    res["lse"] = lse
    return res


def assert_within(got, want, what):
    """got within 1.01 of its bound of want, everywhere (0.01: second-order
    terms of the bound); values beyond any bound (NaN) fail."""
    val, err = want
    diff = np.abs(got.detach().double().cpu().numpy() - val)
    bad = ~(diff <= 1.01 * err + 1e-30)
    if bad.any():
        i = tuple(np.argwhere(bad)[0])
        raise AssertionError(f"{what}: {bad.sum()} of {bad.size} off, first at {i}: "
                             f"{float(got[i])} for {val[i]}, bound {err[i]}")
