"""Packed causal attention in 64 bits, with elementwise bounds on what a kernel may be off by.

The bounds follow the roundings of the kernels, U being half a step of a type (``finfo.eps / 2``):
  scores     a sum of hs products in fp32:           ds  <= (hs + 8) U32 sum|q||k| / sqrt(hs) + 4 U32 |s|
  p = e^s    exp to a few units, weights rounded to the input type before the second product: dp/p <= 2 ds + 16 U32 + Up
  output     n terms added in fp32, rounded to the type:  U|o| + (dp/p + (n + 8) U32) sum p|v|
and the chain rule carries them through the gradients."""
import math

import torch

U = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8}
U32 = 2.0 ** -24


def weight_rounding(dtype):
    """Probabilities and score gradients enter the tensor-core products as bf16; the fp32 kernels keep them."""
    return U[torch.bfloat16] if dtype == torch.bfloat16 else 0.0


def spans(lens, gap=0):
    out, at = [], gap
    for n in lens:
        out.append((at, at + n))
        at += n
    return out


def forward(q, k, v, lens, heads, kv_heads, gap=0):
    """o, lse, bound of o, bound of lse: fp64 [T, heads*hs] / [heads, T]; rows of no sequence stay NaN (bound inf)."""
    T, hs, group = q.shape[0], q.shape[1] // heads, heads // kv_heads
    dt, dev = q.dtype, q.device
    o = torch.full((T, heads * hs), math.nan, dtype=torch.float64, device=dev)
    lse = torch.full((heads, T), math.nan, dtype=torch.float64, device=dev)
    bo, bl = torch.full_like(o, math.inf), torch.full_like(lse, math.inf)
    for a, b in spans(lens, gap):
        n = b - a
        if n == 0:
            continue
        hide = torch.ones(n, n, dtype=torch.bool, device=dev).triu(1)
        for h in range(heads):
            qc, kc = slice(h * hs, (h + 1) * hs), slice((h // group) * hs, (h // group + 1) * hs)
            Q, K, V = q[a:b, qc].double(), k[a:b, kc].double(), v[a:b, kc].double()
            s = (Q @ K.T / math.sqrt(hs)).masked_fill(hide, -math.inf)
            m = torch.logsumexp(s, 1)
            p = torch.exp(s - m[:, None])
            ds = score_bound(Q, K, s, hide, hs)
            rel = 2 * ds + 16 * U32 + weight_rounding(dt)
            o[a:b, qc], lse[h, a:b] = p @ V, m
            bo[a:b, qc] = U[dt] * (p @ V).abs() + ((rel + (n + 8) * U32) * p) @ V.abs()
            bl[h, a:b] = ds.max(1).values + (n + 8) * U32 + 8 * U32 * m.abs()
    return o, lse, bo, bl


def score_bound(Q, K, s, hide, hs):
    ds = (hs + 8) * U32 * (Q.abs() @ K.abs().T) / math.sqrt(hs) + 4 * U32 * s.abs().nan_to_num(posinf=0.0)
    ds = ds.masked_fill(hide, 0.0)
    return ds.max(1, keepdim=True).values.expand_as(ds)  # every weight of a row depends on all its scores


def backward(q, k, v, d_o, lens, heads, kv_heads, gap=0):
    """(dq, dk, dv) and their bounds, for a kernel that is given its own forward's o and lse."""
    T, hs, group = q.shape[0], q.shape[1] // heads, heads // kv_heads
    dt, dev, sc = q.dtype, q.device, 1 / math.sqrt(q.shape[1] // heads)
    new = lambda w: torch.zeros(T, w, dtype=torch.float64, device=dev)
    dq, dk, dv = new(heads * hs), new(kv_heads * hs), new(kv_heads * hs)
    bq, bk, bv = new(heads * hs), new(kv_heads * hs), new(kv_heads * hs)
    w = weight_rounding(dt)
    for a, b in spans(lens, gap):
        n = b - a
        if n == 0:
            continue
        hide = torch.ones(n, n, dtype=torch.bool, device=dev).triu(1)
        for h in range(heads):
            qc, kc = slice(h * hs, (h + 1) * hs), slice((h // group) * hs, (h // group + 1) * hs)
            Q, K, V, G = q[a:b, qc].double(), k[a:b, kc].double(), v[a:b, kc].double(), d_o[a:b, qc].double()
            s = (Q @ K.T * sc).masked_fill(hide, -math.inf)
            m = torch.logsumexp(s, 1, keepdim=True)
            p = torch.exp(s - m)
            O, dP = p @ V, G @ V.T
            delta = (O * G).sum(1, keepdim=True)
            dS = p * (dP - delta) * sc
            ds = score_bound(Q, K, s, hide, hs)
            # o and lse of the forward are off by their own bounds
            eo = U[dt] * O.abs() + ((2 * ds + 16 * U32 + w + (n + 8) * U32) * p) @ V.abs()
            el = ds[:, :1] + (n + 8) * U32 + 8 * U32 * m.abs()
            ep = (ds + el + 16 * U32 + 4 * U32 * m.abs())  # relative, of a weight taken against the given lse
            edelta = (G.abs() * eo).sum(1, keepdim=True) + (hs + 8) * U32 * (G.abs() * O.abs()).sum(1, keepdim=True)
            edp = (hs + 8) * U32 * (G.abs() @ V.abs().T) + 4 * U32 * (dP.abs() + delta.abs())
            eds = (ep + w + 4 * U32) * dS.abs() + (1 + ep) * p * (edp + edelta) * sc
            dq[a:b, qc] += dS @ K
            dk[a:b, kc] += dS.T @ Q
            dv[a:b, kc] += p.T @ G
            add = (n * group + 8) * U32
            bq[a:b, qc] += (eds + add * dS.abs()) @ K.abs()
            bk[a:b, kc] += (eds + add * dS.abs()).T @ Q.abs()
            bv[a:b, kc] += ((ep + w + add) * p).T @ G.abs()
    for g, bound in ((dq, bq), (dk, bk), (dv, bv)):
        bound += U[dt] * (g.abs() + bound) + 1e-30
    return (dq, dk, dv), (bq, bk, bv)
