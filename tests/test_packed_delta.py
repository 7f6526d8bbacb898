"""delta = rowsum(P dP) of the packed backward does not depend on how the forward's output was rounded: the kernels correct
rowsum(dO o) by what P and dP themselves say.  The output is moved by a step of its type, towards the cotangent in every
element, so that what the rounding of o would do to delta adds up; the gradients have to stay within a bound that has no
term for it."""
import math

import pytest
import torch

import b200_llama as B
import packed_reference as R

U32, W = R.U32, 2.0 ** -8   # half a step of fp32, of bf16


def moved(o, d_o):
    """o, one bf16 step up where the cotangent is positive, one down where it is negative."""
    bits = o.view(torch.int16).int()
    up = torch.where(bits >= 0, bits + 1, bits - 1)   # (a negative number's bits grow with its magnitude)
    down = torch.where(bits >= 0, bits - 1, bits + 1)
    there = torch.where(d_o > 0, up, down)
    return torch.where((bits & 0x7fff) == 0, bits, there).to(torch.int16).view(torch.bfloat16)


def gradients(q, k, v, d_o, o, lens, heads, kv_heads, corrected=True):
    """(dq, dk, dv) in 64 bits from the given output, and bounds of a kernel in bf16.  With p off by ep (relative; the scores'
    and the log-sum-exp's bounds) and dP by edp, delta = delta0 + sum p (dP - delta0) is off by
      sum p (ep (|dP| + |delta0|) + edp) + (n + 16) U32 sum p |dP - delta0| + 4 U32 |delta0|
    and nothing else.  dS is rounded once; dQ either as sum dS K, or as sum dS0 K - eps sum P K with dS0 = p (dP - delta0) and P
    rounded and eps = delta - delta0.  ``corrected`` False: delta0 itself is taken."""
    T, hs, group = q.shape[0], q.shape[1] // heads, heads // kv_heads
    sc, dev = 1 / math.sqrt(hs), q.device
    new = lambda w: torch.zeros(T, w, dtype=torch.float64, device=dev)
    out = [new(heads * hs), new(kv_heads * hs), new(kv_heads * hs)]
    bounds = [torch.zeros_like(x) for x in out]
    for a, b in R.spans(lens):
        n = b - a
        hide = torch.ones(n, n, dtype=torch.bool, device=dev).triu(1)
        for h in range(heads):
            qc, kc = slice(h * hs, (h + 1) * hs), slice((h // group) * hs, (h // group + 1) * hs)
            Q, K, V, G, O = (x[a:b, c].double() for x, c in ((q, qc), (k, kc), (v, kc), (d_o, qc), (o, qc)))
            s = (Q @ K.T * sc).masked_fill(hide, -math.inf)
            m = torch.logsumexp(s, 1, keepdim=True)
            p, dP = torch.exp(s - m), G @ V.T
            delta0 = (G * O).sum(1, keepdim=True)
            delta = (p * dP).sum(1, keepdim=True) if corrected else delta0
            dS, dS0, eps = p * (dP - delta), p * (dP - delta0).abs(), (delta - delta0).abs()
            ds = R.score_bound(Q, K, s, hide, hs)
            ep = ds + ds[:, :1] + (n + 24) * U32 + 12 * U32 * m.abs()
            edp = (hs + 8) * U32 * (G.abs() @ V.abs().T) + 4 * U32 * (dP.abs() + delta0.abs())
            edelta = ((p * (ep * (dP.abs() + delta0.abs()) + edp)).sum(1, keepdim=True) + (n + 16) * U32 * dS0.sum(1, keepdim=True)
                      + 4 * U32 * delta0.abs())
            eds = (ep + 4 * U32) * dS.abs() + (1 + ep) * p * (edp + edelta)
            add = (n * group + 8) * U32
            out[0][a:b, qc] += dS @ K * sc
            out[1][a:b, kc] += dS.T @ Q * sc
            out[2][a:b, kc] += p.T @ G
            bounds[0][a:b, qc] += (eds + (W + add) * (dS.abs() + dS0 + eps * p)) @ K.abs() * sc
            bounds[1][a:b, kc] += (eds + (W + add) * dS.abs()).T @ Q.abs() * sc
            bounds[2][a:b, kc] += ((ep + W + add) * p).T @ G.abs()
    for x, bd in zip(out, bounds):
        bd += W * (x.abs() + bd) + 1e-30
    return out, bounds


def inputs(lens, heads, kv, hs, dev, seed):
    g = torch.Generator(device=dev).manual_seed(seed)
    return [torch.randn(sum(lens), n * hs, generator=g, device=dev).bfloat16() for n in (heads, kv, kv, heads)]


LENS = [9, 1, 70, 300]


@pytest.mark.parametrize("hs", [64, 128])
def test_the_bound_tells_delta_from_the_output_apart(hs):
    """The oracle with delta taken from the moved output leaves the bounds of dq and dk; with the corrected one it does not."""
    q, k, v, d_o = inputs(LENS, 2, 1, hs, "cpu", 3)
    o = moved(R.forward(q, k, v, LENS, 2, 1)[0].bfloat16(), d_o)
    want, bounds = gradients(q, k, v, d_o, o, LENS, 2, 1)
    wrong, _ = gradients(q, k, v, d_o, o, LENS, 2, 1, corrected=False)
    assert all(bool(((w - r).abs() > b).any()) for w, r, b in list(zip(wrong, want, bounds))[:2])
    plain, _ = R.backward(q, k, v, d_o, LENS, 2, 1)
    assert all(torch.allclose(x, r, rtol=1e-9, atol=1e-12) for x, r in zip(plain, want))


@pytest.mark.gpu
@pytest.mark.parametrize("impl", [0, 2])
@pytest.mark.parametrize("heads,kv,hs", [(4, 2, 64), (4, 2, 128), (2, 2, 64), (3, 1, 128)])
def test_gradients_do_not_follow_the_output_s_rounding(heads, kv, hs, impl):
    q, k, v, d_o = inputs(LENS, heads, kv, hs, "cuda", 4)
    cu = torch.tensor([0] + torch.tensor(LENS).cumsum(0).tolist(), dtype=torch.int32, device="cuda")
    o, lse = B.attention_packed(q, k, v, cu, heads, kv, impl=impl)
    for out in (o, moved(o, d_o), moved(moved(o, d_o), d_o)):
        got = B.attention_packed_backward(q, k, v, out, lse, d_o, cu, heads, kv, impl=impl)
        assert B.device_status() == 0
        want, bounds = gradients(q, k, v, d_o, out, LENS, heads, kv)
        for name, x, r, b in zip(("dq", "dk", "dv"), got, want, bounds):
            err = (x.double() - r).abs()
            assert bool((err <= b).all()), (name, float((err / b).max()))
