"""causal_attention against a float64 restatement, forward and gradients, with element-wise error bounds.

Bounds (u = half a step of the inputs' type, e = what fp32 leaves of an exponent): the kernels round the probabilities
(and in the backward dS) to 16 bits before the products with v, do, k and q, and each result once at the end:
    |o  - o64|  <= (u + e) sum_j P_ij |v_j| + u |o|
    |dv - dv64| <= (u + e) sum_i P_ij |do_i| + u |dv|
    |dS - dS64| <= (u + e) |dS| + P (|delta - delta64| + e sum_d |do| |v|),
    |delta - delta64| <= sum_d |do| (bound of o)      (delta is taken from the rounded o)
and dq, dk are sums of dS with |k|, |q| as weights, plus their own rounding.  e is twice the error of the exponent
(head_dim + 8 roundings of 2^-24 on scale sum |q| |k|, largest pair) plus 2^-20 for the two exponentials and the sums."""
import math

import pytest
import torch

import cute_mma_b200 as cp

gpu = pytest.mark.gpu
DEV = "cuda"


def _exact(q, k, v, do, lens, scale, slack=1.0):
    """(values, bounds) of o, dq, dk, dv in float64 for packed tensors; sequences in turn from row 0."""
    u = torch.finfo(q.dtype).eps / 2
    T, hq, d = q.shape
    hkv = k.shape[1]
    g = hq // hkv
    outs = [torch.zeros(t.shape, dtype=torch.float64, device=t.device) for t in (q, q, k, v)]
    tols = [torch.zeros_like(t) for t in outs]
    at = 0
    for n in lens:
        sl = slice(at, at + n)
        at += n
        if n == 0:
            continue
        keep = torch.ones(n, n, dtype=torch.bool, device=q.device).tril()
        for h in range(hq):
            Q, K, V, G = q[sl, h].double(), k[sl, h // g].double(), v[sl, h // g].double(), do[sl, h].double()
            P = torch.softmax((Q @ K.T * scale).masked_fill(~keep, -math.inf), 1)
            e = 2 * (d + 8) * 2.0 ** -24 * scale * (Q.abs() @ K.abs().T).max() + 2.0 ** -20
            O = P @ V
            tO = (u + e) * (P @ V.abs()) + u * O.abs()
            delta = (G * O).sum(1, keepdim=True)
            tDelta = (G.abs() * tO).sum(1, keepdim=True) + e * (G.abs() * O.abs()).sum(1, keepdim=True)
            dS = P * (G @ V.T - delta)
            tS = (u + e) * dS.abs() + P * (tDelta + e * (G.abs() @ V.abs().T))
            dQ, dK, dV = scale * dS @ K, scale * dS.T @ Q, P.T @ G
            outs[0][sl, h] += O
            tols[0][sl, h] += tO
            outs[1][sl, h] += dQ
            tols[1][sl, h] += scale * tS @ K.abs() + u * dQ.abs()
            outs[2][sl, h // g] += dK
            tols[2][sl, h // g] += scale * tS.T @ Q.abs() + e * scale * dS.abs().T @ Q.abs()
            outs[3][sl, h // g] += dV
            tols[3][sl, h // g] += (u + e) * (P.T @ G.abs())
    tols[2] += u * outs[2].abs()
    tols[3] += u * outs[3].abs()
    # below the smallest normal number of the type a rounding is half a step of that size
    tiny = torch.finfo(q.dtype).tiny * u * 2 if q.dtype == torch.float16 else 0.0
    return outs, [t + tiny * (1 + 64 * (i > 0)) for i, t in enumerate(tols)]


def _inputs(lens, hq, hkv, d, dt, seed=0, rows=None):
    gen = torch.Generator(device=DEV).manual_seed(seed)
    T = sum(lens) if rows is None else rows
    r = lambda h: torch.randn(T, h, d, device=DEV, generator=gen).to(dt)
    return r(hq), r(hkv), r(hkv), r(hq)


def _cu(lens):
    return torch.tensor([0] + list(lens), device=DEV).cumsum(0).to(torch.int32)


def _run(q, k, v, do, cu=None, scale=None):
    q, k, v = [t.detach().requires_grad_() for t in (q, k, v)]
    o = cp.causal_attention(q, k, v, cu, scale)
    return [o.detach(), *torch.autograd.grad(o, [q, k, v], do)]


def _close(got, want, tol, what=""):
    for name, a, b, t in zip(("o", "dq", "dk", "dv"), got, want, tol):
        bad = ~((a.double() - b).abs() <= t)   # NaN counts as bad
        assert not bad.any(), (what, name, int(bad.sum()), float((a.double() - b).abs().max()),
                               bad.nonzero()[:4].tolist())


@gpu
@pytest.mark.parametrize("lens", [(1,), (2, 1, 3), (16, 17, 15), (127,), (128,), (129,), (255, 256, 257), (300, 1, 0, 640, 33)])
@pytest.mark.parametrize("heads", [(2, 2, 64), (4, 2, 128)])
@pytest.mark.parametrize("dt", [torch.bfloat16, torch.float16])
def test_packed_lengths(lens, heads, dt):
    hq, hkv, d = heads
    q, k, v, do = _inputs(lens, hq, hkv, d, dt, seed=sum(lens) + d)
    got = _run(q, k, v, do, _cu(lens))
    cp.check_device_status()
    _close(got, *_exact(q, k, v, do, lens, d ** -0.5))


@gpu
@pytest.mark.parametrize("d", [8, 16, 32, 40, 72, 80, 96, 104, 120])
def test_head_dims(d):
    lens = (150, 7)
    q, k, v, do = _inputs(lens, 3, 1, d, torch.bfloat16, seed=d)
    got = _run(q, k, v, do, _cu(lens))
    cp.check_device_status()
    _close(got, *_exact(q, k, v, do, lens, d ** -0.5))


@gpu
@pytest.mark.parametrize("heads", [(1, 1), (5, 5), (6, 3), (7, 1), (16, 2)])
def test_head_groups_and_a_dense_batch(heads):
    hq, hkv = heads
    B, S, d = 3, 200, 64
    q, k, v, do = _inputs((S,) * B, hq, hkv, d, torch.float16, seed=hq)
    shape = lambda t: t.view(B, S, *t.shape[1:])
    got = _run(shape(q), shape(k), shape(v), shape(do), scale=0.3)
    cp.check_device_status()
    _close([t.flatten(0, 1) for t in got], *_exact(q, k, v, do, (S,) * B, 0.3))
