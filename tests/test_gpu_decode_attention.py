"""decode_attention against a float64 restatement, with an element-wise error bound.

|o - o64| <= (u + e) sum_j P_j |v_j| + u |o|: the probabilities are rounded to the inputs' type once (u: half a step), the
result once, and e is what fp32 leaves of an exponent (see the bound of the prompt's attention).  In fp16 probabilities
below 2^-14 of the largest are off by up to 2^-25 of it, each with its value's weight."""
import pytest
import torch

import cute_mma_b200 as cp

gpu = pytest.mark.gpu
DEV = "cuda"


def _inputs(b, room, hq, hkv, d, dt, seed=0):
    gen = torch.Generator(device=DEV).manual_seed(seed)
    r = lambda *s: torch.randn(*s, device=DEV, generator=gen).to(dt)
    return r(b, hq, d), r(b, room, hkv, d), r(b, room, hkv, d)


def _check(o, q, k, v, lens, scale):
    u = torch.finfo(q.dtype).eps / 2
    g, d = q.shape[1] // k.shape[2], q.shape[2]
    for i, n in enumerate(lens):
        if n == 0:
            assert torch.count_nonzero(o[i]) == 0
            continue
        Q = q[i].double().unflatten(0, (-1, g))
        K, V = k[i, :n].double().transpose(0, 1), v[i, :n].double().transpose(0, 1)
        P = torch.softmax(Q @ K.transpose(1, 2) * scale, -1)
        e = 2 * (d + 8) * 2.0 ** -24 * scale * (Q.abs() @ K.abs().transpose(1, 2)).max() + 2.0 ** -20
        O = (P @ V).flatten(0, 1)
        tol = (u + e) * (P @ V.abs()).flatten(0, 1) + u * O.abs()
        if q.dtype == torch.float16:
            tol = tol + 2.0 ** -25 * (P.amax(-1, keepdim=True) * V.abs().sum(1, keepdim=True)).flatten(0, 1) + 2.0 ** -24
        bad = ~((o[i].double() - O).abs() <= tol)
        assert not bad.any(), (i, n, int(bad.sum()), float((o[i].double() - O).abs().max()))


@gpu
@pytest.mark.parametrize("lens", [(1,), (63, 64, 65), (0, 5, 0, 1000, 128, 0), (2000,), (17,) * 70])
@pytest.mark.parametrize("heads", [(1, 1, 64), (12, 12, 64), (8, 2, 128), (6, 2, 72), (40, 2, 32), (16, 1, 128)])
@pytest.mark.parametrize("dt", [torch.bfloat16, torch.float16])
def test_lengths_and_heads(lens, heads, dt):
    hq, hkv, d = heads
    q, k, v = _inputs(len(lens), max(lens) + 9, hq, hkv, d, dt, seed=sum(lens) + d)
    for i, n in enumerate(lens):   # what is behind the length does not matter
        k[i, n:], v[i, n:] = float("nan"), float("inf")
    o = cp.decode_attention(q, k, v, torch.tensor(lens, device=DEV, dtype=torch.int32))
    _check(o, q, k, v, lens, d ** -0.5)


@gpu
@pytest.mark.parametrize("d", [8, 16, 24, 40, 56, 80, 96, 104, 112, 120])
def test_head_dims(d):
    lens = (300, 33)
    q, k, v = _inputs(2, 310, 4, 2, d, torch.bfloat16, seed=d)
    o = cp.decode_attention(q, k, v, torch.tensor(lens, device=DEV, dtype=torch.int32), scale=0.2)
    _check(o, q, k, v, lens, 0.2)
