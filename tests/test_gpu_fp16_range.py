"""Weights and gradients that 16-bit floats of 5 exponent bits can only hold if the kernels use all of their range: many keys
that weigh little each, and small output gradients over thousands of keys."""
import math

import pytest
import torch

import cute_mma_b200 as cp

gpu = pytest.mark.gpu
DEV = "cuda"
U = 2.0 ** -11   # half a step of fp16


def _one_loud_key(n, hkv, d, at, seed=0):
    """Scores (scale 1) of one key 17 nats above a spread of a half; the loud key's values are zeros, so that results are made
    of the others alone.  q: one head for every key head."""
    gen = torch.Generator(device=DEV).manual_seed(seed)
    k = torch.randn(n, hkv, d, device=DEV, generator=gen).half()
    k[..., 0] = (0.5 * torch.randn(n, hkv, device=DEV, generator=gen)).half()
    k[at, :, 0] = 17.0
    v = (1 + torch.randn(n, hkv, d, device=DEV, generator=gen)).half()
    v[at] = 0
    q = torch.zeros(hkv, d, device=DEV, dtype=torch.float16)
    q[:, 0] = 1
    return q, k, v


def _exponent_error(d, q, k, scale):
    """Twice what d + 8 roundings of fp32 leave of a score, and 2^-20 for exponentials and sums."""
    return 2 * (d + 8) * 2.0 ** -24 * scale * float((q.double().abs()[:, None] * k.double().abs().transpose(0, 1)).sum(-1).max()) + 2.0 ** -20


@gpu
@pytest.mark.parametrize("case", [(100003, 1, 2, 64, 7), (4099, 700, 2, 64, 0), (2500, 900, 1, 128, 17), (3000, 1000, 3, 24, 40)])
def test_decode_keys_that_weigh_little(case):
    """|o - o64| <= (u + e) sum P |v| + u |o|, and what fp16 with a largest weight of 2^15 rounds away below its normal
    numbers: 2^-25 of 2^-15 of the largest weight, a key.  Many sequences (of one cache) leave whole ones to a CTA."""
    n, b, hkv, d, at = case
    q, k, v = _one_loud_key(n, hkv, d, at, seed=d)
    lengths = torch.full((b,), n, device=DEV, dtype=torch.int32)
    o = cp.decode_attention(q.expand(b, hkv, d), k.expand(b, n, hkv, d), v.expand(b, n, hkv, d), lengths, scale=1.0).double()
    P = torch.softmax(torch.einsum("hd,jhd->hj", q.double(), k.double()), -1)
    want = torch.einsum("hj,jhd->hd", P, v.double())
    e = _exponent_error(d, q, k, 1.0)
    tol = (U + e) * torch.einsum("hj,jhd->hd", P, v.double().abs()) + U * want.abs()
    tol += 2.0 ** -40 * P.amax(-1, keepdim=True) * v.double().abs().sum(0) + 2.0 ** -25
    assert ((o - want).abs() <= tol).all(), float(((o - want).abs() / tol).max())


@gpu
@pytest.mark.parametrize("case", [(4099, 2, 64, 0), (3000, 1, 128, 17), (2500, 3, 80, 1)])
def test_prompt_keys_that_weigh_little(case):
    """As above, with a largest weight of 2^7 to 2^15 (its reference is the row's maximum or one 2^8 below)."""
    n, hkv, d, at = case
    q, k, v = _one_loud_key(n, hkv, d, at, seed=d)
    o = cp.causal_attention(q.expand(n, hkv, d), k, v, scale=1.0).double()
    s = torch.einsum("hd,jhd->hj", q.double(), k.double())[:, None].expand(hkv, n, n)
    P = torch.softmax(s.masked_fill(~torch.ones(n, n, device=DEV, dtype=torch.bool).tril(), -math.inf), -1)
    want = torch.einsum("hij,jhd->ihd", P, v.double())
    e = _exponent_error(d, q, k, 1.0)
    tol = (U + e) * torch.einsum("hij,jhd->ihd", P, v.double().abs()) + U * want.abs()
    tol += 2.0 ** -32 * P.amax(-1).T[..., None] * v.double().abs().cumsum(0) + 2.0 ** -25
    assert ((o - want).abs() <= tol).all(), float(((o - want).abs() / tol).max())


def _causal(n):
    return torch.ones(n, n, device=DEV, dtype=torch.bool).tril()


def _gradients(q, k, v, do, scale):
    leaves = [t.detach().requires_grad_() for t in (q, k, v)]
    out = torch.autograd.grad(cp.causal_attention(*leaves, scale=scale), leaves, do)
    cp.check_device_status()
    return [t.double() for t in out]


@gpu
@pytest.mark.parametrize("case", [(4099, 64, 0), (3000, 128, 17), (2500, 80, 1)])
def test_value_gradients_of_keys_that_weigh_little(case):
    """|dv - dv64| <= (u + e) sum_i P |do| + u |dv|, and 2^-25 of 2^-15 a row: P has a factor of 2^15."""
    n, d, at = case
    q, k, v = _one_loud_key(n, 1, d, at, seed=d)
    do = (1 + torch.randn(n, 1, d, device=DEV, generator=torch.Generator(device=DEV).manual_seed(n))).half()
    dv = _gradients(q.expand(n, 1, d), k, v, do, 1.0)[2][:, 0]
    s = (k[:, 0].double() @ q[0].double()).expand(n, n)
    P = torch.softmax(s.masked_fill(~_causal(n), -math.inf), -1)
    G = do[:, 0].double()
    want = P.T @ G
    e = _exponent_error(d, q, k, 1.0)
    tol = (U + e) * (P.T @ G.abs()) + U * want.abs() + 2.0 ** -40 * G.abs().flip(0).cumsum(0).flip(0) + 2.0 ** -25
    assert ((dv - want).abs() <= tol).all(), float(((dv - want).abs() / tol).max())
