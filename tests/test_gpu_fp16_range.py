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


def _backward_parts(q, k, v, do, scale):
    """One head in 64 bits: P, dS, o, and the results dq, dk, dv."""
    Q, K, V, G = (t.double() for t in (q, k, v, do))
    P = torch.softmax((Q @ K.T * scale).masked_fill_(~_causal(len(Q)), -math.inf), -1)
    O = P @ V
    dS = P * (G @ V.T - (G * O).sum(1, keepdim=True))
    return P, dS, O, (scale * dS @ K, scale * dS.T @ Q, P.T @ G)


@gpu
@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("size", [1.0, 1e-2, 1e-3])
def test_small_output_gradients_over_long_rows(d, size):
    """8192 keys: the errors of dq and dk as norms are at most twice what independent roundings of half a step make of them.
    A rounding has a mean square of u^2 / 3 of its value; dS is rounded once, P once on the way to o, which gives delta an error
    of its own, what the second rounding of o leaves is 2^-3 of it, and the results are rounded at the end."""
    n, scale = 8192, d ** -0.5
    gen = torch.Generator(device=DEV).manual_seed(d)
    q, k, v, do = (torch.randn(n, 1, d, device=DEV, generator=gen) for _ in range(4))
    q, k, v, do = q.half(), k.half(), v.half(), (do * size).half()
    got = _gradients(q, k, v, do, scale)
    P, dS, O, want = _backward_parts(q[:, 0], k[:, 0], v[:, 0], do[:, 0], scale)
    Q, K, V, G = (t[:, 0].double() for t in (q, k, v, do))
    r = U * U / 3
    delta = r * ((P * (G @ V.T)) ** 2).sum(1) + r * 2.0 ** -6 * ((G * O) ** 2).sum(1)
    var = [scale ** 2 * (r * (dS ** 2 @ (K ** 2).sum(1)).sum() + (delta * ((P @ K) ** 2).sum(1)).sum()),
           scale ** 2 * (r * (dS.T ** 2 @ (Q ** 2).sum(1)).sum() + (delta[None] * P.T ** 2 @ (Q ** 2).sum(1)).sum()),
           r * (P.T ** 2 @ (G ** 2).sum(1)).sum()]
    for name, a, b, x in zip(("dq", "dk", "dv"), got, want, var):
        x = x + r * (b ** 2).sum() + 2.0 ** -50 / 3 * b.numel()
        err = (a[:, 0] - b).norm()
        assert err <= 2 * x.sqrt(), (name, float(err / b.norm()), float(x.sqrt() / b.norm()))


@gpu
@pytest.mark.parametrize("d", [64, 80, 128])
def test_large_output_gradients(d):
    """dS beyond fp16's largest number while dq and dk are far below it: |dS| is off by (u + e) |dS|, by the error of delta, and
    by 2^-25 of a step that puts the largest dS at 2^14 to 2^15."""
    n, scale = 300, d ** -0.5
    gen = torch.Generator(device=DEV).manual_seed(d)
    q, k, v, do = (torch.randn(n, 1, d, device=DEV, generator=gen) for _ in range(4))
    q, k, v, do = (0.02 * q).half(), (0.02 * k).half(), (8 * v).half(), (5000 * do).half()
    got = _gradients(q, k, v, do, scale)
    P, dS, O, want = _backward_parts(q[:, 0], k[:, 0], v[:, 0], do[:, 0], scale)
    assert dS.abs().max() > 65504 and max(float(w.abs().max()) for w in want) < 60000
    Q, K, V, G = (t[:, 0].double() for t in (q, k, v, do))
    e = _exponent_error(d, q[0], k, scale)
    # (delta from o and what its rounding took, which is kept to 2^-3 of itself)
    t_delta = (G.abs() * ((U + e) * (P @ V.abs()) + U / 8 * O.abs())).sum(1, keepdim=True) + e * (G.abs() * O.abs()).sum(1, keepdim=True)
    bound = 2 * G.norm(dim=1).max() * V.norm(dim=1).max()
    t_s = (U + e) * dS.abs() + P * (t_delta + e * (G.abs() @ V.abs().T)) + 2.0 ** -39 * bound * _causal(n)
    tol = [scale * t_s @ K.abs(), scale * t_s.T @ Q.abs(), (U + e) * (P.T @ G.abs()) + 2.0 ** -40 * G.abs().sum(0)]
    for name, a, b, t in zip(("dq", "dk", "dv"), got, want, tol):
        t = t + U * b.abs() + 2.0 ** -25
        bad = ~((a[:, 0] - b).abs() <= t)
        assert not bad.any(), (name, int(bad.sum()), float(((a[:, 0] - b).abs() / t).max()))


@gpu
@pytest.mark.parametrize("d", [64, 128])
def test_what_the_range_is_taken_from(d):
    """Rows of no sequence, whatever they hold, do not move the other rows' gradients; nor do rows that are not finite.  Zeros
    give zeros."""
    lens, front, T, hq, hkv = (130, 0, 61, 200), 7, 500, 4, 2
    gen = torch.Generator(device=DEV).manual_seed(d)
    q, k, v, do = (torch.randn(T, h, d, device=DEV, generator=gen).half() for h in (hq, hkv, hkv, hq))
    cu = torch.tensor([0] + list(lens), device=DEV).cumsum(0).to(torch.int32) + front
    end = int(cu[-1])

    def grads():
        leaves = [t.detach().requires_grad_() for t in (q, k, v)]
        return torch.autograd.grad(cp.causal_attention(*leaves, cu), leaves, do)

    for t in (q, k, v, do):
        t[:front], t[end:] = 0, 0
    clean = grads()
    for fill in (6e4, float("inf"), float("nan")):
        for t in (q, k, v, do):
            t[:front], t[end:] = fill, fill
        assert all(torch.equal(a, b) for a, b in zip(clean, grads()))
    lo, hi = int(cu[2]), int(cu[3])
    v[lo:hi] *= 0.01
    do[lo:hi] *= 0.01
    clean = grads()
    do[lo + 5, 1, 3] = float("inf")
    v[lo + 9, 0, 2] = float("nan")
    for a, b in zip(clean, grads()):
        assert torch.equal(a[:lo], b[:lo]) and torch.equal(a[hi:], b[hi:])
    do.zero_()
    assert all(torch.count_nonzero(t[:lo]) == 0 and torch.count_nonzero(t[hi:]) == 0 for t in grads())
    cp.check_device_status()


@gpu
def test_gradients_of_a_strided_batch_on_several_streams_and_in_graphs():
    """A batch of 4D column ranges of one matrix: the bits of contiguous tensors, on any stream, and from two graphs at once, whose
    calls each have a range of their own."""
    B, S, hq, hkv, d = 3, 333, 4, 2, 64
    gen = torch.Generator(device=DEV).manual_seed(6)
    qkv = torch.randn(B, S, hq + 2 * hkv, d, device=DEV, generator=gen).half()
    do = [(torch.randn(B, S, hq, d, device=DEV, generator=gen) * s).half() for s in (1.0, 1e-3)]
    parts = [t.detach().requires_grad_() for t in qkv.split([hq, hkv, hkv], 2)]
    whole = [t.detach().contiguous().requires_grad_() for t in parts]
    call = lambda ts, g: torch.autograd.grad(cp.causal_attention(*ts), ts, g)
    want = [call(whole, g) for g in do]
    streams = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    outs = []
    for i in range(8):
        with torch.cuda.stream(streams[i % 2]):
            outs.append(call(parts, do[i % 2]))
    torch.cuda.synchronize()
    for i, got in enumerate(outs):
        assert all(torch.equal(a, b) for a, b in zip(got, want[i % 2]))
    graphs, results = [torch.cuda.CUDAGraph() for _ in do], []
    for graph, g in zip(graphs, do):
        with torch.cuda.graph(graph):
            results.append(call(parts, g))
    for _ in range(5):
        for graph, stream in zip(graphs, streams):
            with torch.cuda.stream(stream):
                graph.replay()
    torch.cuda.synchronize()
    for got, w in zip(results, want):
        assert all(torch.equal(a, b) for a, b in zip(got, w))
    cp.check_device_status()
