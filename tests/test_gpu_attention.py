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
    # below the smallest normal number of the type a rounding is half a step of that size; in bf16, whose exponents are
    # fp32's, probabilities below 2^-126 are 0 or 2^-126: up to 2^13 of them in a sum, with weights and scores of up to
    # 2^13 here, are 2^-100 at most
    tiny = torch.finfo(q.dtype).tiny * u * 2 if q.dtype == torch.float16 else 2.0 ** -100
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


def _grads_and_out(q, k, v, do, cu=None, **kw):
    return _run(q, k, v, do, cu, **kw)


@gpu
@pytest.mark.parametrize("d", [64, 128])
def test_column_ranges_of_one_matrix_are_read_in_place(d):
    """Queries, keys and values as they leave one linear layer: the same bits as from tensors of their own."""
    hq, hkv, T = 6, 2, 333
    gen = torch.Generator(device=DEV).manual_seed(1)
    qkv = torch.randn(T, (hq + 2 * hkv) * d, device=DEV, generator=gen).bfloat16()
    q, k, v = [t.unflatten(1, (-1, d)) for t in qkv.split([hq * d, hkv * d, hkv * d], 1)]
    do = torch.randn(T, hq, 2 * d, device=DEV, generator=gen).bfloat16()[..., :d]
    a = _run(q, k, v, do, _cu((200, 133)))
    b = _run(q.contiguous(), k.contiguous(), v.contiguous(), do.contiguous(), _cu((200, 133)))
    for x, y in zip(a, b):
        assert torch.equal(x, y)
    # other layouts: heads before rows, an expanded head, an odd start
    c = _run(q.transpose(0, 1).contiguous().transpose(0, 1), k, v, do, _cu((200, 133)))
    for x, y in zip(a, c):
        assert torch.equal(x, y)
    one = k[:, :1].expand(T, hkv, d)
    assert torch.equal(cp.causal_attention(q, one, one), cp.causal_attention(q, one.contiguous(), one.contiguous()))
    off = torch.empty(T * hq * d + 1, device=DEV, dtype=torch.bfloat16)[1:].view(T, hq, d).copy_(q)
    assert off.data_ptr() % 16 and torch.equal(cp.causal_attention(off, k, v), cp.causal_attention(q, k, v))


@gpu
@pytest.mark.parametrize("d", [64, 72, 128])
def test_rows_of_no_sequence_are_zeros_and_reach_nothing(d):
    """Rows in front of the first and behind the last sequence hold infinities; sequences hold NaN next to each other."""
    lens, front, T = (130, 0, 61, 200), 7, 500
    q, k, v, do = _inputs(lens, 4, 2, d, torch.bfloat16, seed=d, rows=T)
    cu = _cu(lens) + front
    end = int(cu[-1])
    for t in (q, k, v, do):
        t[:front], t[end:] = float("inf"), float("nan")
    clean = _run(q, k, v, do, cu)
    for t in clean:
        assert torch.count_nonzero(t[:front]) == 0 and torch.count_nonzero(t[end:]) == 0
    mid = slice(front, end)
    _close([t[mid] for t in clean], *_exact(q[mid], k[mid], v[mid], do[mid], lens, d ** -0.5))
    # the third sequence spoiled: the others keep their bits
    lo, hi = int(cu[2]), int(cu[3])
    for t in (q, k, v, do):
        t[lo:hi] = float("nan")
    spoiled = _run(q, k, v, do, cu)
    for a, b in zip(clean, spoiled):
        assert torch.equal(a[:lo], b[:lo]) and torch.equal(a[hi:], b[hi:])
        assert torch.isnan(b[lo:hi]).all()
    cp.check_device_status()


@gpu
def test_many_sequences():
    """More than the 256 whose lengths a CTA keeps."""
    gen = torch.Generator().manual_seed(3)
    lens = torch.randint(0, 6, (600,), generator=gen).tolist() + [140]
    q, k, v, do = _inputs(lens, 2, 1, 64, torch.float16)
    _close(_run(q, k, v, do, _cu(lens)), *_exact(q, k, v, do, lens, 0.125))
    cp.check_device_status()


@gpu
def test_many_sequences_take_a_cta_several_searches():
    """1500 sequences, some empty: every CTA works on several of their tiles and looks for each from where it found the last."""
    gen = torch.Generator().manual_seed(4)
    lens = torch.randint(0, 40, (1500,), generator=gen).tolist()
    q, k, v, do = _inputs(lens, 4, 2, 64, torch.bfloat16)
    _close(_run(q, k, v, do, _cu(lens)), *_exact(q, k, v, do, lens, 0.125))
    cp.check_device_status()


@gpu
def test_a_padded_list_of_offsets():
    """A few sequences and 100000 empty ones behind them, whose tiles of the grid have nothing to work on."""
    lens = (130, 1, 0, 300, 40)
    q, k, v, do = _inputs(lens, 4, 2, 64, torch.bfloat16, seed=9)
    cu = torch.cat([_cu(lens), torch.full((100000,), sum(lens), dtype=torch.int32, device=DEV)])
    _close(_run(q, k, v, do, cu), *_exact(q, k, v, do, lens, 0.125))
    cp.check_device_status()


@gpu
@pytest.mark.parametrize("case", [(5000, 2, 1, 128), (3001, 3, 3, 64)])
def test_long_sequences(case):
    n, hq, hkv, d = case
    q, k, v, do = _inputs((n,), hq, hkv, d, torch.bfloat16, seed=n)
    _close(_run(q, k, v, do), *_exact(q, k, v, do, (n,), d ** -0.5))


@gpu
def test_large_scores_and_growing_maxima():
    """Scores of several hundred, and rows whose maximum grows with every block of keys (O is rescaled each time)."""
    n, d = 700, 64
    q, k, v, do = _inputs((n,), 2, 2, d, torch.bfloat16, seed=5)
    q, k = q * 6, k * 6
    k = (k * torch.linspace(0.2, 1.5, n, device=DEV)[:, None, None].bfloat16())
    _close(_run(q, k, v, do), *_exact(q, k, v, do, (n,), d ** -0.5))
    r = torch.arange(n, device=DEV)
    q = torch.zeros_like(q)
    q[..., 0] = 1
    k = torch.zeros_like(k)
    k[..., 0] = (r[:, None] * 2).bfloat16()
    _close(_run(q, k, v, do, scale=1.0), *_exact(q, k, v, do, (n,), 1.0))


@gpu
def test_infinities_and_nan_among_the_scores():
    """A key at infinity (scores of +-infinity) and rows at NaN do what the formula does with them, and only there."""
    n, d = 300, 64
    q, k, v, _ = _inputs((n,), 2, 2, d, torch.float16)
    q = q.abs()
    k[150, 0] = float("-inf")                # scores of -infinity: the key has no weight
    k[:3, 1] = float("-inf")                 # rows 0, 1 and 2 of head 1 have nothing else: 0 / 0
    q[40] = float("nan")
    o = cp.causal_attention(q, k, v)
    s = torch.einsum("ihd,jhd->hij", q.double(), k.double()) * d ** -0.5
    keep = torch.ones(n, n, dtype=torch.bool, device=DEV).tril()
    p = torch.softmax(s.masked_fill(~keep, -math.inf), -1)
    want = torch.einsum("hij,jhd->ihd", p, v.double())
    assert torch.equal(torch.isnan(o), torch.isnan(want))
    fine = ~torch.isnan(want)
    assert ((o.double() - want).abs()[fine] <= 2.0 ** -9 * v.double().abs().max()).all()


@gpu
@pytest.mark.parametrize("d", [64, 128])
def test_same_bits_every_time_and_on_every_stream(d):
    lens = (500, 77, 1, 300)
    q, k, v, do = _inputs(lens, 8, 2, d, torch.bfloat16, seed=9)
    cu = _cu(lens)
    first = _run(q, k, v, do, cu)
    streams = [torch.cuda.Stream() for _ in range(3)]
    outs = []
    torch.cuda.synchronize()
    for i in range(12):
        with torch.cuda.stream(streams[i % 3]):
            outs.append(_run(q, k, v, do, cu))
    torch.cuda.synchronize()
    for got in outs:
        for a, b in zip(first, got):
            assert torch.equal(a, b)
    cp.check_device_status()


@gpu
def test_captured_graph_follows_new_inputs_and_lengths():
    lens = (100, 60)
    q, k, v, do = [t.clone() for t in _inputs(lens, 4, 2, 64, torch.bfloat16, rows=200)]
    cu = _cu(lens)
    leaves = [t.detach().requires_grad_() for t in (q, k, v)]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        o = cp.causal_attention(*leaves, cu)
        torch.autograd.grad(o, leaves, do)
        del o
    torch.cuda.current_stream().wait_stream(side)
    g1, g2 = torch.cuda.CUDAGraph(), torch.cuda.CUDAGraph()
    with torch.cuda.graph(g1):
        o1 = cp.causal_attention(*leaves, cu)
        grads1 = torch.autograd.grad(o1, leaves, do)
    with torch.cuda.graph(g2):
        o2 = cp.causal_attention(*leaves, cu)
        grads2 = torch.autograd.grad(o2, leaves, do)
    for new in ((33, 150), (200, 0), (1, 1)):
        cu.copy_(_cu(new))
        fresh = _inputs(new, 4, 2, 64, torch.bfloat16, seed=sum(new), rows=200)
        for t, f in zip((*leaves, do), fresh):
            t.data.copy_(f)
        # two graphs at once: neither uses memory of the other
        with torch.cuda.stream(side):
            side.wait_stream(torch.cuda.default_stream())
            g1.replay()
        g2.replay()
        torch.cuda.synchronize()
        n = sum(new)
        want, tol = _exact(*[t[:n] for t in fresh], new, 0.125)
        for got in ([o1, *grads1], [o2, *grads2]):
            _close([t[:n] for t in got], want, tol, new)
            assert all(torch.count_nonzero(t[n:]) == 0 for t in got)
    cp.check_device_status()


@gpu
def test_traced_calls_and_saved_tensor_hooks_agree_with_eager_ones():
    q, k, v, do = _inputs((90, 40), 4, 2, 64, torch.bfloat16)
    cu = _cu((90, 40))
    want = _run(q, k, v, do, cu)
    leaves = [t.detach().requires_grad_() for t in (q, k, v)]
    o, _, _ = torch.ops.prism_b200.causal_attention(*leaves, cu, 0.125)
    for a, b in zip([o, *torch.autograd.grad(o, leaves, do)], want):
        assert torch.equal(a, b)
    with torch.autograd.graph.saved_tensors_hooks(lambda t: t.transpose(0, -1).contiguous(), lambda t: t.transpose(0, -1)):
        o = cp.causal_attention(*leaves, cu)
    for a, b in zip([o, *torch.autograd.grad(o, leaves, do)], want):
        assert torch.equal(a, b)
    only_v = torch.autograd.grad(cp.causal_attention(q, k, leaves[2], cu), leaves[2], do)[0]
    assert torch.equal(only_v, want[3])
    only_q = torch.autograd.grad(cp.causal_attention(leaves[0], k, v, cu), leaves[0], do)[0]
    assert torch.equal(only_q, want[1])


@gpu
def test_gradients_against_differences():
    """grad . direction against central differences of the 64-bit forward: the third-order rest of a step of 2^-6 along a
    direction of unit entries is below 2^-12 of the sum of absolute products here; the gradient itself has its bound."""
    lens, d = (40, 70), 64
    q, k, v, do = _inputs(lens, 2, 1, d, torch.float16, seed=11)
    got = _run(q, k, v, do, _cu(lens))
    _, tol = _exact(q, k, v, do, lens, d ** -0.5)
    gen = torch.Generator(device=DEV).manual_seed(2)

    def loss(*t):
        out = torch.zeros(q.shape, dtype=torch.float64, device=DEV)
        at = 0
        for n in lens:
            s = torch.einsum("ihd,jd->hij", t[0][at:at + n], t[1][at:at + n, 0]) * d ** -0.5
            s = s.masked_fill(~torch.ones(n, n, dtype=torch.bool, device=DEV).tril(), -math.inf)
            out[at:at + n] = torch.einsum("hij,jd->ihd", torch.softmax(s, -1), t[2][at:at + n, 0])
            at += n
        return (out * do.double()).sum()

    base = [t.double() for t in (q, k, v)]
    h = 2.0 ** -10
    for i in range(3):
        e = torch.randn(base[i].shape, device=DEV, generator=gen, dtype=torch.float64).sign()
        plus, minus = [list(base) for _ in range(2)]
        plus[i], minus[i] = base[i] + h * e, base[i] - h * e
        num = (loss(*plus) - loss(*minus)) / (2 * h)
        ana = (got[i + 1].double() * e).sum()
        slack = tol[i + 1].sum() + 2.0 ** -12 * got[i + 1].double().abs().sum()
        assert (num - ana).abs() <= slack, (i, float(num), float(ana), float(slack))


@gpu
def test_offsets_past_32_bits():
    """The last heads of rows that lie 64 KB apart, 2.3e9 elements from the first to the last."""
    T, width, d = 70000, 32832, 64
    if torch.cuda.mem_get_info()[0] < 24 << 30:
        pytest.skip("needs 24 GB")
    buf = torch.zeros(T, width, device=DEV, dtype=torch.bfloat16)
    gen = torch.Generator(device=DEV).manual_seed(4)
    buf[:, -256:] = torch.randn(T, 256, device=DEV, generator=gen).bfloat16()
    lens = (69000, 700, 300)
    q, k, v = buf[:, -256:-128].unflatten(1, (2, d)), buf[:, -128:-64].unflatten(1, (1, d)), buf[:, -64:].unflatten(1, (1, d))
    do = torch.randn(T, 2, d, device=DEV, generator=gen).bfloat16()
    got = _run(q, k, v, do, _cu(lens))
    tail = slice(69000, T)
    _close([t[tail] for t in got], *_exact(q[tail].contiguous(), k[tail].contiguous(), v[tail].contiguous(), do[tail], lens[1:], 0.125))
    small = _run(q.contiguous(), k.contiguous(), v.contiguous(), do, _cu(lens))
    for a, b in zip(got, small):
        assert torch.equal(a, b)
    del buf


@gpu
def test_empty_calls_and_offsets_out_of_range():
    q, k, v, do = _inputs((50,), 2, 1, 64, torch.bfloat16)
    assert cp.causal_attention(q[:0], k[:0], v[:0]).shape == (0, 2, 64)
    assert cp.causal_attention(q[None, :0], k[None, :0], v[None, :0]).shape == (1, 0, 2, 64)
    o = cp.causal_attention(q, k, v, _cu((0, 0)))
    assert torch.count_nonzero(o) == 0
    # offsets that run backwards or out of the rows are taken into range (their values are the caller's business)
    for bad in ([5, 3, 400, -7], [-9, 20, 20, 90], [60, 70, 80, 90]):
        _run(q, k, v, do, torch.tensor(bad, device=DEV, dtype=torch.int32))
    torch.cuda.synchronize()
    cp.check_device_status()


@gpu
@pytest.mark.parametrize("heads", [(4, 2, 64), (3, 3, 64), (4, 2, 128), (3, 1, 80)])
@pytest.mark.parametrize("dt", [torch.bfloat16, torch.float16])
def test_what_later_rows_hold_does_not_reach_earlier_ones(heads, dt):
    """Infinities and NaN in the keys and values of later rows of the same sequence (a padded batch holds anything behind
    its lengths): earlier rows keep their bits, rows from there on are what the formula makes of them."""
    hq, hkv, d = heads
    n = 300
    q, k, v, _ = _inputs((n,) * 3, hq, hkv, d, dt, seed=d)
    q, k, v = [t.view(3, n, *t.shape[1:]) for t in (q, k, v)]
    clean = cp.causal_attention(q, k, v)
    at = (5, 140, 270)
    for b, i in enumerate(at):
        k[b, i + 1:], v[b, i + 1:], q[b, i + 1:] = float("nan"), float("nan"), float("nan")
    got = cp.causal_attention(q, k, v)
    for b, i in enumerate(at):
        assert torch.equal(got[b, :i + 1], clean[b, :i + 1])
        assert torch.isnan(got[b, i + 1:]).all()
    q, k, v, _ = _inputs((n,), hq, hkv, d, dt, seed=d)
    v[20, 0, 3], v[150, 0, 3], v[299, 0, 5], v[33, 0, 1] = float("inf"), float("-inf"), float("nan"), float("-inf")
    got = cp.causal_attention(q, k, v).float()
    g = hq // hkv
    assert torch.isfinite(got[:20, :g]).all() and (got[20:150, :g, 3] == float("inf")).all() and torch.isnan(got[150:, :g, 3]).all()
    assert (got[33:, :g, 1] == float("-inf")).all() and torch.isfinite(got[:33, :g, 1]).all() and torch.isnan(got[299, :g, 5]).all()
    rest = got.clone()
    rest[:, :g, 1] = rest[:, :g, 3] = 0
    rest[299, :g, 5] = 0
    assert torch.isfinite(rest).all()
    cp.check_device_status()
