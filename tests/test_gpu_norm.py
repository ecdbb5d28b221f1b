"""layer_norm against a float64 restatement, forward and gradients, with element-wise error bounds.

Bounds (u = half a step of the result's type, f = 2^-24): a thread adds up to 32 values one after the other and its row's
threads join in a tree, 50 roundings at most, so a mean is off by 50 f mean|s|, a normalised value by
    eh = rstd 50 f (mean|s| + |s|) + 60 f |xh|
and y by u |y| + |w| eh + 4 f (|y| + |b|).  dx = rstd (g - c0 - xh c1): each term by its own roundings and eh times what it
is multiplied with.  The parameters' gradients are sums over the rows: eh |dy| a row and one rounding a row."""
import pytest
import torch

import cute_mma_b200 as cp

gpu = pytest.mark.gpu
DEV = "cuda"
F = 2.0 ** -24


def _inputs(m, n, dt, wt, seed=0, offset=0.0):
    gen = torch.Generator(device=DEV).manual_seed(seed)
    r = lambda *s: torch.randn(*s, device=DEV, generator=gen)
    x = (r(m, n) + offset).to(dt)
    return x, (1 + 0.2 * r(n)).to(wt), (0.3 * r(n)).to(wt), r(m, n).to(dt), r(m, n).to(dt), r(m, n).to(dt)


def _check(x, w, b, dy, res, ds, got, eps=1e-5):
    """got: y, s or None, dx, dw, db."""
    dt, u = x.dtype, torch.finfo(x.dtype).eps / 2
    uw = torch.finfo(w.dtype).eps / 2
    s = x.double()
    if res is not None:
        total = x.float() + res.float()
        assert torch.equal(got[1], total.to(dt))
        s = total.to(dt).double()
    W, B, G = w.double(), b.double(), dy.double()
    mean = s.mean(1, keepdim=True)
    rstd = ((s - mean) ** 2).mean(1, keepdim=True).add(eps).rsqrt()
    xh = (s - mean) * rstd
    y = xh * W + B
    eh = rstd * 50 * F * (s.abs().mean(1, keepdim=True) + s.abs()) + 60 * F * xh.abs()
    ty = u * y.abs() + W.abs() * eh + 4 * F * (y.abs() + B.abs())
    g = G * W
    c0, c1 = g.mean(1, keepdim=True), (g * xh).mean(1, keepdim=True)
    own = rstd * (g - c0 - xh * c1)
    dx = own + (ds.double() if ds is not None else 0)
    a0, a1 = g.abs().mean(1, keepdim=True), (g * xh).abs().mean(1, keepdim=True)
    tx = (u * dx.abs() + rstd * (60 * F * (g.abs() + a0 + xh.abs() * a1) + eh * c1.abs() + xh.abs() * (g.abs() * eh).mean(1, keepdim=True))
          + rstd * (g.abs() + a0 + xh.abs() * a1) * (60 * F + (rstd * 50 * F * s.abs().mean(1, keepdim=True)) ** 2) + 4 * F * dx.abs())
    dw, db = (G * xh).sum(0), G.sum(0)
    rows = x.shape[0] + 50
    tw = uw * dw.abs() + (G.abs() * eh).sum(0) + rows * F * (G * xh).abs().sum(0)
    tb = uw * db.abs() + rows * F * G.abs().sum(0)
    tiny = 2.0 ** -24 if dt == torch.float16 else 0.0   # a rounding below the smallest normal fp16 number
    tiny_w = 2.0 ** -24 if w.dtype == torch.float16 else 0.0
    for name, a, r, t in (("y", got[0], y, ty + tiny), ("dx", got[2], dx, tx + tiny), ("dw", got[3], dw, tw + tiny_w),
                          ("db", got[4], db, tb + tiny_w)):
        bad = ~((a.double() - r).abs() <= t)
        assert not bad.any(), (name, int(bad.sum()), float((a.double() - r).abs().max()), bad.nonzero()[:4].tolist())


def _run(x, w, b, dy, res=None, ds=None, eps=1e-5):
    x, w, b = [t.detach().requires_grad_() for t in (x, w, b)]
    if res is None:
        y = cp.layer_norm(x, w, b, eps)
        return [y.detach(), None, *torch.autograd.grad(y, [x, w, b], dy)]
    res = res.detach().requires_grad_()
    y, s = cp.layer_norm(x, w, b, eps, residual=res)
    if ds is None:
        dx, dw, db, dr = torch.autograd.grad(y, [x, w, b, res], dy)
    else:
        dx, dw, db, dr = torch.autograd.grad([y, s], [x, w, b, res], [dy, ds])
    assert torch.equal(dx, dr)
    return [y.detach(), s.detach(), dx, dw, db]


@gpu
@pytest.mark.parametrize("n", [1, 2, 7, 8, 31, 33, 64, 200, 256, 257, 264, 512, 513, 520, 768, 776, 1000, 1024, 1025, 1537, 4096,
                               4098, 4104, 8192, 8193, 9000, 12288, 16384])
@pytest.mark.parametrize("m", [1, 3, 37])
def test_widths(m, n):
    x, w, b, dy, _, _ = _inputs(m, n, torch.bfloat16, torch.bfloat16, seed=n)
    _check(x, w, b, dy, None, None, _run(x, w, b, dy))


@gpu
@pytest.mark.parametrize("n", [24, 300, 768, 1023, 4096, 5001])
@pytest.mark.parametrize("types", [(torch.bfloat16, torch.float32), (torch.float16, torch.float16), (torch.float16, torch.float32)])
@pytest.mark.parametrize("with_ds", [False, True])
def test_residual_and_types(n, types, with_ds):
    m = 700
    x, w, b, dy, res, ds = _inputs(m, n, *types, seed=n + with_ds)
    ds = ds if with_ds else None
    _check(x, w, b, dy, res, ds, _run(x, w, b, dy, res, ds))


@gpu
def test_rows_far_from_zero_and_constant_rows():
    x, w, b, dy, _, _ = _inputs(40, 768, torch.float16, torch.float32, offset=100.0)
    x[5] = 7.0
    x[6] = 0.0
    _check(x, w, b, dy, None, None, _run(x, w, b, dy))


@gpu
@pytest.mark.parametrize("n", [768, 1537, 512])
def test_strided_rows_and_odd_starts(n):
    m = 200
    x, w, b, dy, res, ds = _inputs(m, n, torch.bfloat16, torch.bfloat16, seed=n)
    want = _run(x, w, b, dy, res, ds)
    wide = lambda t: torch.cat([t, t], 1)[:, :n]
    got = _run(wide(x), w, b, wide(dy), wide(res), wide(ds))
    odd = lambda t: torch.empty(m * n + 1, device=DEV, dtype=t.dtype)[1:].view(m, n).copy_(t)
    got2 = _run(odd(x), w, b, odd(dy), odd(res), odd(ds))
    flipped = lambda t: t.t().contiguous().t()
    got3 = _run(flipped(x), w, b, flipped(dy), flipped(res), flipped(ds))
    for other in (got, got2, got3):
        for name, i in (("y", 0), ("s", 1), ("dx", 2)):
            # (rows read in other pieces are summed in another order)
            assert torch.allclose(other[i].float(), want[i].float(), rtol=2.0 ** -7, atol=2.0 ** -10), name
        _check(x, w, b, dy, res, ds, other)


@gpu
def test_leading_dimensions_single_values_and_no_rows():
    x, w, b, dy, _, _ = _inputs(24, 96, torch.float16, torch.float16)
    y = cp.layer_norm(x, w, b)
    assert torch.equal(cp.layer_norm(x.view(2, 3, 4, 96), w, b), y.view(2, 3, 4, 96))
    assert torch.equal(cp.layer_norm(x[5], w, b), y[5])
    assert cp.layer_norm(x[:0], w, b).shape == (0, 96)
    e, w1, b1 = x[:0].detach().requires_grad_(), w.detach().requires_grad_(), b.detach().requires_grad_()
    for g in torch.autograd.grad(cp.layer_norm(e, w1, b1), [e, w1, b1], x[:0])[1:]:
        assert torch.count_nonzero(g) == 0
    no_bias = cp.layer_norm(x, w)
    assert torch.allclose(no_bias.float() + b.float(), y.float(), atol=2e-2)


@gpu
@pytest.mark.parametrize("n", [96, 768, 4096])
def test_a_spoiled_row_stays_in_its_row(n):
    x, w, b, dy, _, _ = _inputs(70, n, torch.bfloat16, torch.float32)
    clean = _run(x, w, b, dy)
    x[33, 5], dy[20] = float("inf"), float("nan")
    got = _run(x, w, b, dy)
    keep = torch.ones(70, dtype=torch.bool, device=DEV)
    keep[33] = False
    assert torch.equal(got[0][keep], clean[0][keep]) and torch.isnan(got[0][33]).all()
    keep[20] = False
    assert torch.equal(got[2][keep], clean[2][keep]) and torch.isnan(got[2][20]).all()
    assert torch.isnan(got[3]).all() and torch.isnan(got[4]).all()


@gpu
def test_same_bits_every_time_streams_and_graphs():
    x, w, b, dy, res, ds = _inputs(3000, 768, torch.bfloat16, torch.float32)
    first = _run(x, w, b, dy, res, ds)
    streams = [torch.cuda.Stream() for _ in range(3)]
    torch.cuda.synchronize()
    outs = []
    for i in range(9):
        with torch.cuda.stream(streams[i % 3]):
            outs.append(_run(x, w, b, dy, res, ds))
    torch.cuda.synchronize()
    for got in outs:
        for a, c in zip(first, got):
            assert torch.equal(a, c)
    leaves = [t.detach().clone().requires_grad_() for t in (x, w, b, res)]
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y, s = cp.layer_norm(*leaves[:3], residual=leaves[3])
        grads = torch.autograd.grad([y, s], leaves[:3], [dy, ds])
    with torch.no_grad():
        leaves[0].copy_(x.flip(0))
        leaves[3].copy_(res.flip(0))
    dy.copy_(dy.flip(0))
    ds.copy_(ds.flip(0))
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(y, first[0].flip(0)) and torch.equal(s, first[1].flip(0)) and torch.equal(grads[0], first[2].flip(0))
    assert torch.allclose(grads[1], first[3], rtol=1e-4, atol=1e-3)


@gpu
def test_unused_outputs_traced_calls_and_hooks():
    x, w, b, dy, res, ds = _inputs(50, 264, torch.bfloat16, torch.bfloat16)
    want = _run(x, w, b, dy, res, ds)
    l = [t.detach().requires_grad_() for t in (x, w, b, res)]
    y, s, _ = torch.ops.prism_b200.layer_norm(*l[:3], 1e-5, l[3])
    got = [y, s, *torch.autograd.grad([y, s], l, [dy, ds])]
    for a, c in zip(got, want):
        assert torch.equal(a, c)
    y, s = cp.layer_norm(*l[:3], residual=l[3])
    dx, dr = torch.autograd.grad(s, [l[0], l[3]], ds)
    assert torch.equal(dx, ds) and torch.equal(dr, ds)
    with torch.autograd.graph.saved_tensors_hooks(lambda t: t.t().contiguous(), lambda t: t.t()):
        y, s = cp.layer_norm(*l[:3], residual=l[3])
    for a, c in zip(torch.autograd.grad([y, s], l[:3], [dy, ds]), want[2:]):
        assert torch.equal(a, c)


@gpu
def test_gradients_against_differences():
    """Central differences of the 64-bit forward along directions of unit entries; their third-order rest is below 2^-12
    of the sum of absolute products for a step of 2^-10."""
    x, w, b, dy, _, _ = _inputs(30, 200, torch.float16, torch.float32, seed=8)
    got = _run(x, w, b, dy)
    gen = torch.Generator(device=DEV).manual_seed(5)

    def loss(x, w, b):
        return (torch.nn.functional.layer_norm(x, (200,), w, b, 1e-5) * dy.double()).sum()

    base, h = [x.double(), w.double(), b.double()], 2.0 ** -10
    for i in range(3):
        e = torch.randn(base[i].shape, device=DEV, generator=gen, dtype=torch.float64).sign()
        plus, minus = [list(base) for _ in range(2)]
        plus[i], minus[i] = base[i] + h * e, base[i] - h * e
        num = (loss(*plus) - loss(*minus)) / (2 * h)
        g = got[2 + i].double()
        assert (num - (g * e).sum()).abs() <= (2.0 ** -11 + 2.0 ** -12) * g.abs().sum() + 1e-3


@gpu
def test_module_matches_torch_and_many_rows():
    a, c = torch.nn.LayerNorm(320, device=DEV), cp.LayerNorm(320, device=DEV)
    with torch.no_grad():
        a.weight.normal_(), a.bias.normal_()
    c.load_state_dict(a.state_dict())
    x = torch.randn(200000, 320, device=DEV).bfloat16()
    assert torch.allclose(c(x).float(), a(x.float()), atol=2e-2, rtol=2.0 ** -8)
    y, s = c(x, x)
    assert torch.equal(s, x + x) and torch.equal(y, c(s))


@gpu
def test_offsets_past_32_bits():
    m, n, ld = 70000, 512, 32768
    if torch.cuda.mem_get_info()[0] < 16 << 30:
        pytest.skip("needs 16 GB")
    buf = torch.zeros(m, ld, device=DEV, dtype=torch.bfloat16)
    x = buf[:, -n:]
    x.normal_()
    _, w, b, dy, _, _ = _inputs(m, n, torch.bfloat16, torch.float32)
    got, want = _run(x, w, b, dy), _run(x.contiguous(), w, b, dy)
    for i in (0, 2, 3, 4):
        assert torch.equal(got[i], want[i])
    del buf, x
