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
