"""What the forward keeps of o's rounding for the backward: o + low is what o was before it was rounded, and delta is taken from both."""
import ctypes
import math

import pytest
import torch

import cute_mma_b200 as cp
from cute_mma_b200 import _attention, _lib
from cute_mma_b200 import _functional as F

gpu = pytest.mark.gpu
DEV = "cuda"


def _case(dt, hq, hkv, d, lens, rows, seed):
    gen = torch.Generator(device=DEV).manual_seed(seed)
    q, k, v, do = (torch.randn(rows, h, d, device=DEV, generator=gen).to(dt) for h in (hq, hkv, hkv, hq))
    return q, k, v, do, torch.tensor([0] + list(lens), device=DEV).cumsum(0).to(torch.int32)


def _low(low, dt):
    """e5m2 bytes, of 2^8 (bf16) or 2^11 (fp16) times what the rounding took."""
    return low.view(torch.float8_e5m2).double() / (256 if dt == torch.bfloat16 else 2048)


@gpu
@pytest.mark.parametrize("heads", [(2, 2, 8), (3, 3, 40), (4, 2, 64), (3, 1, 80), (8, 2, 128)])
@pytest.mark.parametrize("dt", [torch.bfloat16, torch.float16])
def test_low_is_the_rest_of_o(heads, dt):
    """A row of one key is its value, and low next to nothing: the exponent, 0 or fp16's 7 in the end, has two fp32 roundings of at
    most 2^-24 (|score| + 7), scores here are below 16, ex2 adds 2^-22 and 1 / l 2^-23, together below 2^-18 of o.  Elsewhere low is at most half a step of o (u |o|, or 2^-25 below
    fp16's normal numbers), with e5m2's own rounding of 2^-3 on top, and o + low has P's rounding and 2^-3 of o's:
    |o + low - o64| <= (u + e) sum P |v| + (u / 8) |o|."""
    hq, hkv, d = heads
    lens, rows = (1, 130, 0, 77, 256, 3), 500
    q, k, v, _, cu = _case(dt, hq, hkv, d, lens, rows, d)
    u = torch.finfo(dt).eps / 2
    o, lse, low = _attention._attn_forward(q, k, v, cu, d ** -0.5, True)
    cp.check_device_status()
    rest = _low(low, dt)
    total = o.double() + rest
    step = torch.clamp(u * o[:467].double().abs() * (1 + 2 * u), min=2.0 ** -25 if dt == torch.float16 else 0)   # (|o| may have been rounded down)
    assert (rest[:467].abs() <= 1.125 * step).all(), float((rest[:467].abs() - 1.125 * step).max())
    assert torch.equal(o[0], v[0].repeat_interleave(hq // hkv, 0))
    assert (rest[0].abs() <= 2.0 ** -18 * o[0].double().abs()).all()
    at, errs, errs_o = 0, 0.0, 0.0
    for n in lens:
        sl = slice(at, at + n)
        at += n
        for h in range(hq):
            Q, K, V = q[sl, h].double(), k[sl, h // (hq // hkv)].double(), v[sl, h // (hq // hkv)].double()
            S = (Q @ K.T * d ** -0.5).masked_fill(~torch.ones(n, n, device=DEV, dtype=torch.bool).tril(), -math.inf)
            P = torch.softmax(S, -1) if n else S
            want = P @ V
            e = 2 * (d + 8) * 2.0 ** -24 * float((Q.abs() @ K.abs().T).max() if n else 0) + 2.0 ** -20
            tiny = 2.0 ** -25 if dt == torch.float16 else 2.0 ** -120
            assert ((total[sl, h] - want).abs() <= (u + e) * (P @ V.abs()) + u / 8 * want.abs() + tiny).all()
            errs += float(((total[sl, h] - want) ** 2).sum())
            errs_o += float(((o[sl, h].double() - want) ** 2).sum())
    # with the rest o is clearly closer: P's rounding is averaged over a row's keys, o's own is not
    assert errs < 0.5 * errs_o, (errs, errs_o)


@gpu
@pytest.mark.parametrize("heads", [(2, 2, 8), (3, 3, 40), (4, 2, 64), (3, 1, 80), (8, 2, 128)])
@pytest.mark.parametrize("dt", [torch.bfloat16, torch.float16])
def test_low_is_where_its_element_is(heads, dt):
    """Two keys of the same score: o is the mean of two values and P is exact in 16 bits, so that o + low is that mean to 2^-3 of
    a rounding, element by element."""
    hq, hkv, d = heads
    rows = 2 * 150
    gen = torch.Generator(device=DEV).manual_seed(d)
    q = torch.zeros(rows, hq, d, device=DEV, dtype=dt)
    k, v = (torch.randn(rows, hkv, d, device=DEV, generator=gen).to(dt) for _ in range(2))
    cu = torch.arange(0, rows + 1, 2, device=DEV, dtype=torch.int32)
    o, _, low = _attention._attn_forward(q, k, v, cu, 1.0, True)
    cp.check_device_status()
    u = torch.finfo(dt).eps / 2
    mean = ((v[0::2].double() + v[1::2].double()) / 2).repeat_interleave(hq // hkv, 1)
    total = (o.double() + _low(low, dt))[1::2]
    assert ((total - mean).abs() <= u / 8 * mean.abs() + 2.0 ** -22 * (v[0::2].double().abs() + v[1::2].double().abs())
            .repeat_interleave(hq // hkv, 1) + 2.0 ** -28).all()
    assert int((o[1::2].double() != mean).sum()) > mean.numel() // 8     # (there is something that rounding takes)


@gpu
@pytest.mark.parametrize("heads", [(2, 2, 8), (3, 3, 40), (4, 2, 64), (5, 1, 80), (8, 2, 128)])
@pytest.mark.parametrize("dt", [torch.bfloat16, torch.float16])
def test_delta_takes_both(heads, dt):
    """The backward's scratch: delta = do . (o + low) to fp32's roundings of its 2 d terms, and do . o where low is not given."""
    hq, hkv, d = heads
    lens, rows = (130, 1, 200), 333
    q, k, v, do, cu = _case(dt, hq, hkv, d, lens, rows, d + 1)
    o, lse, low = _attention._attn_forward(q, k, v, cu, d ** -0.5, True)
    end = sum(lens)
    low[end:] = 0   # (rows of no sequence are not written)
    L = _lib.lib()
    strides = _attention._STRIDES12(*(x for t in (q, k, v, do) for x in _attention._steps(t)))
    for given in (low, None):
        delta = torch.full((hq, rows), float("nan"), device=DEV)
        norms = torch.full((2,), float("nan"), device=DEV)
        ws = F._workspace.get(q.device, 256)
        dq = torch.empty_like(q)
        _lib.check(L.prism_attn_bwd_scaled(
            do.data_ptr(), q.data_ptr(), k.data_ptr(), v.data_ptr(), o.data_ptr(), lse.data_ptr(), F._ptr(given), dq.data_ptr(), None, None,
            delta.data_ptr(), norms.data_ptr(), cu.data_ptr(), len(lens), 0, rows, hq, hkv, d, F._DTYPES[dt], ctypes.c_float(d ** -0.5),
            strides, ws.data_ptr(), ws.numel(), F._raw_stream(q.device)))
        cp.check_device_status()
        both = o.double() + (_low(low, dt) if given is not None else 0)
        want, size = (do.double() * both).sum(-1).T, (do.double().abs() * (o.double().abs() + _low(low, dt).abs())).sum(-1).T
        assert ((delta.double() - want).abs() <= 2 * d * 2.0 ** -24 * size + 1e-30).all()
        if dt == torch.float16:   # the largest squares of the norms of do's and of v's rows of sequences
            for got, t in zip(norms.tolist(), (do, v)):
                exact = float((t[:end].double() ** 2).sum(-1).max())
                assert abs(got - exact) <= d * 2.0 ** -24 * exact
