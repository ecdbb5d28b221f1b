"""Layer norm and attention without a GPU: refusals of the Python calls and of the C entry points, shapes as traced calls
see them, the layer norm module's state, and how the autograd nodes hand tensors on."""
import ctypes

import pytest
import torch
import torch.nn as nn
from torch._subclasses.fake_tensor import FakeTensorMode

import cute_mma_b200 as cp
from cute_mma_b200 import _attention, _norm


@pytest.fixture
def fake():
    with FakeTensorMode() as mode:
        yield lambda *shape, dt=torch.bfloat16, dev="cuda": torch.empty(*shape, dtype=dt, device=dev)
        del mode


def test_cpu_tensors_are_refused():
    x = torch.randn(4, 16, dtype=torch.bfloat16)
    with pytest.raises(ValueError, match="CUDA"):
        cp.layer_norm(x, x[0])
    q = torch.randn(4, 2, 16, dtype=torch.bfloat16)
    with pytest.raises(ValueError, match="CUDA"):
        cp.causal_attention(q, q, q)
    with pytest.raises(ValueError, match="CUDA"):
        cp.decode_attention(q, q[None].expand(4, 4, 2, 16), q[None].expand(4, 4, 2, 16), torch.ones(4, dtype=torch.int32))


def test_attention_refusals(fake):
    q, k, cu = fake(10, 4, 64), fake(10, 2, 64), fake(3, dt=torch.int32)
    call = cp.causal_attention
    for bad, match in (
            (lambda: call(q.float(), k, k), "float16 or bfloat16"),
            (lambda: call(q, k.half(), k), "same dtype"),
            (lambda: call(q, k, fake(10, 2, 32)), "same shape"),
            (lambda: call(fake(10, 4, 32), k, k), "head_dim mismatch"),
            (lambda: call(fake(10, 4, 60), fake(10, 2, 60), fake(10, 2, 60)), "multiple of 8"),
            (lambda: call(fake(10, 4, 136), fake(10, 2, 136), fake(10, 2, 136)), "up to 128"),
            (lambda: call(fake(10, 3, 64), k, k), "multiple of those"),
            (lambda: call(q, fake(9, 2, 64), fake(9, 2, 64)), "same rows"),
            (lambda: call(q[0], k[0], k[0]), "3D"),
            (lambda: call(q, k[None], k[None]), "3D"),
            (lambda: call(q[None], k[None], k[None], cu), "packed"),
            (lambda: call(q, k, k, cu.long()), "int32"),
            (lambda: call(q, k, k, cu[:1]), "sequences \\+ 1"),
            (lambda: call(q, k, k, fake(6, dt=torch.int32)[::2]), "contiguous"),
            (lambda: call(q, k, k, fake(3, dt=torch.int32, dev="cpu")), "device of q"),
            (lambda: call(q, k, k, scale=0.0), "positive"),
            (lambda: call(q, k, k, scale=-1.0), "positive"),
            (lambda: call(q, k, k, scale=float("nan")), "positive"),
            (lambda: call(q, k, k, scale=float("inf")), "finite")):
        with pytest.raises(ValueError, match=match):
            bad()


def test_decode_refusals(fake):
    q, k, n = fake(3, 4, 64), fake(3, 20, 2, 64), fake(3, dt=torch.int32)
    call = cp.decode_attention
    for bad, match in (
            (lambda: call(q[None], k, k, n), "3D"),
            (lambda: call(q, k[0], k[0], n), "4D"),
            (lambda: call(q[:2], k, k, n), "same sequences"),
            (lambda: call(q, k, k, n.long()), "int32"),
            (lambda: call(q, k, k, n[:2]), "sequences"),
            (lambda: call(q, fake(3, 20, 64, 2).transpose(2, 3), k, n), "contiguous features"),
            (lambda: call(q, k, fake(3, 20, 2, 68)[..., :64], n), "multiples of 8"),
            (lambda: call(q.requires_grad_(), k, k, n), "no backward")):
        with pytest.raises(ValueError, match=match):
            bad()


def test_layer_norm_refusals(fake):
    x, w = fake(5, 48), fake(48)
    call = cp.layer_norm
    for bad, match in (
            (lambda: call(x.float(), w), "float16 or bfloat16"),
            (lambda: call(fake(5, 0), fake(0)), "last dimension"),
            (lambda: call(fake(5, 16385), fake(16385)), "last dimension"),
            (lambda: call(x, None), "weight"),
            (lambda: call(x, fake(47)), "weight"),
            (lambda: call(x, w.half()), "weight"),
            (lambda: call(x, w, fake(48, dt=torch.float32)), "same dtype"),
            (lambda: call(x, w, eps=-1e-5), "eps"),
            (lambda: call(x, w, eps=float("nan")), "eps"),
            (lambda: call(x, w, residual=fake(4, 48)), "residual"),
            (lambda: call(x, w, residual=x.half()), "residual")):
        with pytest.raises(ValueError, match=match):
            bad()
    with pytest.raises(ValueError, match="last dimension only"):
        cp.LayerNorm((4, 8))
    with pytest.raises(ValueError, match="normalized_shape"):
        cp.LayerNorm(0)


def test_shapes_of_traced_calls(fake):
    """Fake tensors take the custom ops, which say what comes back."""
    q, k = fake(2, 10, 4, 64), fake(2, 10, 2, 64)
    o = cp.causal_attention(q, k, k)
    assert o.shape == q.shape and o.dtype == q.dtype
    o, lse, low = _attention._attention_op(q, k, k, None, 0.1)
    assert lse.shape == (4, 20) and lse.dtype == torch.float32 and low.shape == q.shape
    dq, dk, dv = _attention._attention_bwd_op(o, q, k, k, o, lse, low, None, 0.1)
    assert dq.shape == q.shape and dk.shape == dv.shape == k.shape
    assert cp.decode_attention(fake(3, 4, 64), fake(3, 9, 2, 64), fake(3, 9, 2, 64), fake(3, dt=torch.int32)).shape == (3, 4, 64)
    x, w = fake(2, 7, 48), fake(48, dt=torch.float32)
    y, s = cp.layer_norm(x, w, None, residual=x)
    assert y.shape == s.shape == x.shape and cp.layer_norm(x, w, w).shape == x.shape
    y, s, stats = _norm._norm_op(x, w, None, 1e-5, x)
    assert stats.shape == (2, 14) and stats.dtype == torch.float32
    dx, dw, db = _norm._norm_bwd_op(y, None, s, w, stats)
    assert dx.shape == x.shape and dw.shape == db.shape == (48,) and dw.dtype == torch.float32


def test_layer_norm_module_takes_torch_checkpoints():
    a, b = nn.LayerNorm(24), cp.LayerNorm(24)
    with torch.no_grad():
        a.weight.normal_(), a.bias.normal_()
    b.load_state_dict(a.state_dict())
    assert torch.equal(a.weight, b.weight) and torch.equal(a.bias, b.bias) and b.eps == a.eps
    assert cp.LayerNorm(24, bias=False).bias is None
    assert cp.LayerNorm((24,)).normalized_shape == a.normalized_shape
    assert set(cp.LayerNorm(24).state_dict()) == set(a.state_dict())


def test_autograd_nodes_hand_on_what_was_asked_for(monkeypatch):
    """The eager nodes on the CPU with the library calls replaced by recorders."""
    monkeypatch.setattr(_norm, "_plain_eager", lambda *t: True)
    monkeypatch.setattr(_attention, "_plain_eager", lambda *t: True)
    monkeypatch.setattr(_norm, "_norm_forward", lambda x, w, b, eps, r, stats: (
        x * 2, None if r is None else x + r, torch.zeros(2, x.shape[0])))
    seen = {}

    def norm_backward(dy, dsum, s, w, stats, need_dbias):
        seen.update(dy=dy, dsum=dsum, need_dbias=need_dbias)
        return torch.ones_like(s), torch.full_like(w, 2.0), torch.full_like(w, 3.0) if need_dbias else None

    monkeypatch.setattr(_norm, "_norm_backward", norm_backward)
    x, r = torch.randn(3, 8, requires_grad=True), torch.randn(3, 8, requires_grad=True)
    w = torch.randn(8, requires_grad=True)
    y, s = _norm._NormFn.apply(x, w, None, 1e-5, r)
    y.sum().backward()                      # only the norm's output is used
    assert seen["dsum"] is None and not seen["need_dbias"]
    assert torch.equal(x.grad, torch.ones(3, 8)) and torch.equal(r.grad, x.grad) and torch.equal(w.grad, torch.full((8,), 2.0))
    x.grad = r.grad = None
    y, s = _norm._NormFn.apply(x, w, None, 1e-5, r)
    s.sum().backward()                      # only the sum is used: no kernel at all
    assert torch.equal(x.grad, torch.ones(3, 8)) and torch.equal(r.grad, x.grad)
    y = _norm._NormFn.apply(x, w, None, 1e-5, None)
    g, = torch.autograd.grad((y * x).sum(), x, create_graph=True)
    with pytest.raises(RuntimeError, match="once_differentiable"):
        g.sum().backward()

    monkeypatch.setattr(_attention, "_attn_forward", lambda q, k, v, cu, sc, train: (q * 1, torch.zeros(2, 3), torch.zeros(3)))

    def attn_backward(do, q, k, v, o, lse, low, cu, sc, need_dq, need_dkv):
        seen.update(need_dq=need_dq, need_dkv=need_dkv)
        return (torch.ones_like(q) if need_dq else None, *(torch.ones_like(k) if need_dkv else None for _ in range(2)))

    monkeypatch.setattr(_attention, "_attn_backward", attn_backward)
    q, k, v = (torch.randn(3, 2, 8) for _ in range(3))
    for which in ("q", "k", "v", "qkv"):
        ts = [t.clone().requires_grad_(n in which) for n, t in zip("qkv", (q, k, v))]
        o = _attention._AttentionFn.apply(*ts, None, 1.0)
        o.sum().backward()
        assert seen["need_dq"] == ("q" in which) and seen["need_dkv"] == (which != "q")
        assert [t.grad is not None for t in ts] == [n in which for n in "qkv"]


# ------------------------------------------------------------------------------------------------ the C entry points
P = ctypes.c_void_p(0x1000)
LL = ctypes.c_longlong


def _attn(L, n=1, length=8, rows=8, hq=4, hkv=2, d=64, dt=1, scale=0.1, strides=(64 * 4,) * 9, ws=256, cu=None, ptr=P, wsp=P):
    return L.prism_attn_fwd(ptr, P, P, P, None, None, cu, n, length, rows, hq, hkv, d, dt, ctypes.c_float(scale),
                            (LL * 9)(*strides) if strides else None, wsp, ws, None)


@pytest.mark.parametrize("kw,code", [
    (dict(n=0), 1), (dict(length=-1), 1), (dict(rows=9), 1), (dict(hq=5), 1), (dict(hkv=0), 1), (dict(d=12), 2), (dict(d=136), 2),
    (dict(dt=2), 1), (dict(scale=0.0), 1), (dict(scale=float("inf")), 1), (dict(strides=None), 1), (dict(strides=(64,) * 8 + (60,)), 1),
    (dict(strides=(64,) * 8 + (0,)), 1), (dict(ptr=None), 1), (dict(ptr=ctypes.c_void_p(0x1008)), 1), (dict(ws=128), 3), (dict(wsp=None), 3),
    (dict(wsp=ctypes.c_void_p(0x1010)), 1)])
def test_c_attention_refuses_before_it_launches(built_lib, kw, code):
    assert _attn(built_lib, **kw) == code
    assert len(built_lib.prism_last_error_string()) > 0


def test_c_attention_backward_and_decode_refuse(built_lib):
    s = (LL * 12)(*(256,) * 12)
    args = lambda do=P, dk=P, dv=P: built_lib.prism_attn_bwd(do, P, P, P, P, P, None, P, dk, dv, P, None, 1, 8, 8, 4, 2, 64, 1,
                                                            ctypes.c_float(0.1), s, P, 128, None)
    assert args() == 3                       # (the last check of all: nothing was launched)
    assert args(do=None) == 1
    assert args(dk=None) == 1 and b"go together" in built_lib.prism_last_error_string()
    need = built_lib.prism_attn_decode_scratch_bytes(64)
    assert need > 0 and built_lib.prism_attn_decode_scratch_bytes(200) == 0
    s8 = (LL * 8)(*(256,) * 8)
    dec = lambda n=2, room=8, hq=4, d=64, st=s8, scratch=P, nbytes=need - 1, q=P: built_lib.prism_attn_decode(
        q, P, P, P, P, n, room, hq, 2, d, 1, ctypes.c_float(0.1), st, scratch, nbytes, None)
    assert dec() == 3 and dec(scratch=None) == 3
    assert dec(n=-1) == 1 and dec(room=-1) == 1 and dec(hq=3) == 1 and dec(d=20) == 2 and dec(q=None) == 1
    assert dec(st=(LL * 8)(*(256,) * 7, 12)) == 1 and dec(st=None) == 1
    assert dec(n=0) == 0


def test_c_layer_norm_refuses(built_lib):
    L = built_lib
    f = lambda rows=4, cols=8, dt=1, wdt=1, eps=1e-5, x=P, res=None, s=None, mean=None, rstd=None, w=P: L.prism_layer_norm(
        x, res, w, None, P, s, mean, rstd, rows, cols, dt, wdt, ctypes.c_float(eps), 8, 8, None)
    assert f(rows=0) == 0
    assert f(rows=-1) == 1 and f(cols=0) == 2 and f(cols=16385) == 2 and f(dt=2) == 1 and f(wdt=0) == 1 and f(eps=-1.0) == 1
    assert f(x=None) == 1 and f(w=None) == 1 and f(res=P) == 1 and f(s=P) == 1 and f(mean=P) == 1
    need = L.prism_layer_norm_scratch_bytes(4, 8)
    assert need >= 64 and L.prism_layer_norm_scratch_bytes(-1, 8) == 0 and L.prism_layer_norm_scratch_bytes(4, 20000) == 0
    g = lambda dy=P, scratch=P, nbytes=need - 1: L.prism_layer_norm_bwd(dy, None, P, P, P, P, P, P, P, 4, 8, 1, 1, 8, 8, 8, scratch,
                                                                      nbytes, None)
    assert g() == 3 and g(scratch=None) == 3 and g(dy=None) == 1


def test_more_rows_than_row_numbers_hold_are_refused(built_lib):
    """Row numbers rounded up to whole tiles are 32-bit in the kernels."""
    most = (1 << 31) - 257
    assert _attn(built_lib, length=most + 1, rows=most + 1) == 2 and _attn(built_lib, cu=P, rows=most + 1) == 2
    assert _attn(built_lib, length=most, rows=most, ws=128) == 3   # (the last check of all)
    assert _attn(built_lib, cu=P, n=(1 << 20) + 1, rows=8) == 2 and _attn(built_lib, cu=P, n=1 << 20, rows=8, ws=128) == 3
    need = built_lib.prism_attn_decode_scratch_bytes(64)
    dec = lambda room: built_lib.prism_attn_decode(P, P, P, P, P, 2, room, 4, 2, 64, 1, ctypes.c_float(0.1), (LL * 8)(*(256,) * 8),
                                                   P, need - 1, None)
    assert dec(most + 1) == 2 and dec(most) == 3
