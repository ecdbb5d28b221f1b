"""The decoder operators' C entry points without a GPU: the two attention backwards refuse alike, and what is not aligned to its
elements is refused, before anything is launched."""
import ctypes

import pytest

P = ctypes.c_void_p(0x1000)


@pytest.mark.parametrize("norms", [None, P])
def test_scaled_backward_refuses_like_the_plain_one(built_lib, norms):
    s = (ctypes.c_longlong * 12)(*(256,) * 12)

    def call(do=P, dk=P, dv=P, delta=P, dt=0, heads=4, ws=128):
        return built_lib.prism_attn_bwd_scaled(do, P, P, P, P, P, None, P, dk, dv, delta, norms, None, 1, 8, 8, heads, 2, 64, dt,
                                               ctypes.c_float(0.1), s, P, ws, None)
    assert call() == 3 and call(dt=1) == 3   # (the last check of all)
    assert call(do=None) == 1 and call(delta=None) == 1 and call(heads=3) == 1 and call(dt=2) == 1
    assert call(dv=None) == 1 and b"go together" in built_lib.prism_last_error_string()


def test_pointers_between_elements_are_refused(built_lib):
    L, LL = built_lib, ctypes.c_longlong
    odd, two = ctypes.c_void_p(0x1001), ctypes.c_void_p(0x1002)
    scale = ctypes.c_float(0.1)
    fwd = lambda lse=None, cu=None: L.prism_attn_fwd(P, P, P, P, lse, None, cu, 1, 8, 8, 4, 2, 64, 1, scale, (LL * 9)(*(256,) * 9), P, 128, None)
    assert fwd() == 3 and fwd(lse=P, cu=P) == 3 and fwd(lse=two) == 1 and fwd(cu=two) == 1
    s12 = (LL * 12)(*(256,) * 12)
    bwd = lambda lse=P, delta=P, norms=P, cu=None: L.prism_attn_bwd_scaled(
        P, P, P, P, P, lse, None, P, P, P, delta, norms, cu, 1, 8, 8, 4, 2, 64, 0, scale, s12, P, 128, None)
    assert bwd() == 3 and bwd(lse=two) == 1 and bwd(delta=two) == 1 and bwd(norms=two) == 1 and bwd(cu=odd) == 1
    need = L.prism_attn_decode_scratch_bytes(64)
    dec = lambda n=P: L.prism_attn_decode(P, P, P, P, n, 2, 8, 4, 2, 64, 1, scale, (LL * 8)(*(256,) * 8), P, need - 1, None)
    assert dec() == 3 and dec(two) == 1
    norm = lambda x=P, res=None, w=P, b=None, y=P, s=None, mean=None, rstd=None, wdt=1: L.prism_layer_norm(
        x, res, w, b, y, s, mean, rstd, 0, 8, 1, wdt, ctypes.c_float(1e-5), 8, 8, None)
    assert norm() == 0 and norm(x=two, w=two, y=two) == 0 and norm(wdt=2) == 0 and norm(w=two, wdt=2) == 1 and norm(x=odd) == 1 and norm(b=odd) == 1
    assert norm(y=odd) == 1 and norm(res=odd, s=P) == 1 and norm(mean=two, rstd=P) == 1
    need = L.prism_layer_norm_scratch_bytes(4, 8)
    back = lambda dy=P, ds=None, dx=P, dw=P, mean=P: L.prism_layer_norm_bwd(
        dy, ds, P, P, mean, P, dx, dw, P, 4, 8, 1, 1, 8, 8, 8, P, need - 1, None)
    assert back() == 3 and back(dy=odd) == 1 and back(ds=odd) == 1 and back(dx=odd) == 1 and back(dw=odd) == 1 and back(mean=two) == 1
