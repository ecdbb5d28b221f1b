"""The attention backward's C entry points without a GPU: both refuse alike, before anything is launched."""
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
