"""Layer norm of the decoder that Prism layers stand in, with the residual sum before it (``layer_norm``, ``LayerNorm``).

The reference's training model uses PyTorch's norm and a separate addition around its Prism layers
(integration/model.py); here both are one pass over the rows, and the weight's gradient is summed in a fixed order.
"""
from __future__ import annotations

import torch
import torch.nn as nn

from . import _functional as F
from . import _lib
from ._module import _plain_eager, _plain_grad, _refuse_tangents

MAX_COLS = 16384


def _check_norm(x, weight, bias, eps, residual) -> None:
    if not x.is_cuda:
        raise ValueError(f"x must be a CUDA tensor, got device={x.device}")
    if x.dtype not in F._DTYPES:
        raise ValueError(f"x must be float16 or bfloat16, got dtype={x.dtype}")
    if x.dim() < 1 or not 1 <= x.shape[-1] <= MAX_COLS:
        raise ValueError(f"the last dimension of x must be in [1, {MAX_COLS}], got shape {tuple(x.shape)}")
    n = x.shape[-1]
    for name, t in (("weight", weight), ("bias", bias)):
        if t is None:
            if name == "weight":
                raise ValueError("weight must be a tensor")
            continue
        if t.shape != (n,) or not t.is_contiguous() or t.device != x.device or t.dtype not in (x.dtype, torch.float32):
            raise ValueError(f"{name} must be a contiguous ({n},) tensor of float32 or {x.dtype} on the device of x")
    if bias is not None and bias.dtype != weight.dtype:
        raise ValueError(f"weight and bias must have the same dtype, got {weight.dtype} and {bias.dtype}")
    if not eps >= 0.0:
        raise ValueError(f"eps must not be negative, got {eps}")
    if residual is not None and (residual.shape != x.shape or residual.dtype != x.dtype or residual.device != x.device):
        raise ValueError(f"residual must be a {tuple(x.shape)} tensor of the same dtype and device as x")
    if x.numel() // n >= 1 << 31:
        raise ValueError("more than 2^31 rows")


def _rows(t):
    """t as rows with contiguous columns, and the step between them."""
    if t.dim() != 2:
        t = t.reshape(-1, t.shape[-1])
    if t.stride(1) != 1 and t.shape[1] != 1:
        t = t.contiguous()
    return t, t.stride(0)


def _w_code(weight):
    return F.DTYPE_F32 if weight.dtype == torch.float32 else F._DTYPES[weight.dtype]


def _norm_forward(x, weight, bias, eps, residual, stats):
    """(y, sum or None, statistics or None): means and reciprocal standard deviations of the rows as a (2, rows) tensor."""
    # (new_empty with contiguous strides: less host time than torch.empty with its keywords)
    y = x.new_empty(x.shape)
    s = x.new_empty(x.shape) if residual is not None else None
    n = x.shape[-1]
    m = x.numel() // n
    st = x.new_empty((2, m), dtype=torch.float32) if stats else None
    if m == 0:
        return y, s, st
    x2, ldx = _rows(x)
    r2, ldr = _rows(residual) if residual is not None else (None, 0)
    mean = st.data_ptr() if stats else None
    with F._device_scope(x.device):
        _lib.check(_lib.lib().prism_layer_norm(
            x2.data_ptr(), F._ptr(r2), weight.data_ptr(), F._ptr(bias), y.data_ptr(), F._ptr(s), mean,
            mean + 4 * m if stats else None, m, n, F._DTYPES[x.dtype], _w_code(weight), eps, ldx, ldr, F._raw_stream(x.device)))
    return y, s, st


_scratch_cache: dict = {}


def _scratch_bytes(L, m, n, device) -> int:
    """``prism_layer_norm_scratch_bytes`` on the current device, remembered for the latest shapes."""
    key = (m, n, device.index)
    nbytes = _scratch_cache.get(key)
    if nbytes is None:
        if len(_scratch_cache) >= 512:
            _scratch_cache.clear()
        nbytes = _scratch_cache[key] = L.prism_layer_norm_scratch_bytes(m, n)
    return nbytes


def _norm_backward(dy, dsum, s, weight, stats, need_dbias):
    """(dx, dweight, dbias or None) for the rows s that were normalised."""
    weight, stats = weight.contiguous(), stats.contiguous()   # (saved-tensor hooks may have handed back another layout)
    dx = s.new_empty(s.shape)
    dw = torch.empty_like(weight)
    db = torch.empty_like(weight) if need_dbias else None
    n = s.shape[-1]
    m = s.numel() // n
    if m == 0:
        return dx, dw.zero_(), None if db is None else db.zero_()
    s2, lds = _rows(s)
    dy2, lddy = _rows(dy)
    ds2, ldds = _rows(dsum) if dsum is not None else (None, 0)
    L = _lib.lib()
    with F._device_scope(s.device):
        nbytes = _scratch_bytes(L, m, n, s.device)
        scratch = stats.new_empty(nbytes >> 2)
        mean = stats.data_ptr()
        _lib.check(L.prism_layer_norm_bwd(
            dy2.data_ptr(), F._ptr(ds2), s2.data_ptr(), weight.data_ptr(), mean, mean + 4 * m, dx.data_ptr(), dw.data_ptr(),
            F._ptr(db), m, n, F._DTYPES[s.dtype], _w_code(weight), lddy, ldds, lds, scratch.data_ptr(), nbytes,
            F._raw_stream(s.device)))
    return dx, dw, db


# ---------------------------------------------------------------------------
# custom ops (traced, compiled and transformed calls) and the eager autograd node, as for the layer itself
# ---------------------------------------------------------------------------
@torch.library.custom_op("prism_b200::layer_norm", mutates_args=())
def _norm_op(x: torch.Tensor, weight: torch.Tensor, bias: torch.Tensor | None, eps: float, residual: torch.Tensor | None
             ) -> tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
    y, s, stats = _norm_forward(x, weight, bias, eps, residual, True)
    return y, x.new_empty(0) if s is None else s, stats


@_norm_op.register_fake
def _(x, weight, bias, eps, residual):
    return (x.new_empty(x.shape), x.new_empty(0 if residual is None else x.shape),
            x.new_empty((2, x.shape[:-1].numel()), dtype=torch.float32))


@torch.library.custom_op("prism_b200::layer_norm_backward", mutates_args=())
def _norm_bwd_op(dy: torch.Tensor, dsum: torch.Tensor | None, s: torch.Tensor, weight: torch.Tensor, stats: torch.Tensor
                 ) -> tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
    return _norm_backward(dy, dsum, s, weight, stats, True)


@_norm_bwd_op.register_fake
def _(dy, dsum, s, weight, stats):
    return s.new_empty(s.shape), torch.empty_like(weight), torch.empty_like(weight)


def _norm_setup(ctx, inputs, output):
    x, weight, bias, eps, residual = inputs
    _, s, stats = output
    ctx.save_for_backward(x if residual is None else s, weight, stats)
    ctx.has_bias, ctx.has_residual = bias is not None, residual is not None
    ctx.mark_non_differentiable(stats, *(() if residual is not None else (s,)))


def _norm_grad(ctx, dy, dsum, _dstats):
    s, weight, stats = ctx.saved_tensors
    dx, dw, db = _norm_bwd_op(dy, dsum if ctx.has_residual else None, s, weight, stats)
    return dx, dw, db if ctx.has_bias else None, None, dx.clone() if ctx.has_residual else None


_norm_op.register_autograd(_norm_grad, setup_context=_norm_setup)


class _NormFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, bias, eps, residual):
        y, s, stats = _norm_forward(x, weight, bias, eps, residual, True)
        ctx.save_for_backward(x if residual is None else s, weight, stats)
        ctx.has_bias, ctx.has_residual = bias is not None, residual is not None
        ctx.set_materialize_grads(False)
        return y if residual is None else (y, s)

    @staticmethod
    def backward(ctx, dy, dsum=None):
        # (the decorator costs 14 us of host time, and only a backward that is itself recorded needs it)
        return (_NormFn._recorded if torch.is_grad_enabled() else _NormFn._grads)(ctx, dy, dsum)

    @staticmethod
    def _grads(ctx, dy, dsum):
        s, weight, stats = ctx.saved_tensors
        if dy is None:
            # only the sum was used: its gradient is x's and the residual's
            return dsum, None, None, None, dsum
        plain = _plain_eager(dy, dsum, s, weight, stats) and _plain_grad(dy) and (dsum is None or _plain_grad(dsum))
        if plain:
            dx, dw, db = _norm_backward(dy, dsum, s, weight, stats, ctx.has_bias)
        else:
            dx, dw, db = _norm_bwd_op(dy, dsum, s, weight, stats)
        return dx, dw, db if ctx.has_bias else None, None, dx if ctx.has_residual else None

    _recorded = staticmethod(torch.autograd.function.once_differentiable(lambda ctx, dy, dsum: _NormFn._grads(ctx, dy, dsum)))


def layer_norm(x, weight, bias=None, eps: float = 1e-5, residual=None):
    """``(s - mean(s)) / sqrt(var(s) + eps) * weight + bias`` over the last dimension; differentiable.

    ``s`` is x, or ``x + residual`` rounded to x's type; with a residual the result is ``(y, s)``, so that the residual
    stream goes on from ``s``.  x (and residual): float16 or bfloat16, any leading dimensions, the last one up to 16384;
    weight and bias: float32 or x's type, their gradients likewise.  Statistics are taken in fp32 from deviations from
    the mean; the sums over rows of the parameters' gradients have a fixed order.
    """
    _check_norm(x, weight, bias, eps, residual)
    eps = float(eps)
    if _plain_eager(x, weight, bias, residual):
        if torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in (x, weight, bias, residual)):
            return _NormFn.apply(x, weight, bias, eps, residual)
        y, s, _ = _norm_forward(x, weight, bias, eps, residual, False)
        return y if residual is None else (y, s)
    _refuse_tangents("layer_norm", x, weight, bias, residual)
    y, s, _ = _norm_op(x, weight, bias, eps, residual)
    return y if residual is None else (y, s)


class LayerNorm(nn.Module):
    """``nn.LayerNorm`` over the last dimension on ``layer_norm``: same parameters and initialisation, so that its
    checkpoints load.  ``forward(x, residual)`` adds the residual first and returns ``(y, x + residual)``."""

    def __init__(self, normalized_shape: int, eps: float = 1e-5, bias: bool = True, device=None, dtype=None):
        super().__init__()
        if not isinstance(normalized_shape, int):
            if len(normalized_shape) != 1:
                raise ValueError(f"LayerNorm is over the last dimension only, got normalized_shape={normalized_shape}")
            normalized_shape = int(normalized_shape[0])
        if not 1 <= normalized_shape <= MAX_COLS:
            raise ValueError(f"normalized_shape must be in [1, {MAX_COLS}], got {normalized_shape}")
        self.normalized_shape, self.eps = (normalized_shape,), eps
        self.weight = nn.Parameter(torch.ones(normalized_shape, device=device, dtype=dtype))
        if bias:
            self.bias = nn.Parameter(torch.zeros(normalized_shape, device=device, dtype=dtype))
        else:
            self.register_parameter("bias", None)

    def forward(self, x, residual=None):
        return layer_norm(x, self.weight, self.bias, self.eps, residual)

    def extra_repr(self) -> str:
        return f"{self.normalized_shape[0]}, eps={self.eps}, bias={self.bias is not None}"
