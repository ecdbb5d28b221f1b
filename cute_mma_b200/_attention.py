"""Attention of the decoder that Prism layers stand in: whole prompts (``causal_attention``, differentiable) and single
tokens (``decode_attention``).

The reference's training model calls PyTorch's attention between its Prism layers (integration/model.py:95-117); here
it is the library's own kernels, so that queries, keys and values are read where the QKV layer's output holds them
(column ranges of one matrix) and sequences of different lengths are packed without padding.
"""
from __future__ import annotations

import ctypes
import math

import torch

from . import _functional as F
from . import _lib
from ._module import _plain_eager, _plain_grad, _refuse_tangents

_MOST_ROWS = (1 << 31) - 257   # (the kernels' row numbers, rounded up to whole tiles, are 32-bit)
_MOST_SEQUENCES = 1 << 20      # (packed)
_STRIDES8, _STRIDES9, _STRIDES12 = (ctypes.c_longlong * n for n in (8, 9, 12))


def _check_heads(q, k, v) -> None:
    for name, t in (("q", q), ("k", k), ("v", v)):
        if not t.is_cuda:
            raise ValueError(f"{name} must be a CUDA tensor, got device={t.device}")
        if t.dtype not in F._DTYPES:
            raise ValueError(f"{name} must be float16 or bfloat16, got dtype={t.dtype}")
    if not (q.dtype == k.dtype == v.dtype):
        raise ValueError(f"All tensors must have the same dtype, got q={q.dtype}, k={k.dtype}, v={v.dtype}")
    if not (q.device == k.device == v.device):
        raise ValueError("All tensors must be on the same CUDA device")
    if k.shape != v.shape:
        raise ValueError(f"k and v must have the same shape, got {tuple(k.shape)} and {tuple(v.shape)}")
    if q.shape[-1] != k.shape[-1]:
        raise ValueError(f"head_dim mismatch: q has {q.shape[-1]} but k has {k.shape[-1]}")
    d, hq, hkv = q.shape[-1], q.shape[-2], k.shape[-2]
    if d % 8 != 0 or not 8 <= d <= 128:
        raise ValueError(f"head_dim must be a multiple of 8 up to 128 for the sm_100a kernels, got {d}")
    if hkv < 1 or hq < 1 or hq % hkv != 0:
        raise ValueError(f"the heads of q ({hq}) must be a multiple of those of k and v ({hkv})")


def _check_scale(scale, head_dim) -> float:
    if scale is None:
        return head_dim ** -0.5
    scale = float(scale)
    if not (scale > 0.0 and math.isfinite(scale)):
        raise ValueError(f"scale must be positive and finite, got {scale}")
    return scale


def _check_prompt(q, k, v, cu_seqlens) -> None:
    if not (q.dim() == k.dim() == v.dim()) or q.dim() not in (3, 4):
        raise ValueError("q, k and v must be 3D (rows, heads, head_dim) or 4D (batch, rows, heads, head_dim), "
                         f"got {q.dim()}D, {k.dim()}D and {v.dim()}D")
    _check_heads(q, k, v)
    if q.shape[:-2] != k.shape[:-2]:
        raise ValueError(f"q and k must have the same rows, got {tuple(q.shape[:-2])} and {tuple(k.shape[:-2])}")
    if q.shape[:-2].numel() > _MOST_ROWS:
        raise ValueError(f"more than {_MOST_ROWS} rows")
    if cu_seqlens is None:
        return
    if q.dim() != 3:
        raise ValueError("cu_seqlens goes with packed (rows, heads, head_dim) tensors")
    if (cu_seqlens.dtype != torch.int32 or cu_seqlens.dim() != 1 or cu_seqlens.numel() < 2
            or not cu_seqlens.is_contiguous() or cu_seqlens.device != q.device):
        raise ValueError("cu_seqlens must be a contiguous int32 tensor (sequences + 1,) on the device of q")
    if cu_seqlens.numel() - 1 > _MOST_SEQUENCES:
        raise ValueError(f"more than {_MOST_SEQUENCES} packed sequences")


def _steps(t):
    """(batch, row, head) strides of a (rows, heads, dim) or (batch, rows, heads, dim) tensor; a single entry has none,
    and stands as 8."""
    n, s = t.shape, t.stride()
    if len(s) == 3:
        return 8, s[0] if n[0] != 1 else 8, s[1] if n[1] != 1 else 8
    return s[0] if n[0] != 1 else 8, s[1] if n[1] != 1 else 8, s[2] if n[2] != 1 else 8


def _tma_rows(t):
    """t as the kernels can read it: features contiguous, 16-byte steps between rows, heads and batches (a copy where
    that is not so, e.g. of an expanded tensor), and its (batch, row, head) strides."""
    s = b, r, h = _steps(t)
    if t.stride(-1) != 1 or b <= 0 or r <= 0 or h <= 0 or (b | r | h) & 7 or t.data_ptr() & 15:
        t = t.contiguous()
        if t.data_ptr() & 15:
            t = t.clone()
        s = _steps(t)
    return t, s


def _whole(t):
    """A saved tensor as it was saved: contiguous from a 16-byte boundary (saved-tensor hooks may have handed back another layout)."""
    t = t.contiguous()
    return t.clone() if t.data_ptr() & 15 else t


def _attn_forward(q, k, v, cu_seqlens, scale, train):
    """(o, lse, o_low), the latter two for the backward and None without it: the rows' log-sums, and what rounding o took
    (the backward needs do . o of every row more exactly than o as rounded gives it).  q, k, v as checked."""
    hq, d = q.shape[-2:]
    o = q.new_empty(q.shape)   # (contiguous; less host time than torch.empty with its keywords)
    rows = q.shape[:-2].numel()
    lse = q.new_empty((hq, rows), dtype=torch.float32) if train else None
    low = q.new_empty(q.shape, dtype=torch.uint8) if train else None
    if rows == 0:
        return o, lse, low
    q, sq = _tma_rows(q)
    k, sk = _tma_rows(k)
    v, sv = _tma_rows(v)
    n, length = _sequences(q, cu_seqlens)
    with F._device_scope(q.device):
        ws = F._workspace.get(q.device, 256)
        _lib.check(_lib.lib().prism_attn_fwd(
            q.data_ptr(), k.data_ptr(), v.data_ptr(), o.data_ptr(), F._ptr(lse), F._ptr(low), F._ptr(cu_seqlens), n, length, rows,
            hq, k.shape[-2], d, F._DTYPES[q.dtype], scale, _STRIDES9(*sq, *sk, *sv), ws.data_ptr(), ws.numel(),
            F._raw_stream(q.device)))
    return o, lse, low


def _sequences(q, cu_seqlens):
    """(number of sequences, rows of each; rows 0 where cu_seqlens holds them)."""
    if cu_seqlens is not None:
        return cu_seqlens.numel() - 1, 0
    return (q.shape[0], q.shape[1]) if q.dim() == 4 else (1, q.shape[0])


def _attn_backward(d_o, q, k, v, o, lse, low, cu_seqlens, scale, need_dq=True, need_dkv=True):
    """(dq, dk, dv), None for what is not asked for."""
    hq, d = q.shape[-2:]
    rows = q.shape[:-2].numel()
    dq = q.new_empty(q.shape) if need_dq else None
    dk, dv = (k.new_empty(k.shape) if need_dkv else None for _ in range(2))
    if rows == 0 or not (need_dq or need_dkv):
        return dq, dk, dv
    o, lse, low = _whole(o), _whole(lse), _whole(low)
    cu_seqlens = None if cu_seqlens is None else _whole(cu_seqlens)
    d_o, sdo = _tma_rows(d_o)
    q, sq = _tma_rows(q)
    k, sk = _tma_rows(k)
    v, sv = _tma_rows(v)
    n, length = _sequences(q, cu_seqlens)
    with F._device_scope(q.device):
        delta = lse.new_empty(lse.numel() + 2)   # (and the largest norms of d_o and v behind it)
        ws = F._workspace.get(q.device, 256)
        _lib.check(_lib.lib().prism_attn_bwd_scaled(
            d_o.data_ptr(), q.data_ptr(), k.data_ptr(), v.data_ptr(), o.data_ptr(), lse.data_ptr(), F._ptr(low), F._ptr(dq),
            F._ptr(dk), F._ptr(dv), delta.data_ptr(), delta.data_ptr() + 4 * lse.numel(), F._ptr(cu_seqlens), n, length, rows,
            hq, k.shape[-2], d, F._DTYPES[q.dtype], scale, _STRIDES12(*sq, *sk, *sv, *sdo), ws.data_ptr(), ws.numel(), F._raw_stream(q.device)))
    return dq, dk, dv


# ---------------------------------------------------------------------------
# custom ops (traced, compiled and transformed calls) and the eager autograd node, as for the layer itself
# ---------------------------------------------------------------------------
@torch.library.custom_op("prism_b200::causal_attention", mutates_args=())
def _attention_op(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, cu_seqlens: torch.Tensor | None,
                  scale: float) -> tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
    return _attn_forward(q, k, v, cu_seqlens, scale, True)


@_attention_op.register_fake
def _(q, k, v, cu_seqlens, scale):
    return (q.new_empty(q.shape), q.new_empty((q.shape[-2], q.shape[:-2].numel()), dtype=torch.float32),
            q.new_empty(q.shape, dtype=torch.uint8))


@torch.library.custom_op("prism_b200::causal_attention_backward", mutates_args=())
def _attention_bwd_op(d_o: torch.Tensor, q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, o: torch.Tensor,
                      lse: torch.Tensor, low: torch.Tensor, cu_seqlens: torch.Tensor | None, scale: float
                      ) -> tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
    return _attn_backward(d_o, q, k, v, o, lse, low, cu_seqlens, scale)


@_attention_bwd_op.register_fake
def _(d_o, q, k, v, o, lse, low, cu_seqlens, scale):
    return q.new_empty(q.shape), k.new_empty(k.shape), v.new_empty(v.shape)


def _attention_setup(ctx, inputs, output):
    q, k, v, cu_seqlens, scale = inputs
    ctx.save_for_backward(q, k, v, *output, cu_seqlens)
    ctx.scale = scale
    ctx.mark_non_differentiable(*output[1:])


def _attention_grad(ctx, d_o, _d_lse, _d_low):
    return *_attention_bwd_op(d_o, *ctx.saved_tensors, ctx.scale), None, None


_attention_op.register_autograd(_attention_grad, setup_context=_attention_setup)


class _AttentionFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, v, cu_seqlens, scale):
        o, lse, low = _attn_forward(q, k, v, cu_seqlens, scale, True)
        ctx.save_for_backward(q, k, v, o, lse, low, cu_seqlens)
        ctx.scale = scale
        return o

    @staticmethod
    def backward(ctx, d_o):
        # (the decorator costs 14 us of host time, and only a backward that is itself recorded needs it)
        return (_AttentionFn._recorded if torch.is_grad_enabled() else _AttentionFn._grads)(ctx, d_o)

    @staticmethod
    def _grads(ctx, d_o):
        q, k, v, o, lse, low, cu_seqlens = ctx.saved_tensors
        if _plain_eager(d_o, q, k, v, o, lse, low) and _plain_grad(d_o):
            need = ctx.needs_input_grad
            dq, dk, dv = _attn_backward(d_o, q, k, v, o, lse, low, cu_seqlens, ctx.scale, need[0], need[1] or need[2])
            return dq, dk if need[1] else None, dv if need[2] else None, None, None
        return *_attention_bwd_op(d_o, q, k, v, o, lse, low, cu_seqlens, ctx.scale), None, None

    _recorded = staticmethod(torch.autograd.function.once_differentiable(lambda ctx, d_o: _AttentionFn._grads(ctx, d_o)))


def causal_attention(q, k, v, cu_seqlens=None, scale=None):
    """``softmax(scale * q @ k^T, keys up to the query's own row) @ v`` for every head of every sequence; differentiable.

    Packed: q ``(rows, heads, head_dim)``, k and v ``(rows, kv_heads, head_dim)`` with ``cu_seqlens``
    ``(sequences + 1,)`` int32 on the same device, sequence i in rows ``cu_seqlens[i]`` up to ``cu_seqlens[i + 1]``
    (ascending; lengths of zero are allowed; up to 2^20 sequences; never read by the host).  Rows that belong to no sequence are zeros in the
    output and in the gradients.  Without ``cu_seqlens`` the tensors are one sequence, or, 4D
    ``(batch, rows, heads, head_dim)``, a batch of them.  float16 or bfloat16; ``heads`` a multiple of ``kv_heads``
    (neighbouring query heads share a key head); ``head_dim`` a multiple of 8 up to 128; ``scale`` positive, by default
    ``head_dim ** -0.5``.  Column ranges of one QKV matrix are read in place.
    Rounded to the inputs' type on the way are the probabilities, before they meet ``v`` (and ``do``), and in the backward their
    gradients, before they meet ``k`` and ``q``, in fp16 with factors that keep them in its range; all else is summed in fp32.
    Infinities and NaN reach the rows that see them.  In the gradients they also reach rows of the same 128 rows of their sequence.
    """
    _check_prompt(q, k, v, cu_seqlens)
    scale = _check_scale(scale, q.shape[-1])
    if _plain_eager(q, k, v, cu_seqlens):
        if torch.is_grad_enabled() and (q.requires_grad or k.requires_grad or v.requires_grad):
            return _AttentionFn.apply(q, k, v, cu_seqlens, scale)
        return _attn_forward(q, k, v, cu_seqlens, scale, False)[0]
    _refuse_tangents("causal_attention", q, k, v)
    return _attention_op(q, k, v, cu_seqlens, scale)[0]


# ---------------------------------------------------------------------------
# single tokens
# ---------------------------------------------------------------------------
def _check_decode(q, k, v, lengths) -> None:
    if q.dim() != 3 or k.dim() != 4 or v.dim() != 4:
        raise ValueError("q must be 3D (sequences, heads, head_dim), k and v 4D (sequences, room, kv_heads, head_dim), "
                         f"got {q.dim()}D, {k.dim()}D and {v.dim()}D")
    _check_heads(q, k, v)
    if q.shape[0] != k.shape[0]:
        raise ValueError(f"q and k must have the same sequences, got {q.shape[0]} and {k.shape[0]}")
    if k.shape[1] > _MOST_ROWS or q.shape[0] * q.shape[1] > _MOST_ROWS:
        raise ValueError(f"more than {_MOST_ROWS} rows")
    if (lengths.dtype != torch.int32 or lengths.shape != (q.shape[0],) or not lengths.is_contiguous()
            or lengths.device != q.device):
        raise ValueError("lengths must be a contiguous int32 tensor (sequences,) on the device of q")
    for name, t in (("k", k), ("v", v)):
        # (a copy of a whole cache per token is not what a caller wants)
        x, y, z = _steps(t)
        if t.numel() and (t.stride(-1) != 1 or (x | y | z) & 7):
            raise ValueError(f"{name} must have contiguous features and strides that are multiples of 8 elements")
    if torch.is_grad_enabled() and (q.requires_grad or k.requires_grad or v.requires_grad):
        raise ValueError("decode_attention has no backward pass; call it under torch.no_grad(), or causal_attention")


@torch.library.custom_op("prism_b200::decode_attention", mutates_args=())
def _decode_op(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, lengths: torch.Tensor, scale: float) -> torch.Tensor:
    return _decode(q, k, v, lengths, scale)


@_decode_op.register_fake
def _(q, k, v, lengths, scale):
    return q.new_empty(q.shape)


_scratch_bytes: dict = {}   # (head_dim, device): prism_attn_decode_scratch_bytes there


def _decode(q, k, v, lengths, scale):
    o = q.new_empty(q.shape)
    b, hq, d = q.shape
    if b == 0:
        return o
    for name, t in (("k", k), ("v", v)):
        if t.data_ptr() & 15:
            raise ValueError(f"{name} must start on a 16-byte boundary")
    q, (_, sb, sh) = _tma_rows(q)
    L = _lib.lib()
    with F._device_scope(q.device):
        key = d, q.device.index
        nbytes = _scratch_bytes.get(key)
        if nbytes is None:
            nbytes = _scratch_bytes[key] = L.prism_attn_decode_scratch_bytes(d)
        scratch = q.new_empty(nbytes >> 1)
        _lib.check(L.prism_attn_decode(
            q.data_ptr(), k.data_ptr(), v.data_ptr(), o.data_ptr(), lengths.data_ptr(), b, k.shape[1], hq, k.shape[2], d,
            F._DTYPES[q.dtype], scale, _STRIDES8(sb, sh, *_steps(k), *_steps(v)), scratch.data_ptr(), nbytes,
            F._raw_stream(q.device)))
    return o


def decode_attention(q, k, v, lengths, scale=None):
    """Attention of the newest token of every sequence over that sequence's keys and values, without gradients.

    q ``(sequences, heads, head_dim)``; k, v ``(sequences, room, kv_heads, head_dim)`` of any strides with contiguous
    features and 16-byte steps (a slice of a larger cache is read in place); ``lengths`` ``(sequences,)`` int32 on the
    same device: the rows of k and v that count, the newest token's own among them; nothing behind them is read, so
    that it may hold anything.  A length of 0 gives a row of zeros; lengths are taken into ``[0, room]`` and never read by
    the host.  Types, heads and ``scale`` as for ``causal_attention``.
    """
    _check_decode(q, k, v, lengths)
    scale = _check_scale(scale, q.shape[-1])
    if _plain_eager(q, k, v, lengths):
        return _decode(q, k, v, lengths, scale)
    _refuse_tangents("decode_attention", q, k, v)
    return _decode_op(q, k, v, lengths, scale)
