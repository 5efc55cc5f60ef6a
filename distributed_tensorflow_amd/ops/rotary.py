"""Rotary positions (kernel K23, ``csrc/rotary_kernels.hip``).

``rotary(q, k, inv_freq, positions)`` turns pairs of the first ``2 * len(inv_freq)`` elements of every head by the angle
``position * inv_freq[pair]``; the rest of the head passes through.  ``rotary_frequencies`` makes ``inv_freq`` -- plain, or
scaled for contexts longer than the trained one.  bf16 or fp32 operands, any strides with a dense head dimension (slices of
a packed projection are read in place); CPU tensors take :func:`rotary_reference`, the oracle of the kernel tests.
"""
from __future__ import annotations

import ctypes
import math
import operator
import struct

import torch

from . import hip

_fn = None


def _kernel():
    global _fn
    if _fn is None:
        _fn = hip.declare("dtf_rotary", [ctypes.c_char_p, ctypes.c_void_p])
    return _fn


def rotary_frequencies(dim, base=10000.0, scaling="none", factor=1.0, original_length=None, beta_fast=32.0, beta_slow=1.0,
                       device=None):
    """-> (``inv_freq`` fp64 ``[dim / 2]``, amplitude).  ``scaling`` for contexts ``factor`` times the trained length:

    * ``"linear"``: every frequency / factor (positions interpolated);
    * ``"ntk"``: the base grows to ``base * factor ** (dim / (dim - 2))``, so that the slowest pair is stretched by
      ``factor`` and the fastest not at all;
    * ``"by_parts"``: pairs that make more than ``beta_fast`` turns in ``original_length`` tokens keep their frequency, those
      under ``beta_slow`` turns get frequency / factor, a linear ramp between; amplitude ``0.1 ln(factor) + 1``."""
    if dim <= 0 or dim % 2:
        raise ValueError("rotary: dim must be even and positive, got %d" % dim)
    if not base > 0 or not factor > 0:
        raise ValueError("rotary: base and factor must be positive")
    j = torch.arange(0, dim, 2, dtype=torch.float64) / dim
    amplitude = 1.0
    if scaling == "ntk":
        f = (base * factor ** (dim / (dim - 2)) if dim > 2 else base) ** -j
    elif scaling in ("none", "linear", "by_parts"):
        f = float(base) ** -j
        if scaling == "linear":
            f = f / factor
        elif scaling == "by_parts":
            if not original_length or not beta_fast > beta_slow:
                raise ValueError("rotary: by_parts needs original_length, and beta_fast > beta_slow")
            turns = original_length * f / (2 * math.pi)
            keep = ((turns - beta_slow) / (beta_fast - beta_slow)).clamp(0, 1)
            f = f * keep + f / factor * (1 - keep)
            amplitude = 0.1 * math.log(factor) + 1.0 if factor > 1 else 1.0
    else:
        raise ValueError("rotary: unknown scaling %r (none, linear, ntk, by_parts)" % (scaling,))
    return f.to(device=device), amplitude


def _checked(q, k, inv_freq, positions):
    shape, dtype, device = q.shape, q.dtype, q.device
    if len(shape) != 4 or (k is not None and k.dim() != 4):
        raise ValueError("rotary: q and k are [B, S, heads, D], got %s" % ", ".join(str(tuple(t.shape)) for t in (q, k) if t is not None))
    hip.dt(q)
    B, S, _, D = shape
    if k is not None:
        if k.dtype != dtype or k.device != device:
            raise ValueError("rotary: q and k must share dtype and device")
        Bk, Sk, _, Dk = k.shape
        if Bk != B or Sk != S or Dk != D:
            raise ValueError("rotary: q %s and k %s differ in more than their heads" % (tuple(shape), tuple(k.shape)))
    if D % 2:
        raise ValueError("rotary: the head dimension must be even, got %d" % D)
    if inv_freq.dim() != 1 or inv_freq.dtype != torch.float64 or not inv_freq.is_contiguous() or inv_freq.device != device:
        raise ValueError("rotary: inv_freq is a contiguous float64 vector on the operands' device (rotary_frequencies)")
    if inv_freq.requires_grad:
        raise ValueError("rotary: inv_freq gets no gradient (pass inv_freq.detach())")
    m = inv_freq.numel()
    if not 0 < 2 * m <= D or m > 1024:
        raise ValueError("rotary: %d pairs do not fit a head of %d" % (m, D))
    if positions is not None:
        if positions.dtype not in (torch.int64, torch.int32) or positions.device != device:
            raise ValueError("rotary: positions are int32 / int64 on the operands' device")
        if positions.shape not in ((B, S), (S,), (1, S)):
            raise ValueError("rotary: positions are [S] or [B, S], got %s for B=%d S=%d" % (tuple(positions.shape), B, S))


def _turn(x, cos, sin, interleaved):
    d = 2 * cos.shape[-1]
    a, b = (x[..., 0:d:2], x[..., 1:d:2]) if interleaved else (x[..., :d // 2], x[..., d // 2:d])
    ya, yb = a * cos - b * sin, a * sin + b * cos
    y = torch.stack([ya, yb], -1).flatten(-2) if interleaved else torch.cat([ya, yb], -1)
    return torch.cat([y, x[..., d:]], -1)


def rotary_reference(q, k, inv_freq, positions=None, *, interleaved=False, amplitude=1.0, offset=0):
    """The definition in elementary operations (angles in 64 bits, products in fp32)."""
    if positions is None:
        positions = torch.arange(q.shape[1], device=q.device) + offset
    angle = (positions.double().reshape(-1, q.shape[1], 1) * inv_freq).unsqueeze(2)
    cos, sin = (angle.cos() * amplitude).float(), (angle.sin() * amplitude).float()
    return tuple(None if t is None else _turn(t.float(), cos, sin, interleaved).to(t.dtype) for t in (q, k))


_call = struct.Struct("<6Q9q9i2f4x").pack          # RoCall of csrc/rotary_kernels.hip


def _operand(t):
    """-> (t with a dense head dimension, its batch, token and head stride)."""
    if t.stride(3) != 1:
        t = t.contiguous()
    return t, t.stride()[:3]


def _launch(q, k, inv_freq, positions, interleaved, amplitude, offset, sign):
    q, sq = _operand(q)
    B, S, Hq, D = q.shape
    qo = torch.empty_like(q, memory_format=torch.contiguous_format)
    if k is None:
        k_at, ko, ko_at, Hk, sk = 0, None, 0, 0, (0, 0, 0)
    else:
        k, sk = _operand(k)
        ko = torch.empty_like(k, memory_format=torch.contiguous_format)
        k_at, ko_at, Hk = k.data_ptr(), ko.data_ptr(), k.shape[2]
    p_at = p_64 = p_bs = p_ss = 0
    if positions is not None:
        p_at, p_64 = positions.data_ptr(), int(positions.dtype == torch.int64)
        *p_bs, p_ss = positions.stride()
        p_bs = p_bs[0] if p_bs and positions.shape[0] > 1 else 0
    rc = hip.launch(q, _kernel(), _call(q.data_ptr(), k_at, qo.data_ptr(), ko_at, p_at, inv_freq.data_ptr(), *sq, *sk, p_bs, p_ss,
                                        offset, hip.dt(q), p_64, B, S, Hq, Hk, D, inv_freq.numel(), interleaved, amplitude, sign))
    hip.check(rc, "dtf_rotary")
    return qo, ko


class _Rotary(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, inv_freq, positions, interleaved, amplitude, offset):
        ctx.save_for_backward(hip.savable(inv_freq), hip.savable(positions))
        ctx.how = interleaved, amplitude, offset
        return _launch(q, k, inv_freq, positions, interleaved, amplitude, offset, 1.0)

    @staticmethod
    @hip.first_order
    def backward(ctx, dq, dk):
        inv_freq, positions = ctx.saved_tensors
        inv_freq = inv_freq.contiguous()                                  # (hooks on saved tensors may have changed that)
        # the transpose of a rotation is the rotation by the negative angle
        gq, gk = _launch(dq, dk, inv_freq, positions, *ctx.how, -1.0)
        return gq, gk, None, None, None, None, None


def rotary(q, k, inv_freq, positions=None, *, interleaved=False, amplitude=1.0, offset=0):
    """-> (q, k) turned to their positions, contiguous, in their dtype.  ``q`` ``[B, S, Hq, D]``, ``k`` ``[B, S, Hk, D]`` or
    ``None``; ``positions`` int32 / int64 ``[S]`` or ``[B, S]`` (default ``offset + arange(S)``); ``interleaved``: pairs are
    neighbours ``(x[2j], x[2j+1])`` instead of the two halves ``(x[j], x[j + m])``.  Gradients flow to q and k."""
    _checked(q, k, inv_freq, positions)
    interleaved, amplitude, offset = int(bool(interleaved)), hip.number(amplitude, "rotary: amplitude"), operator.index(offset)
    if offset and (positions is not None or abs(offset) > 1 << 52):
        raise ValueError("rotary: offset goes with the default positions, and to 2**52 either way")
    if not q.is_cuda:
        return rotary_reference(q, k, inv_freq, positions, interleaved=interleaved, amplitude=amplitude, offset=offset)
    if q.numel() == 0 or (k is not None and k.numel() == 0):
        raise ValueError("rotary: q and k must hold at least one element")
    if not hip.recorded(q, k):
        return _launch(q, k, inv_freq, positions, interleaved, amplitude, offset, 1.0)
    return _Rotary.apply(q, k, inv_freq, positions, interleaved, amplitude, offset)
