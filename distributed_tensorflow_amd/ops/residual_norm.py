"""The boundary between two transformer blocks in one pass (kernel K24, ``csrc/residual_norm_kernels.hip``):

    n = post(h);   r = x + scale * gate * n;   y = pre(r)

``x`` is the residual stream, ``h`` a block's output, ``post`` an optional norm behind the block, ``gate`` an optional factor
per element, per sequence or per channel, ``pre`` the norm in front of the next block.  Norms are RMS norms or layer norms.
bf16 or fp32, any width to 16384; parameters in the activations' type or fp32.  CPU tensors take
:func:`residual_norm_reference`, the oracle of the kernel tests.
"""
from __future__ import annotations

import ctypes
import math
import struct

import torch
import torch.nn as nn

from . import hip

MAX_WIDTH = 16384
_fns = None


def _kernels():
    global _fns
    if _fns is None:
        C, P, L = ctypes.c_char_p, ctypes.c_void_p, ctypes.c_int64
        _fns = (hip.declare("dtf_residual_norm_fwd", [C, C, P]), hip.declare("dtf_residual_norm_bwd", [C, C, P]),
                hip.declare("dtf_residual_norm_ws", [C, L, ctypes.c_int], L))
    return _fns


_call = struct.Struct("<2q4i2f").pack              # RnCall of csrc/residual_norm_kernels.hip
_fwd_tensors, _bwd_tensors = struct.Struct("<10Q").pack, struct.Struct("<17Q").pack


def _normed(v, weight, bias, kind, eps):
    if kind == "layer":
        v = v - v.mean(-1, keepdim=True)
    v = v / torch.sqrt((v * v).mean(-1, keepdim=True) + eps) * weight.float()
    return v if bias is None else v + bias.float()


def residual_norm_reference(x, h, weight, bias=None, *, gate=None, scale=1.0, post_weight=None, post_bias=None, kind="rms",
                            eps=1e-6):
    """The definition in elementary fp32 operations, rounded once at the end."""
    n = h.float() if post_weight is None else _normed(h.float(), post_weight, post_bias, kind, eps)
    r = x.float() + scale * (n if gate is None else n * gate.float())
    return _normed(r, weight, bias, kind, eps).to(x.dtype), r.to(x.dtype)


def _rows_per_gate(x, gate):
    """Rows of x that share a row of the gate: the gate's leading dimensions are x's up to some axis and 1 from there on."""
    if gate.shape == x.shape:
        return 1
    shape = (1,) * (x.dim() - gate.dim()) + tuple(gate.shape)
    if len(shape) == x.dim() and shape[-1] == x.shape[-1]:
        lead = tuple(x.shape[:-1])
        for cut in range(len(lead), -1, -1):
            if shape[:-1] == lead[:cut] + (1,) * (len(lead) - cut):
                rows = 1
                for n in lead[cut:]:
                    rows *= n
                return rows
    raise ValueError("residual_norm: a gate for x %s is x's own shape, or that with 1 for its last leading dimensions (one row a "
                     "sequence), or [%d]; got %s" % (tuple(x.shape), x.shape[-1], tuple(gate.shape)))


def _checked_eps(eps):
    eps = hip.number(eps, "residual_norm: eps")
    if not 0 <= eps < math.inf:
        raise ValueError("residual_norm: eps must be finite and not negative, got %r" % eps)
    return eps


def _checked(x, h, weight, bias, gate, post_weight, post_bias, kind):
    if kind not in ("rms", "layer"):
        raise ValueError("residual_norm: kind is 'rms' or 'layer', got %r" % (kind,))
    shape, dtype, device = x.shape, x.dtype, x.device
    hip.dt(x)
    if not shape or 0 in shape or shape[-1] > MAX_WIDTH:
        raise ValueError("residual_norm: x is [..., H] with 1 <= H <= %d and at least one row, got %s" % (MAX_WIDTH, tuple(shape)))
    if h is not None and (h.shape != shape or h.dtype != dtype or h.device != device):
        raise ValueError("residual_norm: h must match x in shape, dtype and device")
    if gate is not None and (gate.dtype != dtype or gate.device != device):
        raise ValueError("residual_norm: the gate must match x in dtype and device")
    if post_bias is not None and post_weight is None:
        raise ValueError("residual_norm: post_bias without post_weight")
    if kind == "rms" and (bias is not None or post_bias is not None):
        raise ValueError("residual_norm: an RMS norm has no bias")
    width, wdt = shape[-1:], weight.dtype
    for p in (weight, bias, post_weight, post_bias):
        if p is None:
            continue
        if p.shape != width or p.device != device:
            raise ValueError("residual_norm: parameters are [%d] on x's device, got %s" % (shape[-1], tuple(p.shape)))
        if p.dtype != wdt or (wdt != dtype and wdt != torch.float32):
            raise ValueError("residual_norm: parameters share one dtype, x's or float32")
    return None if gate is None else _rows_per_gate(x, gate)


def _dense(t):
    return t if t is None or t.is_contiguous() else t.contiguous()


def _like(t):
    return None if t is None else torch.empty_like(t)


def _forward(x, h, weight, bias, gate, post_weight, post_bias, rpg, scale, layer, eps):
    """-> (y, r, the operands as the kernels read them and the statistics, what the call is about)."""
    x, h, weight, bias, gate, post_weight, post_bias = [
        t if t is None or t.is_contiguous() else t.contiguous() for t in (x, h, weight, bias, gate, post_weight, post_bias)]
    H = x.shape[-1]
    M = x.numel() // H
    y, r = torch.empty_like(x), _like(h)
    stats = x.new_empty(4 * M, dtype=torch.float32)
    how = _call(M, rpg, hip.dt(x), hip.dt(weight), layer, H, scale, eps)
    rc = hip.launch(x, _kernels()[0], _fwd_tensors(
        x.data_ptr(), hip.ptr(h), hip.ptr(gate), weight.data_ptr(), hip.ptr(bias), hip.ptr(post_weight), hip.ptr(post_bias),
        y.data_ptr(), hip.ptr(r), stats.data_ptr()), how)
    hip.check(rc, "dtf_residual_norm_fwd")
    return y, r, (x, h, weight, bias, gate, post_weight, post_bias, stats), (how, M, rpg, scale)


class _ResidualNorm(torch.autograd.Function):
    @staticmethod
    def forward(ctx, *args):
        y, r, operands, ctx.how = _forward(*args)
        ctx.set_materialize_grads(False)
        ctx.save_for_backward(*operands)
        return y, r

    @staticmethod
    @hip.first_order
    def backward(ctx, dy, dr):
        if dy is None and dr is None:
            return (None,) * 11
        x, h, weight, bias, gate, post_weight, post_bias, stats = map(_dense, ctx.saved_tensors)
        how, M, rpg, scale = ctx.how
        dy, dr = _dense(dy), _dense(dr)
        dx = torch.empty_like(x)
        same = post_weight is None and gate is None and scale == 1.0      # then dh = dx, written once
        dh = None if same else _like(h)
        dw, db, dgate, dpw, dpb = _like(weight), _like(bias), _like(gate), _like(post_weight), _like(post_bias)
        groups = M // rpg if gate is not None and rpg > 1 else 0          # rows of a gate that is shared
        narr = 1 + (bias is not None) + (post_weight is not None) + (post_bias is not None) + (groups > 0)
        _, bwd, ws_floats = _kernels()
        ws = stats.new_empty(ws_floats(how, groups or 1, narr))
        rc = hip.launch(x, bwd, _bwd_tensors(
            x.data_ptr(), hip.ptr(h), hip.ptr(gate), weight.data_ptr(), hip.ptr(post_weight), hip.ptr(post_bias), stats.data_ptr(),
            hip.ptr(dy), hip.ptr(dr), dx.data_ptr(), hip.ptr(dh), hip.ptr(dgate), dw.data_ptr(), hip.ptr(db), hip.ptr(dpw),
            hip.ptr(dpb), ws.data_ptr()), how)
        hip.check(rc, "dtf_residual_norm_bwd")
        return dx, dx if same and h is not None else dh, dw, db, dgate, dpw, dpb, None, None, None, None


def residual_norm(x, h, weight, bias=None, *, gate=None, scale=1.0, post_weight=None, post_bias=None, kind="rms", eps=1e-6):
    """-> (y, r): ``r = x + scale * gate * post(h)`` and ``y = pre(r)``.  ``x``, ``h`` ``[..., H]``; ``weight`` / ``bias`` are
    pre's, ``post_weight`` / ``post_bias`` post's (without ``post_weight``, h itself is added).  ``gate``: x's shape, or
    ``[B, 1, H]`` (one row a sequence), or ``[H]``; its gradient is summed over the rows that share it.  ``kind``: ``"rms"``, or
    ``"layer"`` (biases optional).  y is the norm of r before r is rounded to x's type."""
    rpg = _checked(x, h, weight, bias, gate, post_weight, post_bias, kind)
    if h is None:
        raise ValueError("residual_norm: h is missing (rms_norm has no residual)")
    scale, eps = hip.number(scale, "residual_norm: scale"), _checked_eps(eps)
    if not x.is_cuda:
        return residual_norm_reference(x, h, weight, bias, gate=gate, scale=scale, post_weight=post_weight, post_bias=post_bias,
                                       kind=kind, eps=eps)
    args = x, h, weight, bias, gate, post_weight, post_bias, rpg or 1, scale, int(kind == "layer"), eps
    return _ResidualNorm.apply(*args) if hip.recorded(*args[:7]) else _forward(*args)[:2]


def rms_norm(x, weight, eps=1e-6):
    """``x / sqrt(mean(x^2) + eps) * weight`` over the last dimension: the norm in front of a first block."""
    _checked(x, None, weight, None, None, None, None, "rms")
    eps = _checked_eps(eps)
    if not x.is_cuda:
        return _normed(x.float(), weight, None, "rms", eps).to(x.dtype)
    args = x, None, weight, None, None, None, None, 1, 1.0, 0, eps
    return (_ResidualNorm.apply(*args) if hip.recorded(x, weight) else _forward(*args))[0]


class FusedRMSNorm(nn.Module):
    """RMS norm over the last dimension.  ``norm(x)``, or ``norm(x, h, ...)`` -> (y, r) for the boundary between two blocks."""

    def __init__(self, hidden, eps=1e-6):
        super().__init__()
        self.weight = nn.Parameter(torch.ones(hidden))
        self.eps = eps

    def forward(self, x, h=None, **kw):
        if h is None:
            return rms_norm(x, self.weight, self.eps)
        return residual_norm(x, h, self.weight, eps=self.eps, **kw)
