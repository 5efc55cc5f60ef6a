"""Self-attention over a packed projection (kernel K11, ``csrc/attn_kernels.hip``).

``attention_packed(qkv)`` takes the fused QKV projection output ``[B, S, 3, A, 64]`` (bf16, CUDA) and
returns the context ``[B, S, A*64]`` -- the layouts on both sides of BERT's attention, so nothing is
transposed or copied around the kernels.  Head dim 64, S in {128, 256, 384, 512}, optional key-padding lengths, no dropout;
anything else goes through ``F.scaled_dot_product_attention`` (also the oracle of the kernel tests).

``attention(q, k, v)`` (kernel K22, ``csrc/attn_general_kernels.hip``) is the general form: any lengths (one query token
included), head dims that are multiples of 8 to 128, fewer key than query heads, causal or with key lengths, strided
operands; bf16 on the GPU.  CPU tensors take :func:`attention_general_reference`.
"""
from __future__ import annotations

import ctypes
import math
import struct
import os

import torch
import torch.nn.functional as F

from . import hip

_declared = False
_ENABLED = os.environ.get("DTF_ATTN_KERNEL", "1") != "0"      # A/B switch


def _lib():
    global _declared
    lib = hip.lib()
    if not _declared:
        P, I, L, Fl = ctypes.c_void_p, ctypes.c_int, ctypes.c_int64, ctypes.c_float
        hip.declare("dtf_attn_fwd", [P, P, P, P, P, L, L, L, I, I, I, I, I, I, I, Fl, P, P])
        hip.declare("dtf_attn_bwd", [P, P, P, P, P, P, P, P, P, P, L, L, L, I, I, I, L, L, L, I, I, I, I, I, I, I, Fl, P, P])
        _declared = True
    return lib


def kernel_eligible(qkv):
    return (_ENABLED and qkv.is_cuda and qkv.dtype == torch.bfloat16 and qkv.dim() == 5 and qkv.shape[2] == 3
            and qkv.shape[4] == 64 and qkv.shape[1] in (128, 256, 384, 512) and qkv.is_contiguous())


def attn_fwd_packed(qkv, kv_len=None):
    """Raw forward: -> (ctx [B, S, A*64], lse [B, A, S] fp32 in the log2 domain)."""
    B, S, _, A, D = qkv.shape
    o = torch.empty(B, S, A * D, dtype=qkv.dtype, device=qkv.device)
    lse = torch.empty(B, A, S, dtype=torch.float32, device=qkv.device)
    base, esz = qkv.data_ptr(), 2
    rs, bs = 3 * A * D, S * 3 * A * D
    rc = _lib().dtf_attn_fwd(base, base + A * D * esz, base + 2 * A * D * esz, hip.ptr(o), hip.ptr(lse), bs, bs, bs,
                             rs, rs, rs, B, A, S, D, 1.0 / math.sqrt(D), hip.ptr(kv_len), hip.stream())
    hip.check(rc, "dtf_attn_fwd")
    return o, lse


def attn_bwd_packed(qkv, o, lse, do, kv_len=None):
    """Raw backward: -> dqkv [B, S, 3, A, 64] (every element written by the kernels)."""
    B, S, _, A, D = qkv.shape
    if not do.is_contiguous():
        do = do.contiguous()
    dqkv = torch.empty_like(qkv)
    dsum = torch.empty(B, A, S, dtype=torch.float32, device=qkv.device)
    base, gbase, esz = qkv.data_ptr(), dqkv.data_ptr(), 2
    rs, bs = 3 * A * D, S * 3 * A * D
    hd = A * D * esz
    rc = _lib().dtf_attn_bwd(base, base + hd, base + 2 * hd, hip.ptr(o), hip.ptr(do), hip.ptr(lse), hip.ptr(dsum),
                             gbase, gbase + hd, gbase + 2 * hd, bs, bs, bs, rs, rs, rs, bs, bs, bs, rs, rs, rs,
                             B, A, S, D, 1.0 / math.sqrt(D), hip.ptr(kv_len), hip.stream())
    hip.check(rc, "dtf_attn_bwd")
    return dqkv


class _AttentionPacked(torch.autograd.Function):
    @staticmethod
    def forward(ctx, qkv, kv_len):
        o, lse = attn_fwd_packed(qkv, kv_len)
        ctx.save_for_backward(qkv, o, lse, kv_len)
        return o

    @staticmethod
    def backward(ctx, do):
        qkv, o, lse, kv_len = ctx.saved_tensors
        return attn_bwd_packed(qkv, o, lse, do, kv_len), None


def attention_packed(qkv, kv_len=None):
    """``softmax(q k^T / sqrt(64)) v`` per head for the packed projection ``[B, S, 3, A, 64]`` -> ``[B, S, A*64]``.
    ``kv_len`` (int32 ``[B]``, optional): keys at positions >= kv_len[b] are padding and get no weight
    (BERT's attention mask is such a prefix mask); padded QUERY rows still produce (meaningless) output."""
    if kernel_eligible(qkv):
        if kv_len is not None:
            kv_len = kv_len.to(device=qkv.device, dtype=torch.int32).contiguous()
        return _AttentionPacked.apply(qkv, kv_len)
    return attention_reference(qkv, kv_len)


def attention_reference(qkv, kv_len=None):
    B, S, _, A, D = qkv.shape
    q, k, v = qkv.permute(2, 0, 3, 1, 4).unbind(0)
    mask = None
    if kv_len is not None:
        mask = (torch.arange(S, device=qkv.device)[None, :] < kv_len.to(qkv.device)[:, None])[:, None, None, :]
    return F.scaled_dot_product_attention(q, k, v, attn_mask=mask).transpose(1, 2).reshape(B, S, A * D)


# ---------------------------------------------------------------------------------------------------------------------
# K22: any lengths, grouped heads, causal
# ---------------------------------------------------------------------------------------------------------------------
_general = None


def _general_kernels():
    global _general
    if _general is None:
        C, P, L = ctypes.c_char_p, ctypes.c_void_p, ctypes.c_int64
        _general = (hip.declare("dtf_attn_general_fwd", [C, C, P]), hip.declare("dtf_attn_general_bwd", [C, C, P]),
                    hip.declare("dtf_attn_general_fwd_ws", [C], L), hip.declare("dtf_attn_general_bwd_ws", [C], L))
    return _general


_call = struct.Struct("<9qQ7if").pack              # AgCall of csrc/attn_general_kernels.hip
_fwd_tensors, _bwd_tensors = struct.Struct("<6Q").pack, struct.Struct("<10Q").pack


def _operand(t):
    """-> (t, its batch, token and head stride, 0 where there is one): as it is where the kernels can address it (dense head
    dimension, 16-B aligned rows, tokens less than 2^25 elements apart), else a contiguous copy."""
    B, S, H, D = t.shape
    b, s, h, d = t.stride()
    if B == 1:
        b = 0
    if S == 1:
        s = 0
    if H == 1:
        h = 0
    if d == 1 and s < 1 << 25 and not (b | s | h) & 7 and not t.data_ptr() & 15:
        return t, b, s, h
    return t.clone(memory_format=torch.contiguous_format), S * H * D, H * D, D


def _dense(t):
    return t if t.is_contiguous() and not t.data_ptr() & 15 else t.clone(memory_format=torch.contiguous_format)


def _general_operands(q, k, v, kv_len, causal, scale):
    """-> (q, k, v as the kernels read them, what the call is about)."""
    (q, *sq), (k, *sk), (v, *sv) = _operand(q), _operand(k), _operand(v)
    B, Sq, Hq, D = q.shape
    _, Sk, Hk, _ = k.shape
    return q, k, v, _call(*sq, *sk, *sv, hip.ptr(kv_len), B, Sq, Sk, Hq, Hk, D, causal, scale)


def _general_forward(q, k, v, kv_len, causal, scale):
    """-> (q, k, v as the kernels read them, out, log-sum-exp)."""
    q, k, v, how = _general_operands(q, k, v, kv_len, causal, scale)
    B, Sq, Hq, _ = q.shape
    o = torch.empty_like(q, memory_format=torch.contiguous_format)
    lse = q.new_empty((B, Hq, Sq), dtype=torch.float32)
    fwd, _, ws_floats, _ = _general_kernels()
    n = ws_floats(how)
    ws = lse.new_empty(n) if n else None
    rc = hip.launch(q, fwd, _fwd_tensors(q.data_ptr(), k.data_ptr(), v.data_ptr(), o.data_ptr(), lse.data_ptr(), hip.ptr(ws)), how)
    hip.check(rc, "dtf_attn_general_fwd")
    return q, k, v, o, lse


class _Attention(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, v, kv_len, causal, scale):
        q, k, v, o, lse = _general_forward(q, k, v, kv_len, causal, scale)
        ctx.save_for_backward(q, k, v, o, lse, hip.savable(kv_len))
        ctx.how = causal, scale
        return o

    @staticmethod
    @hip.first_order
    def backward(ctx, do):
        q, k, v, o, lse, kv_len = ctx.saved_tensors       # (hooks on saved tensors may bring them back in another layout)
        kv_len = None if kv_len is None else kv_len.contiguous()
        q, k, v, how = _general_operands(q, k, v, kv_len, *ctx.how)
        o, lse, do = _dense(o), _dense(lse), _dense(do)
        dq, dk = torch.empty_like(o), torch.empty_like(k, memory_format=torch.contiguous_format)
        dv = torch.empty_like(dk)
        _, bwd, _, ws_floats = _general_kernels()
        ws = lse.new_empty(ws_floats(how))
        rc = hip.launch(q, bwd, _bwd_tensors(q.data_ptr(), k.data_ptr(), v.data_ptr(), o.data_ptr(), do.data_ptr(), lse.data_ptr(),
                                             dq.data_ptr(), dk.data_ptr(), dv.data_ptr(), ws.data_ptr()), how)
        hip.check(rc, "dtf_attn_general_bwd")
        return dq, dk, dv, None, None, None


def _check_general(q, k, v, kv_len, scale):
    shape, keys, dtype, device = q.shape, k.shape, q.dtype, q.device
    if not len(shape) == len(keys) == v.dim() == 4:
        raise ValueError("attention: q, k and v are [B, S, heads, D], got %s, %s and %s" % (tuple(shape), tuple(keys), tuple(v.shape)))
    if k.dtype != dtype or v.dtype != dtype or k.device != device or v.device != device:
        raise ValueError("attention: q, k and v must share dtype and device")
    if not dtype.is_floating_point:
        raise TypeError("attention: q, k and v are floating-point tensors, got %s" % dtype)
    B, Sq, Hq, D = shape
    Bk, Sk, Hk, Dk = keys
    if keys != v.shape or Bk != B or Dk != D:
        raise ValueError("attention: q %s, k %s and v %s do not fit together" % (tuple(shape), tuple(keys), tuple(v.shape)))
    if 0 in shape or 0 in keys:
        raise ValueError("attention: no dimension may be empty, got q %s and k %s" % (tuple(shape), tuple(keys)))
    if Hq % Hk:
        raise ValueError("attention: %d query heads do not divide over %d key heads" % (Hq, Hk))
    if D % 8 or D > 128:
        raise ValueError("attention: the head dimension must be a multiple of 8 up to 128, got %d" % D)
    if Hq * D >= 1 << 25:
        raise ValueError("attention: %d heads of %d are too many" % (Hq, D))
    if Sq >= 1 << 30 or Sk >= 1 << 30:
        raise ValueError("attention: sequences are shorter than 2**30 tokens")
    if not 0 < scale < math.inf:
        raise ValueError("attention: scale must be positive and finite, got %r" % (scale,))
    if kv_len is not None and (kv_len.shape != (B,) or kv_len.is_floating_point() or kv_len.dtype == torch.bool):
        raise ValueError("attention: kv_len holds one integer for each of the %d sequences" % B)


def attention(q, k, v, causal=False, kv_len=None, scale=None):
    """``softmax(scale q k^T) v`` per head: ``q`` ``[B, Sq, Hq, D]``, ``k`` and ``v`` ``[B, Sk, Hk, D]`` -> ``[B, Sq, Hq, D]``;
    query head h reads key head ``h // (Hq / Hk)``, ``scale`` is ``1 / sqrt(D)`` by default.  ``causal``: query i sees the keys
    ``j <= i + Sk - Sq`` (the last query sees all).  ``kv_len`` (integers ``[B]``, values taken to ``[0, Sk]``): keys at or past
    it are padding and never read.  A query that sees no key gets zeros, and passes no gradient on.  (An infinity or NaN at a
    key that only causality hides may reach queries before it, as in any product with a probability of 0.)

    Scores, softmax statistics and sums are fp32; probabilities and their gradients are rounded to bf16 for the second products.
    Sums run in a fixed order (no atomics): calls of the same shapes give the same bits, and a sequence's do not depend on what
    the other sequences hold or how long they are.  They may depend on how many there are: long sums are split into as many parts
    as it takes to fill the card with the whole call."""
    scale = 1.0 / math.sqrt(max(1, q.shape[-1])) if scale is None else hip.number(scale, "attention: scale")
    _check_general(q, k, v, kv_len, scale)
    if not q.is_cuda:
        return attention_general_reference(q, k, v, causal, kv_len, scale)
    if q.dtype != torch.bfloat16:
        raise TypeError("attention: the GPU kernels take bfloat16, got %s" % q.dtype)
    if kv_len is not None:
        if kv_len.dtype != torch.int32:
            kv_len = kv_len.to(torch.int64).clamp(0, k.shape[1])
        kv_len = kv_len.to(device=q.device, dtype=torch.int32).contiguous()
    if not hip.recorded(q, k, v):
        return _general_forward(q, k, v, kv_len, int(bool(causal)), scale)[3]
    return _Attention.apply(q, k, v, kv_len, int(bool(causal)), scale)


def attention_general_reference(q, k, v, causal=False, kv_len=None, scale=None):
    """The definition in elementary operations (fp32, fp64 for fp64 operands)."""
    B, Sq, Hq, D = q.shape
    Sk, Hk = k.shape[1], k.shape[2]
    dt = torch.float64 if q.dtype == torch.float64 else torch.float32
    scale = 1.0 / math.sqrt(D) if scale is None else scale
    at = torch.arange(Sk, device=q.device)
    seen = torch.ones(B, 1, 1, Sk, dtype=torch.bool, device=q.device)
    if kv_len is not None:
        seen = (at < kv_len.to(q.device)[:, None])[:, None, None, :]
        pad = ~seen.view(B, Sk, 1, 1)
        k, v = k.masked_fill(pad, 0), v.masked_fill(pad, 0)               # whatever padding holds takes no part
    if causal:
        seen = seen & (at <= torch.arange(Sq, device=q.device)[:, None] + (Sk - Sq))
    qt, kt, vt = (t.to(dt).transpose(1, 2) for t in (q, k, v))
    kt, vt = (t.repeat_interleave(Hq // Hk, dim=1) for t in (kt, vt))
    s = (torch.matmul(qt, kt.transpose(2, 3).contiguous()) * scale).masked_fill(~seen, -math.inf)
    e = torch.exp(s - s.detach().amax(-1, keepdim=True).clamp_min(-1e30))
    z = e.sum(-1, keepdim=True)
    p = e / torch.where(z == 0, torch.ones_like(z), z)
    return torch.matmul(p, vt).transpose(1, 2).to(q.dtype).contiguous()
