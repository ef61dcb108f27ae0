"""Attention of queries over an encoder's states of another length (csrc/cross_attn.hip): the clouds of a batch side by side in the
packed layout of the point ops (one cumulative `offset` per cloud) or padded with a mask, shared key heads, head widths up to 128, one
query or thousands.  Stands beside `small_attn.small_attention`, which takes padded (B, L, E) tensors with heads of 64.
"""
import math

import torch
from torch.autograd import Function
from torch.autograd.function import once_differentiable

from .. import _graphs, _lib
from ..pointops import _common
from .._lib import raw_stream as _raw_stream

MAX_HEAD_DIM = 128


def _fit(t, group=1):
    """(t, (batch, row, head) strides in elements, 0 where there is one entry only); t a contiguous copy where its strides or address do
    not fit the kernels' 16-byte accesses, or rows (and the `group` heads of a key head) lie too far apart for offsets of 32 bits in a tile."""
    *st, last = t.stride()
    if not _fits(t, st, last, group):
        st = [s if n > 1 else 0 for s, n in zip(st, t.shape)]
        if not _fits(t, st, last, group):
            t = t.clone(memory_format=torch.contiguous_format)
            st = t.stride()[:-1]
    return t, (st if len(st) == 3 else (0, *st))


def _fits(t, st, last, group):
    return last == 1 and t.data_ptr() % 16 == 0 and not any(s % 8 for s in st) and st[-2] < 1 << 22 and st[-1] * (group - 1) < 1 << 29


def _new(t):
    return torch.empty_like(t) if t.is_contiguous() else torch.empty(t.shape, dtype=t.dtype, device=t.device)


def _arguments(q, k, v, mask, q_offset, kv_offset, scale, backward):
    """The operands as the kernels take them, the arguments that describe them, and the bytes of workspace."""
    qshape, kshape = q.shape, k.shape
    (q, qs), (k, ks), (v, vs) = _fit(q, qshape[-2] // kshape[-2]), _fit(k), _fit(v)
    h, d, hkv = qshape[-2], qshape[-1], kshape[-2]
    b, l, q_rows, qo = (qshape[0], qshape[1], qshape[0] * qshape[1], 0) if len(qshape) == 4 else (q_offset.numel(), 0, qshape[0], q_offset.data_ptr())
    s, kv_rows, ko = (kshape[1], kshape[0] * kshape[1], 0) if len(kshape) == 4 else (0, kshape[0], kv_offset.data_ptr())
    args = (b, h, hkv, d, l, q_rows, qo, s, kv_rows, ko, q.data_ptr(), *qs, k.data_ptr(), *ks, v.data_ptr(), *vs,
            mask.data_ptr() if mask is not None else 0, s, scale)
    return q, k, v, args, _lib.load().pcm_cross_attn_ws_bytes(b, h, hkv, d, l, q_rows, qo != 0, s, kv_rows, ko != 0, backward)


def _forward(q, k, v, mask, q_offset, kv_offset, scale, want_lse, keep):
    """out, its fp32 form for a backward pass (keep), lse, and the operands as the kernels took them."""
    dev = q.device
    with _lib.on_device(dev):
        q, k, v, args, ws_bytes = _arguments(q, k, v, mask, q_offset, kv_offset, scale, False)
        ws = torch.empty(ws_bytes, dtype=torch.uint8, device=dev) if ws_bytes else None
        out = _new(q)
        out32 = torch.empty(q.shape, dtype=torch.float32, device=dev) if keep else None
        lse = torch.empty(q.shape[:-1], dtype=torch.float32, device=dev) if want_lse else None
        rc = _lib.load().pcm_cross_attn_forward_hip(*args, out.data_ptr(), out32.data_ptr() if keep else 0, lse.data_ptr() if want_lse else 0,
                                                    ws.data_ptr() if ws_bytes else 0, ws_bytes, _raw_stream())
    if rc:
        _lib.check(rc, "pcm_cross_attn_forward_hip")
    return out, out32, lse, q, k, v


class _CrossAttention(Function):
    @staticmethod
    def forward(ctx, q, k, v, mask, q_offset, kv_offset, scale):
        out, out32, lse, q, k, v = _forward(q, k, v, mask, q_offset, kv_offset, scale, True, True)
        ctx.mark_non_differentiable(lse)
        ctx.save_for_backward(q, k, v, mask, q_offset, kv_offset, out32, lse)
        ctx.scale = scale
        return out, lse

    @staticmethod
    def backward(ctx, dout, _):
        _graphs.refuse_tangent(dout, "cross_attention")
        return (_backward_once if torch.is_grad_enabled() else _backward)(ctx, dout)


def _backward(ctx, dout):
    q, k, v, mask, q_offset, kv_offset, out32, lse = ctx.saved_tensors
    dev = q.device
    with _lib.on_device(dev):
        q, k, v, args, ws_bytes = _arguments(q, k, v, mask, q_offset, kv_offset, ctx.scale, True)
        dout, gs = _fit(dout, q.shape[-2] // k.shape[-2])
        _, need_k, need_v, *_ = ctx.needs_input_grad
        dq, dk, dv = _new(q), *((_new(k), _new(v)) if need_k or need_v else (None, None))
        at = lse.numel() * 4 + 15 & ~15
        ws = torch.empty(at + ws_bytes, dtype=torch.uint8, device=dev)  # delta, then the workspace
        p = ws.data_ptr()
        rc = _lib.load().pcm_cross_attn_backward_hip(*args, out32.data_ptr(), lse.data_ptr(), dout.data_ptr(), *gs, p, dq.data_ptr(),
                                                     dk.data_ptr() if need_k or need_v else 0, dv.data_ptr() if need_k or need_v else 0, p + at,
                                                     ws_bytes, _raw_stream())
    if rc:
        _lib.check(rc, "pcm_cross_attn_backward_hip")
    return dq, dk if need_k else None, dv if need_v else None, None, None, None, None


_backward_once = once_differentiable(_backward)  # under create_graph: a second derivative is refused; otherwise its checks cost 4 us for nothing


def _check_offset(offset, side, t, name):
    if t.dim() == 4:
        if offset is not None:
            raise ValueError("cross_attention: %s is padded (4 dimensions): it takes no %s_offset" % (name, side))
        return None
    if offset is None:
        raise ValueError("cross_attention: packed %s (3 dimensions) needs %s_offset" % (name, side))
    if offset.dim() != 1 or offset.numel() < 1 or offset.is_floating_point() or offset.device != t.device:
        raise ValueError("cross_attention: %s_offset must be a 1-d integer tensor on %s" % (side, t.device))
    return _common.i32c(offset)


def cross_attention(q, k, v, key_padding_mask=None, q_offset=None, kv_offset=None, scale=None, return_lse=False):
    """softmax(scale * q k^T) v per head; q, k, v bfloat16.

    q: (B, L, H, D), or packed (T, H, D) with `q_offset`; k, v: (B, S, Hkv, D), or packed (T', Hkv, D) with `kv_offset`.  An offset is
    the int tensor (B,) of the point ops: sequence b holds rows [offset[b - 1], offset[b]).  H is a multiple of Hkv (query head h reads
    key head h // (H / Hkv)); D a multiple of 8 up to 128; any strides with the channels contiguous (what 16-byte accesses do not fit is
    copied first).  key_padding_mask: bool (B, S), or (T',) for packed keys, True = ignore (the nn.MultiheadAttention convention);
    whatever stands in masked or absent rows, NaN and infinities included, has no influence.  scale: > 0, 1 / sqrt(D) by default.
    Under bf16 autocast, q, k and v of other floating types are cast first, as linear layers do.

    Returns (.., H, D) like q; a row without a key is zero, so are packed rows behind the last sequence.  return_lse: also the natural
    logarithm of each row's sum of exponentials, fp32, q.shape[:-1] (-inf without a key; no gradient).  Gradients for q, k and v; results
    do not change from run to run (no atomics)."""
    _common.require_hip(q, k, v, key_padding_mask, q_offset, kv_offset)
    if q.dim() not in (3, 4) or k.dim() not in (3, 4) or v.shape != k.shape:
        raise ValueError("cross_attention: shapes q %s, k %s, v %s" % (tuple(q.shape), tuple(k.shape), tuple(v.shape)))
    if not q.dtype == k.dtype == v.dtype == torch.bfloat16:
        if torch.is_autocast_enabled("cuda") and torch.get_autocast_dtype("cuda") == torch.bfloat16:
            q, k, v = (t.to(torch.bfloat16) if t.is_floating_point() else t for t in (q, k, v))
        if not q.dtype == k.dtype == v.dtype == torch.bfloat16:
            raise TypeError("cross_attention: q, k, v must be bfloat16 (or the call under bf16 autocast), got %s, %s, %s" % (q.dtype, k.dtype, v.dtype))
    if not q.device == k.device == v.device:
        raise ValueError("cross_attention: q, k, v are on %s, %s, %s" % (q.device, k.device, v.device))
    h, d = q.shape[-2:]
    hkv = k.shape[-2]
    if k.shape[-1] != d or hkv < 1 or h < 1 or h % hkv:
        raise ValueError("cross_attention: %d heads of %d over %d key heads of %d" % (h, d, hkv, k.shape[-1]))
    if d % 8 or not 8 <= d <= MAX_HEAD_DIM:
        raise ValueError("cross_attention: head width %d is not a multiple of 8 up to %d" % (d, MAX_HEAD_DIM))
    q_offset, kv_offset = _check_offset(q_offset, "q", q, "q"), _check_offset(kv_offset, "kv", k, "k / v")
    b = q.shape[0] if q.dim() == 4 else q_offset.numel()
    if (k.shape[0] if k.dim() == 4 else kv_offset.numel()) != b:
        raise ValueError("cross_attention: %d query sequences, %d key sequences" % (b, k.shape[0] if k.dim() == 4 else kv_offset.numel()))
    mask = key_padding_mask
    if mask is not None:
        if mask.dtype != torch.bool or mask.shape != k.shape[:-2] or mask.device != k.device:
            raise ValueError("cross_attention: key_padding_mask must be a bool tensor %s on %s" % (tuple(k.shape[:-2]), k.device))
        mask = mask.contiguous()
    scale = 1.0 / math.sqrt(d) if scale is None else float(scale)
    if not 0.0 < scale < math.inf:
        raise ValueError("cross_attention: scale must be positive and finite, got %r" % (scale,))
    if _graphs.watched((q, k, v)):
        out, lse = _CrossAttention.apply(q, k, v, mask, q_offset, kv_offset, scale)
        _graphs.guard_leaves(out, "cross_attention")
    else:
        out, _, lse, *_ = _forward(q, k, v, mask, q_offset, kv_offset, scale, return_lse, False)
    return (out, lse) if return_lse else out
