"""Rotary positions over several axes (csrc/rotary.hip): the turn of a token's head channels by its own coordinates -- x, y, z of a
point, or time, height and width of a frame -- that makes q . k depend on the difference of two tokens' positions.  Stands beside the
additive embedding `sa_layer.coord_embedding_sine`; applied to the queries and the keys in front of an attention.
"""
import ctypes
import functools

import torch
from torch.autograd import Function

from .. import _graphs, _lib
from ..pointops import _common
from .._lib import raw_stream as _raw_stream

MAX_PAIRS = 128  # turned pairs of a head
MAX_AXES = 8
_COORDS = {torch.float32: 0, torch.int32: 1, torch.int64: 2}


@functools.lru_cache(maxsize=256)
def _sections(sections):
    return (ctypes.c_int * len(sections))(*sections)  # read by the entry point before it returns


def _launch(x, coords, sections, base, interleaved, inverse):
    if x.stride(-1) != 1:
        x = x.contiguous()
    dev = x.device
    with _lib.on_device(dev):
        out = torch.empty_like(x) if x.is_contiguous() else torch.empty(x.shape, dtype=x.dtype, device=dev)
        xs, os_, cs = x.stride(), out.stride(), coords.stride()
        if len(xs) == 3:
            b, (l, h, d) = 1, x.shape
            x_bs = o_bs = 0
            (x_ls, x_hs, _), (o_ls, o_hs, _) = xs, os_
        else:
            b, l, h, d = x.shape
            (x_bs, x_ls, x_hs, _), (o_bs, o_ls, o_hs, _) = xs, os_
        rc = _lib.load().pcm_rotary_axes_hip(b, l, h, d, x.dtype is torch.bfloat16, x.data_ptr(), x_bs, x_ls, x_hs, out.data_ptr(), o_bs, o_ls, o_hs,
                                             _COORDS[coords.dtype], coords.data_ptr(), cs[0] if len(cs) == 3 else 0, cs[-2], len(sections),
                                             _sections(sections), base, interleaved, inverse, _raw_stream())
    if rc:
        _lib.check(rc, "pcm_rotary_axes_hip")
    return out


class _RotaryAxes(Function):
    @staticmethod
    def forward(ctx, x, coords, sections, base, interleaved, inverse):
        if ctx.needs_input_grad[0]:
            ctx.save_for_backward(coords)
            ctx.meta = (sections, base, interleaved, not inverse)
        return _launch(x, coords, sections, base, interleaved, inverse)

    @staticmethod
    def backward(ctx, dout):
        (coords,) = ctx.saved_tensors
        turn = _RotaryAxes.apply if dout.requires_grad and torch.is_grad_enabled() or _graphs.has_tangent(dout) else _launch  # linear: its own backward, turned back
        return turn(dout, coords, *ctx.meta), None, None, None, None, None


def rotary_axes(x, coords, sections, base=10000.0, interleaved=False):
    """x (T, H, D) or (B, L, H, D), bf16 or fp32, turned by coords (T, A) / (B, L, A) / (L, A) (fp32, int32 or int64; one row for all
    heads of a token).  sections: A pair counts; pair j of axis a turns by ``coords[..., a] * base ** (-j / sections[a])`` radians.  With
    half = sum(sections) the pairs are channels (i, i + half), or (2 i, 2 i + 1) when `interleaved`; channels from 2 * half on pass
    through.  Any strides with the channels contiguous.  Returns a new contiguous tensor of x's type (fp32 arithmetic; angles in fp64,
    off by about 2^-52 of themselves: less than fp32 resolves up to 2^26 radians); x gets a gradient, coords must not ask for one."""
    _common.require_hip(x, coords)
    sections = tuple(sections)
    shape, cshape = x.shape, coords.shape
    if len(shape) not in (3, 4):
        raise ValueError("rotary_axes: x must be (T, H, D) or (B, L, H, D), got %s" % (tuple(shape),))
    if x.dtype not in (torch.bfloat16, torch.float32):
        raise TypeError("rotary_axes: x must be bfloat16 or float32, got %s" % x.dtype)
    if coords.dtype not in _COORDS:
        raise TypeError("rotary_axes: coords must be float32, int32 or int64, got %s" % coords.dtype)
    if coords.requires_grad:
        raise ValueError("rotary_axes: coords get no gradient: detach them")
    if coords.device != x.device:
        raise ValueError("rotary_axes: x is on %s, coords on %s" % (x.device, coords.device))
    if len(cshape) < 2 or (cshape[:-1] != shape[:-2] and cshape[:-1] != shape[-3:-2]):
        raise ValueError("rotary_axes: coords %s do not fit x %s" % (tuple(cshape), tuple(shape)))
    if not 1 <= len(sections) <= MAX_AXES or cshape[-1] != len(sections):
        raise ValueError("rotary_axes: %d sections for %d coordinates (at most %d)" % (len(sections), cshape[-1], MAX_AXES))
    half = sum(sections)
    if min(sections) < 0 or not 1 <= half <= MAX_PAIRS or 2 * half > shape[-1]:
        raise ValueError("rotary_axes: sections %s turn %d channels of a head of %d (at most %d)" % (sections, 2 * half, shape[-1], 2 * MAX_PAIRS))
    if not base > 0:
        raise ValueError("rotary_axes: base must be positive, got %r" % (base,))
    if coords.stride(-1) != 1:
        coords = coords.contiguous()
    if not _graphs.watched((x,)):
        return _launch(x, coords, sections, float(base), bool(interleaved), False)
    return _graphs.guard_leaves(_RotaryAxes.apply(x, coords, sections, float(base), bool(interleaved), False), "rotary_axes")
