"""The gated feed-forward block (csrc/gated_ffn.hip): ``(act(x Wg^T + bg) * (x Wu^T + bu)) Wd^T + bd`` with its backward pass, any
widths, one row or many.  Stands beside `fused_ops.ffn_ln` (LayerNorm(x + W2 relu(W1 x)) of the shipped 32-unit layers).
"""
import torch
from torch.autograd import Function
from torch.autograd.function import once_differentiable

from .. import _graphs, _lib
from ..pointops import _common
from .._lib import raw_stream as _raw_stream

ACTIVATIONS = {"silu": 0, "gelu": 1, "relu": 2}
_NAMES = ("x", "w_gate", "w_up", "w_down", "b_gate", "b_up", "b_down")


def _ptr(t):
    return 0 if t is None else t.data_ptr()


def _rows(t, width):
    """(rows, width) with contiguous channels: a view where the strides allow one."""
    if t.dim() != 2:
        t = t.reshape(-1, width)
    return t if t.stride(-1) == 1 or width == 1 else t.contiguous()


def _empty(n, dev):
    return torch.empty(n, dtype=torch.uint8, device=dev)


def _forward(x, w_gate, w_up, w_down, b_gate, b_up, b_down, act, keep):
    """y, and for a backward pass (keep) the hidden tensors a | u (fp32) | h in one buffer, else None."""
    L_ = _lib.load()
    (rows, e), f, dev = x.shape, w_gate.shape[0], x.device
    with _lib.on_device(dev):
        ld = L_.pcm_gated_ffn_hidden_ld(f)
        n = L_.pcm_gated_ffn_ws_bytes(rows, e, f, False)
        y = torch.empty((rows, e), dtype=x.dtype, device=dev)
        size = 2 * int(rows) * ld  # int: while a call is traced, sizes are tensors, and addresses formed with them would be
        hidden = _empty(5 * size if keep else size + n, dev)  # without a backward pass: h, then the workspace
        p = hidden.data_ptr()
        a, u, h = (p, p + 2 * size, p + 4 * size) if keep else (0, 0, p)
        ws = _empty(n, dev) if keep and n else None
        rc = L_.pcm_gated_ffn_forward_hip(rows, e, f, act, x.data_ptr(), x.stride(0), w_gate.data_ptr(), w_up.data_ptr(), w_down.data_ptr(),
                                          _ptr(b_gate), _ptr(b_up), _ptr(b_down), y.data_ptr(), a, u, h, _ptr(ws) if keep else p + size, n,
                                          _raw_stream())
    if rc:
        _lib.check(rc, "pcm_gated_ffn_forward_hip")
    return y, hidden if keep else None


class _GatedFFN(Function):
    @staticmethod
    def forward(ctx, x, w_gate, w_up, w_down, b_gate, b_up, b_down, act):
        y, hidden = _forward(x, w_gate, w_up, w_down, b_gate, b_up, b_down, act, True)
        ctx.save_for_backward(x, w_gate, w_up, w_down, hidden)
        ctx.act = act
        return y

    @staticmethod
    def backward(ctx, dy):
        _graphs.refuse_tangent(dy, "gated_ffn")
        return (_backward_once if torch.is_grad_enabled() else _backward)(ctx, dy)


def _backward(ctx, dy):
    L_ = _lib.load()
    x, w_gate, w_up, w_down, hidden = ctx.saved_tensors
    need = ctx.needs_input_grad
    (rows, e), f, dev = x.shape, w_gate.shape[0], x.device
    dy = _rows(dy, e)
    with _lib.on_device(dev):
        like = torch.zeros_like if rows == 0 else torch.empty_like  # no rows: no launch, the gradients of the weights are zero
        bias = w_gate.new_zeros if rows == 0 else w_gate.new_empty
        dx = x.new_empty((rows, e)) if need[0] else None
        dwg, dwu = (like(w_gate), like(w_up)) if need[1] or need[2] else (None, None)
        dwd = like(w_down) if need[3] else None
        dbg, dbu = (bias(f), bias(f)) if need[4] or need[5] else (None, None)
        dbd = bias(e) if need[6] else None
        n = L_.pcm_gated_ffn_ws_bytes(rows, e, f, True)
        ws = _empty(n, dev)
        p, size = hidden.data_ptr(), hidden.numel() // 5
        rc = L_.pcm_gated_ffn_backward_hip(rows, e, f, ctx.act, x.data_ptr(), x.stride(0), w_gate.data_ptr(), w_up.data_ptr(),
                                           w_down.data_ptr(), p, p + 2 * size, p + 4 * size, dy.data_ptr(), dy.stride(0), _ptr(dx), _ptr(dwg),
                                           _ptr(dwu), _ptr(dwd), _ptr(dbg), _ptr(dbu), _ptr(dbd), ws.data_ptr(), n, _raw_stream())
    if rc:
        _lib.check(rc, "pcm_gated_ffn_backward_hip")
    return dx, dwg if need[1] else None, dwu if need[2] else None, dwd, dbg if need[4] else None, dbu if need[5] else None, dbd, None


_backward_once = once_differentiable(_backward)  # under create_graph: a second derivative is refused; otherwise its checks cost 4 us for nothing


def gated_ffn(x, w_gate, w_up, w_down, b_gate=None, b_up=None, b_down=None, activation="silu"):
    """x (..., E) -> (act(x w_gate^T + b_gate) * (x w_up^T + b_up)) w_down^T + b_down, bfloat16 with fp32 accumulation.

    w_gate, w_up: (F, E), w_down: (E, F), the layouts of nn.Linear; each bias optional; E and F of any size (a multiple of 8 spares a
    copy into padded rows).  activation: "silu", "gelu" (erf) or "relu".  Under bf16 autocast, operands of other floating types are
    cast first, as linear layers do.  Gradients for x, the weights and the biases; results do not change from run to run."""
    _common.require_hip(x, w_gate, w_up, w_down, b_gate, b_up, b_down)
    if activation not in ACTIVATIONS:
        raise ValueError("gated_ffn: activation should be silu/gelu/relu, not %r" % (activation,))
    given = (x, w_gate, w_up, w_down, b_gate, b_up, b_down)
    if torch.is_autocast_enabled("cuda") and torch.get_autocast_dtype("cuda") == torch.bfloat16:
        given = tuple(t.to(torch.bfloat16) if t is not None and t.is_floating_point() else t for t in given)
    for t, name in zip(given, _NAMES):
        if t is not None and (t.dtype is not torch.bfloat16 or t.device != x.device):
            if t.dtype is not torch.bfloat16:
                raise TypeError("gated_ffn: %s must be bfloat16 (or the call under bf16 autocast), got %s" % (name, t.dtype))
            raise ValueError("gated_ffn: x is on %s, %s on %s" % (x.device, name, t.device))
    x, w_gate, w_up, w_down, b_gate, b_up, b_down = given
    shape, ws = x.shape, w_gate.shape
    if len(shape) < 1 or len(ws) != 2 or ws != w_up.shape or min(ws) < 1:
        raise ValueError("gated_ffn: shapes x %s, w_gate %s, w_up %s" % (tuple(shape), tuple(ws), tuple(w_up.shape)))
    f, e = ws
    if shape[-1] != e or w_down.shape != (e, f):
        raise ValueError("gated_ffn: x %s, w_gate %s, w_down %s" % (tuple(shape), (f, e), tuple(w_down.shape)))
    for b, n, name in ((b_gate, f, "b_gate"), (b_up, f, "b_up"), (b_down, e, "b_down")):
        if b is not None and b.shape != (n,):
            raise ValueError("gated_ffn: %s must be (%d,), got %s" % (name, n, tuple(b.shape)))
    args = [_rows(x, e)] + [t if t is None or t.is_contiguous() else t.contiguous() for t in (w_gate, w_up, w_down, b_gate, b_up, b_down)]
    if _graphs.watched(given):
        y = _graphs.guard_leaves(_GatedFFN.apply(*args, ACTIVATIONS[activation]), "gated_ffn")
    else:
        y, _ = _forward(*args, ACTIVATIONS[activation], False)
    return y if len(shape) == 2 else y.view(shape)
