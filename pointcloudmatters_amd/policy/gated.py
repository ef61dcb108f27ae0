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


def _ptr(t):
    return 0 if t is None else t.data_ptr()


def _workspace(L_, rows, e, f, backward, dev):
    n = L_.pcm_gated_ffn_ws_bytes(rows, e, f, int(backward))
    return n, (torch.empty(n, dtype=torch.uint8, device=dev) if n else None)


def _rows(t, width):
    """(rows, width) with contiguous channels: a view where the strides allow one."""
    t = t.reshape(-1, width)
    return t if t.stride(-1) == 1 or width == 1 else t.contiguous()


class _GatedFFN(Function):
    @staticmethod
    def forward(ctx, x, w_gate, w_up, w_down, b_gate, b_up, b_down, act):
        L_ = _lib.load()
        rows, e = x.shape
        f = w_gate.shape[0]
        w_gate, w_up, w_down = w_gate.contiguous(), w_up.contiguous(), w_down.contiguous()
        b_gate, b_up, b_down = (b.contiguous() if b is not None else None for b in (b_gate, b_up, b_down))
        grad = any(ctx.needs_input_grad[:7])
        with torch.cuda.device(x.device):
            ld = L_.pcm_gated_ffn_hidden_ld(f)
            y = torch.empty(rows, e, dtype=x.dtype, device=x.device)
            a, u, h = torch.empty(3 if grad else 1, rows, ld, dtype=x.dtype, device=x.device) if grad else (None, None, torch.empty(rows, ld, dtype=x.dtype, device=x.device))
            n, ws = _workspace(L_, rows, e, f, False, x.device)
            rc = L_.pcm_gated_ffn_forward_hip(rows, e, f, act, x.data_ptr(), x.stride(0), w_gate.data_ptr(), w_up.data_ptr(), w_down.data_ptr(),
                                              _ptr(b_gate), _ptr(b_up), _ptr(b_down), y.data_ptr(), _ptr(a), _ptr(u), h.data_ptr(),
                                              _ptr(ws), n, _raw_stream())
        _lib.check(rc, "pcm_gated_ffn_forward_hip")
        if grad:
            ctx.save_for_backward(x, w_gate, w_up, w_down, a, u, h)
            ctx.act = act
        return y

    @staticmethod
    @once_differentiable
    def backward(ctx, dy):
        L_ = _lib.load()
        x, w_gate, w_up, w_down, a, u, h = ctx.saved_tensors
        need = ctx.needs_input_grad
        (rows, e), f, dev = x.shape, w_gate.shape[0], x.device
        dy = _rows(dy, e)
        with torch.cuda.device(dev):
            new = torch.zeros if rows == 0 else torch.empty  # no rows: no launch, the gradients of the weights are zero
            dx = new(x.shape, dtype=x.dtype, device=dev) if need[0] else None
            dwg, dwu = (new(f, e, dtype=x.dtype, device=dev) if need[1] or need[2] else None for _ in range(2))
            dwd = new(e, f, dtype=x.dtype, device=dev) if need[3] else None
            dbg, dbu = (new(f, dtype=x.dtype, device=dev) if need[4] or need[5] else None for _ in range(2))
            dbd = new(e, dtype=x.dtype, device=dev) if need[6] else None
            n, ws = _workspace(L_, rows, e, f, True, dev)
            rc = L_.pcm_gated_ffn_backward_hip(rows, e, f, ctx.act, x.data_ptr(), x.stride(0), w_gate.data_ptr(), w_up.data_ptr(),
                                               w_down.data_ptr(), a.data_ptr(), u.data_ptr(), h.data_ptr(), dy.data_ptr(), dy.stride(0),
                                               _ptr(dx), _ptr(dwg), _ptr(dwu), _ptr(dwd), _ptr(dbg), _ptr(dbu), _ptr(dbd), _ptr(ws), n,
                                               _raw_stream())
        _lib.check(rc, "pcm_gated_ffn_backward_hip")
        return (dx, dwg if need[1] else None, dwu if need[2] else None, dwd, dbg if need[4] else None, dbu if need[5] else None, dbd, None)


def gated_ffn(x, w_gate, w_up, w_down, b_gate=None, b_up=None, b_down=None, activation="silu"):
    """x (..., E) -> (act(x w_gate^T + b_gate) * (x w_up^T + b_up)) w_down^T + b_down, bfloat16 with fp32 accumulation.

    w_gate, w_up: (F, E), w_down: (E, F), the layouts of nn.Linear; each bias optional; E and F of any size (a multiple of 8 spares a
    copy into padded rows).  activation: "silu", "gelu" (erf) or "relu".  Under bf16 autocast, operands of other floating types are
    cast first, as linear layers do.  Gradients for x, the weights and the biases; results do not change from run to run."""
    _common.require_hip(x, w_gate, w_up, w_down, b_gate, b_up, b_down)
    if activation not in ACTIVATIONS:
        raise ValueError("gated_ffn: activation should be silu/gelu/relu, not %r" % (activation,))
    given = [x, w_gate, w_up, w_down, b_gate, b_up, b_down]
    if torch.is_autocast_enabled("cuda") and torch.get_autocast_dtype("cuda") == torch.bfloat16:
        given = [t.to(torch.bfloat16) if t is not None and t.is_floating_point() else t for t in given]
    for t, name in zip(given, ("x", "w_gate", "w_up", "w_down", "b_gate", "b_up", "b_down")):
        if t is not None and t.dtype != torch.bfloat16:
            raise TypeError("gated_ffn: %s must be bfloat16 (or the call under bf16 autocast), got %s" % (name, t.dtype))
        if t is not None and t.device != x.device:
            raise ValueError("gated_ffn: x is on %s, %s on %s" % (x.device, name, t.device))
    x, w_gate, w_up, w_down, b_gate, b_up, b_down = given
    if x.dim() < 1 or w_gate.dim() != 2 or w_gate.shape != w_up.shape or min(w_gate.shape) < 1:
        raise ValueError("gated_ffn: shapes x %s, w_gate %s, w_up %s" % (tuple(x.shape), tuple(w_gate.shape), tuple(w_up.shape)))
    f, e = w_gate.shape
    if x.shape[-1] != e or tuple(w_down.shape) != (e, f):
        raise ValueError("gated_ffn: x %s, w_gate %s, w_down %s" % (tuple(x.shape), (f, e), tuple(w_down.shape)))
    for b, n, name in ((b_gate, f, "b_gate"), (b_up, f, "b_up"), (b_down, e, "b_down")):
        if b is not None and tuple(b.shape) != (n,):
            raise ValueError("gated_ffn: %s must be (%d,), got %s" % (name, n, tuple(b.shape)))
    rows = _rows(x, e)
    y = _GatedFFN.apply(rows, w_gate, w_up, w_down, b_gate, b_up, b_down, ACTIVATIONS[activation])
    return _graphs.guard_leaves(y, "gated_ffn").view(x.shape)
