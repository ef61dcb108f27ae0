"""gated_ffn (csrc/gated_ffn.hip) against its formula in 64 bits, with element-wise bounds (tests/layer_ops_ref.py)."""
import math

import pytest
import torch

from tests import layer_ops_ref as ref

pytestmark = pytest.mark.gpu
DEV = "cuda"
NAMES = ("y", "dx", "dw_gate", "dw_up", "dw_down", "db_gate", "db_up", "db_down")


def _inputs(r, e, f, bias, seed=0):
    g = torch.Generator().manual_seed(seed)
    n = lambda *s, scale=1.0: (torch.randn(*s, generator=g) * scale).bfloat16()  # noqa: E731
    x, wg, wu, wd = n(r, e), n(f, e, scale=e ** -0.5), n(f, e, scale=e ** -0.5), n(e, f, scale=f ** -0.5)
    bs = (n(f, scale=0.3), n(f, scale=0.3), n(e, scale=0.3)) if bias else (None, None, None)
    return x, wg, wu, wd, *bs, n(r, e)


def _run(x, wg, wu, wd, bg, bu, bd, dy, act):
    from pointcloudmatters_amd.policy import gated_ffn

    leaves = [t.to(DEV).requires_grad_() if t is not None else None for t in (x, wg, wu, wd, bg, bu, bd)]
    y = gated_ffn(*leaves, activation=act)
    grads = torch.autograd.grad(y, [t for t in leaves if t is not None], dy.to(DEV))
    with torch.no_grad():
        assert torch.equal(gated_ffn(*leaves, activation=act), y)  # with and without what the backward pass keeps
    return [y, *grads]


def _check(args, act):
    want = ref.ffn(*args[:7], act, args[7])
    for name, got, (r, e) in zip(NAMES, _run(*args, act), want):
        ref.check(got, r, e, name)


@pytest.mark.parametrize("r,e,f", [(1, 8, 8), (1, 64, 40), (5, 32, 64), (16, 72, 200), (33, 64, 65), (130, 96, 130), (129, 264, 72), (64, 20, 31), (7, 33, 9),
                                   (200, 128, 128)])
@pytest.mark.parametrize("act,bias", [("silu", True), ("gelu", False), ("relu", True)])
def test_forward_and_gradients(r, e, f, act, bias):
    _check(_inputs(r, e, f, bias), act)


@pytest.mark.parametrize("r", [1100, 2050])
def test_weight_gradients_shared_out_over_rows(r):
    _check(_inputs(r, 40, 72, True, seed=1), "silu")


def test_strided_rows_and_leading_dimensions():
    from pointcloudmatters_amd.policy import gated_ffn

    x, wg, wu, wd, bg, bu, bd, dy = _inputs(24, 48, 56, True, seed=2)
    want = _run(x, wg, wu, wd, bg, bu, bd, dy, "silu")
    wide = torch.randn(2, 12, 100).bfloat16().to(DEV)
    for start in (0, 8, 3):  # 3: rows that 16-byte accesses do not fit
        w = wide.clone()
        w[..., start:start + 48] = x.to(DEV).view(2, 12, 48)
        leaf = w[..., start:start + 48].detach().requires_grad_()
        y = gated_ffn(leaf, *(t.to(DEV) for t in (wg, wu, wd, bg, bu, bd)))
        assert y.shape == (2, 12, 48) and torch.equal(y.view(24, 48), want[0])
        g = torch.zeros(2, 12, 60, dtype=torch.bfloat16, device=DEV)
        g[..., start:start + 48] = dy.to(DEV).view(2, 12, 48)
        assert torch.equal(torch.autograd.grad(y, leaf, g[..., start:start + 48])[0].reshape(24, 48), want[1])
    flipped = wg.t().contiguous().t().to(DEV)
    assert torch.equal(gated_ffn(x.to(DEV), flipped, *(t.to(DEV) for t in (wu, wd, bg, bu, bd))), want[0])
    one = x[:1].expand(24, 48)
    assert torch.equal(gated_ffn(x[:1].to(DEV).expand(24, 48), *(t.to(DEV) for t in (wg, wu, wd))),
                       gated_ffn(one.contiguous().to(DEV), *(t.to(DEV) for t in (wg, wu, wd))))


def test_some_gradients_only():
    from pointcloudmatters_amd.policy import gated_ffn

    args = _inputs(40, 64, 72, True, seed=3)
    want = _run(*args, "gelu")
    for keep in ((0,), (1,), (2, 3), (4,), (5, 6), (3,), (6,), (0, 5)):
        leaves = [t.to(DEV).requires_grad_(i in keep) for i, t in enumerate(args[:7])]
        y = gated_ffn(*leaves, activation="gelu")
        got = torch.autograd.grad(y, [leaves[i] for i in keep], args[7].to(DEV))
        assert all(torch.equal(g, want[1 + i]) for g, i in zip(got, keep)), keep


def test_no_rows():
    from pointcloudmatters_amd.policy import gated_ffn

    x, wg, wu, wd, bg, bu, bd, _ = (t.to(DEV).requires_grad_() for t in _inputs(3, 16, 24, True))
    y = gated_ffn(x[:0], wg, wu, wd, bg, bu, bd)
    assert y.shape == (0, 16)
    for g in torch.autograd.grad(y.sum(), (wg, wu, wd, bg, bu, bd)):
        assert (g == 0).all()


def test_large_gate_values():
    """Gates far into both tails: silu and gelu go to 0 and to the identity without an infinity."""
    x, wg, wu, wd, _, _, _, dy = _inputs(9, 32, 48, False, seed=4)
    for act in ("silu", "gelu"):
        _check(((x * 64).bfloat16(), wg, wu, wd, None, None, None, dy), act)


def test_under_autocast_other_types_are_cast():
    from pointcloudmatters_amd.policy import gated_ffn

    x, wg, wu, wd, bg, bu, bd, dy = _inputs(10, 32, 40, True, seed=5)
    want = _run(x, wg, wu, wd, bg, bu, bd, dy, "silu")
    leaves = [t.float().to(DEV).requires_grad_() for t in (x, wg, wu, wd, bg, bu, bd)]
    with torch.autocast("cuda", dtype=torch.bfloat16):
        y = gated_ffn(*leaves)
    assert y.dtype == torch.bfloat16 and torch.equal(y, want[0])
    for got, w in zip(torch.autograd.grad(y, leaves, dy.to(DEV)), want[1:]):
        assert got.dtype == torch.float32 and torch.equal(got, w.float())


def test_gradient_against_differences():
    args = _inputs(6, 24, 40, True, seed=6)
    dy = args[7].double()
    got = _run(*args, "silu")[1:]
    for i in range(7):
        step = torch.randn(args[i].shape, generator=torch.Generator().manual_seed(20 + i)).double() * 1e-5
        vals = []
        for sign in (1, -1):
            t = [a.double() for a in args[:7]]
            t[i] = t[i] + sign * step
            vals.append(float((ref.ffn(*t, "silu")[0][0] * dy).sum().detach()))
        slope, part = (vals[0] - vals[1]) / 2, got[i].double().cpu() * step
        assert abs(slope - float(part.sum())) <= 8 * ref.HALF * float(part.abs().sum()) + 1e-10, (NAMES[i + 1], slope, float(part.sum()))


def test_runs_repeat_bit_for_bit():
    args = _inputs(1500, 64, 100, True, seed=7)
    a, b = _run(*args, "silu"), _run(*args, "silu")
    assert all(torch.equal(x, y) for x, y in zip(a, b))


@pytest.mark.parametrize("r", [2, 3, 8, 9])
def test_few_rows_and_one_more(r):
    _check(_inputs(r, 72, 100, True, seed=8), "silu")


@pytest.mark.parametrize("r,e,f", [(8200, 520, 1700), (8200, 1544, 520)])
def test_large_tiles_at_size(r, e, f):
    """Products of over 200 tiles of 256 x 256, the last of them ragged in rows and columns and half outside the hidden columns."""
    _check(_inputs(r, e, f, True, seed=9), "silu")


def test_weights_of_different_alignment():
    """Gate and up weights as parts of one buffer, the second not at a 16-byte boundary."""
    from pointcloudmatters_amd.policy import gated_ffn

    x, wg, wu, wd, bg, bu, bd, _ = _inputs(40, 48, 72, True, seed=10)
    want = gated_ffn(*(t.to(DEV) for t in (x, wg, wu, wd, bg, bu, bd)))
    for start in (0, 1):
        buf = torch.zeros(start + 2 * wg.numel() + 3, dtype=torch.bfloat16, device=DEV)
        g, u = buf[start:start + wg.numel()].view_as(wg), buf[start + wg.numel() + 3:][:wu.numel()].view_as(wu)
        g.copy_(wg), u.copy_(wu)
        assert torch.equal(gated_ffn(x.to(DEV), g, u, *(t.to(DEV) for t in (wd, bg, bu, bd))), want)


@pytest.mark.parametrize("r,e,f", [(4120, 512, 2040), (4120, 2048, 520)])
def test_rows_past_whole_rounds_at_size(r, e, f):
    """24 rows more than whole rounds of tiles: a second launch for them (both projections and dh; y and dx, with split contractions)."""
    _check(_inputs(r, e, f, True, seed=11), "gelu")
