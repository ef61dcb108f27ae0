"""rotary_axes (csrc/rotary.hip) against complex multiplication in 64 bits."""
import pytest
import torch

from tests import layer_ops_ref as ref

pytestmark = pytest.mark.gpu
DEV = "cuda"


def _case(shape, sections, dtype, coords, seed=0, far=160):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(*shape, generator=g).to(dtype)
    lead = (*shape[:-2], len(sections))
    if coords is torch.float32:
        c = (torch.rand(*lead, generator=g) - 0.5) * far
    else:
        c = torch.randint(-far, far, lead, generator=g, dtype=coords)
    return x, c


@pytest.mark.parametrize("shape,sections,interleaved", [
    ((1, 1, 2), (1,), False), ((1, 8, 64), (11, 11, 10), False), ((3, 8, 64), (11, 11, 10), True), ((37, 3, 72), (5, 0, 7, 9), False),
    ((2, 19, 4, 96), (16, 16, 16), True), ((2, 5, 6, 128), (30, 20), False), ((300, 2, 32), (3, 3, 2), False), ((65, 1, 256), (128,), True),
    ((17, 2, 20), (1, 2), True), ((17, 2, 21), (3, 1, 4), False)])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("coords,far", [(torch.float32, 160), (torch.int32, 1 << 30), (torch.int64, 1 << 40)])
def test_forward_and_gradient(shape, sections, interleaved, dtype, coords, far):
    from pointcloudmatters_amd.policy import rotary_axes

    x, c = _case(shape, sections, dtype, coords, far=far)
    dout = torch.randn(*shape, generator=torch.Generator().manual_seed(9)).to(dtype)
    xd = x.to(DEV).requires_grad_()
    out = rotary_axes(xd, c.to(DEV), sections, interleaved=interleaved)
    assert out.dtype == dtype and out.is_contiguous()
    want, err = ref.rotary(x, c, sections, 10000.0, interleaved)
    ref.check(out, want, ref.rounded(want, err, dtype), "out")
    (dx,) = torch.autograd.grad(out, xd, dout.to(DEV))
    want, err = ref.rotary(dout, c, sections, 10000.0, interleaved, inverse=True)
    ref.check(dx, want, ref.rounded(want, err, dtype), "dx")
    half = 2 * sum(sections)
    assert torch.equal(out[..., half:].detach().cpu(), x[..., half:])


def test_turning_there_and_back_and_relative_positions():
    """q . k depends on the difference of the coordinates; the gradient is the turn back."""
    from pointcloudmatters_amd.policy import rotary_axes

    g = torch.Generator().manual_seed(3)
    q, k = torch.randn(40, 2, 64, generator=g), torch.randn(40, 2, 64, generator=g)
    c = torch.randint(0, 50, (40, 3), generator=g, dtype=torch.int32)
    s = [(rotary_axes(q.to(DEV), (c + off).to(DEV), (11, 11, 10)) * rotary_axes(k.to(DEV), (c * 0 + 7 + off).to(DEV), (11, 11, 10))).sum(-1).cpu()
         for off in (0, 1000)]
    norm = q.norm(dim=-1) * k.norm(dim=-1)
    assert ((s[0] - s[1]).abs() <= 64 * ref.F32 * 16 * norm).all()


@pytest.mark.parametrize("interleaved", [False, True])
def test_strides_and_broadcast_coordinates(interleaved):
    """The queries and keys inside one packed projection (views), heads-first storage, odd offsets, coordinates shared by the batch."""
    from pointcloudmatters_amd.policy import rotary_axes

    g = torch.Generator().manual_seed(5)
    sections = (8, 4, 4)
    qkv = torch.randn(2, 11, 3, 4, 32, generator=g)
    c = torch.randn(11, 3, generator=g) * 40
    full = c.expand(2, 11, 3)
    for dtype in (torch.bfloat16, torch.float32):
        d = qkv.to(dtype).to(DEV)
        views = {"packed": d[:, :, 1], "heads first": d[:, :, 0].transpose(1, 2).contiguous().transpose(1, 2),
                 "odd offset": torch.cat([d[:, :, 2].reshape(-1)[:1], d[:, :, 2].reshape(-1)]).narrow(0, 1, 2 * 11 * 4 * 32).view(2, 11, 4, 32),
                 "channels apart": d[:, :, 2].transpose(-1, -2).contiguous().transpose(-1, -2), "every other": d[:, ::2, 1]}
        for name, x in views.items():
            cc = full[:, ::2] if name == "every other" else full
            want, err = ref.rotary(x, cc, sections, 100.0, interleaved)
            coords = (c[::2] if name == "every other" else c).to(DEV)
            ref.check(rotary_axes(x, coords, sections, base=100.0, interleaved=interleaved), want, ref.rounded(want, err, dtype), name)
            wide = torch.zeros(*cc.shape[:-1], 7)
            wide[..., 2:5] = cc
            ref.check(rotary_axes(x, wide.to(DEV)[..., 2:5], sections, base=100.0, interleaved=interleaved), want, ref.rounded(want, err, dtype), name)


def test_empty_infinite_and_not_a_number():
    from pointcloudmatters_amd.policy import rotary_axes

    e = torch.zeros(0, 4, 32, device=DEV, requires_grad=True)
    out = rotary_axes(e, torch.zeros(0, 2, device=DEV), (4, 4))
    assert out.shape == e.shape and torch.autograd.grad(out.sum(), e)[0].shape == e.shape
    x = torch.ones(3, 1, 8, device=DEV)
    c = torch.tensor([[0.0], [float("nan")], [1.0]], device=DEV)
    out = rotary_axes(x, c, (3,)).cpu()
    assert out[1, :, :6].isnan().all() and (out[1, :, 6:] == 1).all() and out[[0, 2]].isfinite().all() and (out[0] == 1).all()


def test_result_on_another_stream_and_under_capture():
    from pointcloudmatters_amd import _graphs
    from pointcloudmatters_amd.policy import rotary_axes

    x, c = (t.to(DEV) for t in _case((130, 4, 64), (11, 11, 10), torch.bfloat16, torch.float32))
    want = rotary_axes(x, c, (11, 11, 10))
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        got = rotary_axes(x, c, (11, 11, 10))
    s.synchronize()
    assert torch.equal(got, want)
    graph, out = _graphs.captured(lambda: rotary_axes(x, c, (11, 11, 10)))
    for i in range(3):
        x.copy_(torch.randn_like(x))
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, rotary_axes(x, c, (11, 11, 10))), i


def test_second_derivative():
    """The gradient is a turn back and has one itself.  f = sum(y^3) / 3, y = T x: grad = T' y^2, and d(grad . c) / dx = T' (2 y (T c))."""
    from pointcloudmatters_amd.policy import rotary_axes

    x, coords = _case((11, 2, 24), (5, 4), torch.float32, torch.int32, seed=12)
    c = torch.randn(x.shape, generator=torch.Generator().manual_seed(13))
    xd = x.to(DEV).requires_grad_()
    y = rotary_axes(xd, coords.to(DEV), (5, 4))
    (grad,) = torch.autograd.grad((y ** 3).sum() / 3, xd, create_graph=True)
    (second,) = torch.autograd.grad((grad * c.to(DEV)).sum(), xd)
    turn = lambda t, inverse=False: ref.rotary(t, coords, (5, 4), 10000.0, False, inverse)[0]  # noqa: E731
    # three turns of 8 units of 2^-24 of two channels each, two products: a channel is at most the pair's 1-norm, which grows by 2 a turn
    want = turn(2 * turn(x) * turn(c), True)
    pair = lambda t: t.double().abs().unflatten(-1, (2, 12)).amax().item()  # noqa: E731
    assert (second.double().cpu() - want).abs().max().item() <= 2 * (2 * pair(x)) * (2 * pair(c)) * 2 * (3 * 8 + 4) * ref.F32
