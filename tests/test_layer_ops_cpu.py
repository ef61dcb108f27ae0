"""CPU: what rotary_axes, cross_attention and gated_ffn refuse, and their kernel sources on the host wave64 model (tests/wavesim) against
64-bit formulas -- the GPU tests of the same operators at their smaller sizes."""
import ctypes
import importlib
import os
import types

import pytest
import torch

from tests.wavesim import build as _build

needs_model = pytest.mark.skipif(not os.path.exists(_build.CLANG), reason="needs the ROCm clang++ as host compiler (tests/wavesim)")

GPU_FILES = ("test_rotary_gpu", "test_cross_attn_gpu", "test_gated_ffn_gpu", "test_layer_ops_gpu")
NEEDS_HIP_RUNTIME = ("stream", "captur", "at_size")  # at_size: too long for the model


def _adopt():
    for short in GPU_FILES:
        mod = importlib.import_module("tests." + short)
        for name, fn in sorted(vars(mod).items()):
            if name.startswith("test_") and isinstance(fn, types.FunctionType) and not any(w in name for w in NEEDS_HIP_RUNTIME):
                clone = types.FunctionType(fn.__code__, fn.__globals__, "%s__%s" % (short, name[5:]), fn.__defaults__, fn.__closure__)
                clone.pytestmark = [m for m in getattr(fn, "pytestmark", []) if m.name == "parametrize"] + [needs_model.mark]
                globals()["test_" + clone.__name__] = clone


_adopt()


@pytest.fixture(autouse=True)
def _host_wave64_model(request):
    if "_gpu__" not in request.node.name:
        yield
        return
    from tests.wavesim.backend import simulated_device

    mods = [importlib.import_module("tests." + n) for n in GPU_FILES]
    with simulated_device(claim_cuda=True):
        for m in mods:
            m.DEV = "cpu"
        try:
            yield
        finally:
            for m in mods:
                m.DEV = "cuda"


@pytest.fixture
def model():
    from tests.wavesim.backend import simulated_device

    if not os.path.exists(_build.CLANG):
        pytest.skip("needs the ROCm clang++ as host compiler (tests/wavesim)")
    with simulated_device(claim_cuda=True):
        yield


def _bf(*s):
    return torch.zeros(*s, dtype=torch.bfloat16)


def test_host_tensors_are_refused():
    from pointcloudmatters_amd._lib import PointopsLibraryError
    from pointcloudmatters_amd.policy import cross_attention, gated_ffn, rotary_axes

    with pytest.raises(PointopsLibraryError):
        rotary_axes(_bf(2, 1, 8), torch.zeros(2, 1), (2,))
    with pytest.raises(PointopsLibraryError):
        cross_attention(_bf(1, 2, 1, 8), _bf(1, 2, 1, 8), _bf(1, 2, 1, 8))
    with pytest.raises(PointopsLibraryError):
        gated_ffn(_bf(2, 8), _bf(8, 8), _bf(8, 8), _bf(8, 8))


def test_rotary_refusals(model):
    from pointcloudmatters_amd.policy import rotary_axes

    x, c = _bf(4, 2, 16), torch.zeros(4, 2)
    rotary_axes(x, c, (3, 5))
    for bad in ((x.double(), c, (3, 5)), (x.half(), c, (3, 5)), (x, c.double(), (3, 5)), (x, c.half(), (3, 5))):
        with pytest.raises(TypeError):
            rotary_axes(*bad)
    for bad in ((x[0], c, (3, 5)), (x, c[:3], (3, 5)), (x, c, (3,)), (x, c, (4, 5)), (x, c, (0, 0)), (x, c, (-1, 5)), (x, torch.zeros(4, 0), ()),
                (x, c.requires_grad_(), (3, 5)), (_bf(4, 2, 16)[None, None], torch.zeros(4, 2), (3, 5)), (_bf(2, 4, 2, 16), torch.zeros(2, 2), (3, 5)),
                (_bf(4, 1, 600), torch.zeros(4, 1), (129,)), (x, torch.zeros(4, 9), (1,) * 9)):
        with pytest.raises(ValueError):
            rotary_axes(*bad)
    for base in (0.0, -3.0, float("nan")):
        with pytest.raises(ValueError):
            rotary_axes(x, torch.zeros(4, 2), (3, 5), base=base)


def test_cross_attention_refusals(model):
    from pointcloudmatters_amd.policy import cross_attention

    q, k = _bf(2, 3, 4, 16), _bf(2, 5, 2, 16)
    off = torch.tensor([3, 6], dtype=torch.int32)
    cross_attention(q, k, k)
    with pytest.raises(TypeError):
        cross_attention(q.float(), k, k)
    with pytest.raises(TypeError):
        cross_attention(q, k, k.half())
    for args, kw in (((q[0, 0], k, k), {}), ((q, k, _bf(2, 4, 2, 16)), {}), ((q, _bf(2, 5, 3, 16),) * 1 + (_bf(2, 5, 3, 16),), {}),
                     ((q, _bf(2, 5, 2, 24), _bf(2, 5, 2, 24)), {}), ((_bf(2, 3, 4, 12), _bf(2, 5, 2, 12), _bf(2, 5, 2, 12)), {}),
                     ((_bf(2, 3, 4, 136), _bf(2, 5, 2, 136), _bf(2, 5, 2, 136)), {}), ((q, _bf(3, 5, 2, 16), _bf(3, 5, 2, 16)), {}),
                     ((q, k, k), dict(q_offset=off)), ((q, k, k), dict(kv_offset=off)), ((q.flatten(0, 1), k, k), {}),
                     ((q.flatten(0, 1), k, k), dict(q_offset=off.float())), ((q.flatten(0, 1), k, k), dict(q_offset=off[None])),
                     ((q.flatten(0, 1), k, k), dict(q_offset=off[:1])), ((q.flatten(0, 1), k, k), dict(q_offset=off[:0])),
                     ((q, k, k), dict(key_padding_mask=torch.zeros(2, 4, dtype=torch.bool))), ((q, k, k), dict(key_padding_mask=torch.zeros(2, 5))),
                     ((q, k, k), dict(scale=0.0)), ((q, k, k), dict(scale=-1.0)), ((q, k, k), dict(scale=float("nan"))),
                     ((q, k, k), dict(scale=float("inf"))), ((q, _bf(2, 5, 0, 16), _bf(2, 5, 0, 16)), {})):
        with pytest.raises(ValueError):
            cross_attention(*args, **kw)


def test_gated_ffn_refusals(model):
    from pointcloudmatters_amd.policy import gated_ffn

    x, g, d, b, e = _bf(3, 8), _bf(12, 8), _bf(8, 12), _bf(12), _bf(8)
    gated_ffn(x, g, g, d, b, b, e)
    for bad in ((x.float(), g, g, d), (x, g.half(), g, d), (x, g, g, d, b.float())):
        with pytest.raises(TypeError):
            gated_ffn(*bad)
    for bad in ((x, g, _bf(11, 8), d), (_bf(3, 9), g, g, d), (x, g, g, g), (x, g, g, d, e), (x, g, g, d, b, b, b), (x, g[0], g[0], d),
                (_bf(()), g, g, d), (x, _bf(0, 8), _bf(0, 8), _bf(8, 0))):
        with pytest.raises(ValueError):
            gated_ffn(*bad)
    with pytest.raises(ValueError):
        gated_ffn(x, g, g, d, activation="tanh")


def test_entry_points_reject_before_they_touch_the_runtime():
    from pointcloudmatters_amd import _lib

    L, p = _lib.load(), 0x1000  # never dereferenced
    s = (ctypes.c_int * 2)(4, 4)
    rot = lambda D=16, axes=2, sec=s, base=1e4, ct=0, x=p: L.pcm_rotary_axes_hip(1, 4, 2, D, 1, x, 0, 32, 16, p, 0, 32, 16, ct, p, 0, 2, axes, sec, base, 0, 0, None)  # noqa: E731
    assert rot(D=14) == 1 and rot(axes=9) == 1 and rot(axes=0) == 1 and rot(base=0.0) == 1 and rot(ct=3) == 1 and rot(x=None) == 1
    assert rot(sec=(ctypes.c_int * 2)(100, 100), D=512) == 2 and rot(sec=(ctypes.c_int * 2)(-1, 4)) == 2 and rot(sec=(ctypes.c_int * 2)(0, 0)) == 1

    assert rot(D=1 << 22) == 2

    def xa(H=2, Hkv=1, D=64, q=p, q_ls=128, scale=1.0, out=p, ws=None, wsb=0, S=5, kv_rows=5, back=False):
        head = (1, H, Hkv, D, 3, 3, None, S, kv_rows, None, q, 0, q_ls, 64, p, 0, 64, 64, p, 0, 64, 64, None, 0, scale)
        if back:
            return L.pcm_cross_attn_backward_hip(*head, out, p, p, 0, 128, 64, p, p, p, p, ws, wsb, None)
        return L.pcm_cross_attn_forward_hip(*head, out, p, p, ws, wsb, None)

    for back in (False, True):
        assert xa(H=3, Hkv=2, back=back) == 2 and xa(D=60, back=back) == 2 and xa(D=136, back=back) == 2 and xa(q_ls=129, back=back) == 2
        assert xa(q=0x1008, back=back) == 2 and xa(q=None, back=back) == 1 and xa(scale=0.0, back=back) == 1 and xa(out=None, back=back) == 1
        assert xa(scale=float("nan"), back=back) == 1
        assert xa(S=0x7FFFFF00, back=back) == 2 and xa(H=1 << 10, Hkv=1 << 10, S=0x7FFFF000, back=back) == 2  # more threads than a launch takes
        assert xa(S=100000, back=back) == 1  # split keys need their workspace
    assert L.pcm_cross_attn_supported(8, 2, 64) == 1 and L.pcm_cross_attn_supported(8, 3, 64) == 0 and L.pcm_cross_attn_supported(8, 2, 4) == 0
    assert L.pcm_cross_attn_ws_bytes(1, 2, 1, 64, 3, 3, 0, 5, 5, 0, 0) == 0 < L.pcm_cross_attn_ws_bytes(1, 2, 1, 64, 3, 3, 0, 100000, 100000, 0, 0)

    def ff(R=40, E=16, F=8, act=0, x=p, a=None, u=None, h=p, ws=p, wsb=1 << 30):
        return L.pcm_gated_ffn_forward_hip(R, E, F, act, x, E, p, p, p, None, None, None, p, a, u, h, ws, wsb, None)

    assert ff(act=3) == 1 and ff(act=-1) == 1 and ff(x=None) == 1 and ff(a=p) == 1 and ff(h=None) == 1 and ff(h=0x1002) == 1 and ff(E=0) == 1
    assert ff(F=7, ws=None, wsb=0) == 1  # an odd width needs its padded copies
    assert ff(E=1 << 21) == 2 and ff(R=1 << 30) == 2 and ff(E=1 << 17, F=1 << 17) == 2
    fb = lambda wsb, dwu=p: L.pcm_gated_ffn_backward_hip(4, 16, 8, 0, p, 16, p, p, p, p, p, p, p, 16, p, p, dwu, p, None, None, None, p, wsb, None)  # noqa: E731
    need = L.pcm_gated_ffn_ws_bytes(4, 16, 8, 1)
    assert need > 0 and fb(need - 1) == 1 and fb(need, None) == 1
    assert L.pcm_gated_ffn_hidden_ld(1365) == 1408 and L.pcm_gated_ffn_hidden_ld(0) == 0
