"""CPU: which captured calls `_graphs.guard_leaves` refuses -- those whose leaves an eager graph through one of the guarded operators still
holds.  A capture is played by another stream number and a runtime that says it captures (tests/wavesim's host model of the device)."""
import os

import pytest
import torch

from tests.wavesim import build as _build

pytestmark = pytest.mark.skipif(not os.path.exists(_build.CLANG), reason="needs the ROCm clang++ as host compiler (tests/wavesim)")


@pytest.fixture
def capturing(monkeypatch):
    """capturing(f): f() as in a capture on a stream of its own"""
    from pointcloudmatters_amd import _lib
    from tests.wavesim.backend import simulated_device

    def run(f, stream=7):
        with monkeypatch.context() as m:
            m.setattr(torch.cuda, "is_current_stream_capturing", lambda: True)
            m.setattr(_lib, "raw_stream", lambda: stream)
            return f()

    with simulated_device(claim_cuda=True):
        yield run


def _refused(run, f):
    with pytest.raises(RuntimeError, match="eager graph"):
        run(f)


def _leaf(*s):
    return torch.randn(*s).bfloat16().requires_grad_()


def _layer(x, wq, k, v):
    from pointcloudmatters_amd.policy import cross_attention, rotary_axes

    q = (x @ wq.t()).unflatten(-1, (2, 16))
    return cross_attention(rotary_axes(q, torch.zeros(1, 3, 1), (4,)), k, v)


def test_leaves_behind_a_projection(capturing):
    """The operator's own input is no leaf: x and wq stand behind a product of the two."""
    x, wq, k, v = _leaf(1, 3, 32), _leaf(32, 32), _leaf(1, 5, 2, 16).detach(), _leaf(1, 5, 2, 16).detach()
    alive = _layer(x, wq, k, v)
    _refused(capturing, lambda: _layer(x, wq, k, v))
    _refused(capturing, lambda: _layer(x.detach(), wq, k, v))
    capturing(lambda: _layer(_leaf(1, 3, 32), _leaf(32, 32), k, v))  # other leaves
    del alive
    capturing(lambda: _layer(x, wq, k, v))


def test_an_eager_graph_is_seen_through_what_follows_it(capturing):
    from pointcloudmatters_amd.policy import gated_ffn

    x, wg, wu, wd = _leaf(2, 16), _leaf(24, 16), _leaf(24, 16), _leaf(16, 24)
    loss = (gated_ffn(x.detach(), wg, wu, wd) * 2).float().sum()
    loss.backward()
    _refused(capturing, lambda: gated_ffn(x, wg, wu, wd))  # run backward, but alive: so are the leaves' accumulation nodes
    del loss
    capturing(lambda: gated_ffn(x, wg, wu, wd))


def test_graphs_of_the_captures_own_stream_are_none_of_it(capturing):
    from pointcloudmatters_amd.policy import gated_ffn

    x, wg, wu, wd = _leaf(2, 16), _leaf(24, 16), _leaf(24, 16), _leaf(16, 24)
    kept = [capturing(lambda: gated_ffn(gated_ffn(x, wg, wu, wd), wg, wu, wd)) for _ in range(2)]
    _refused(lambda f: capturing(f, stream=8), lambda: gated_ffn(x, wg, wu, wd))
    del kept
    capturing(lambda: gated_ffn(x, wg, wu, wd), stream=8)


def test_a_call_without_gradients_is_never_refused(capturing):
    from pointcloudmatters_amd.policy import gated_ffn

    x, wg, wu, wd = _leaf(2, 16), _leaf(24, 16), _leaf(24, 16), _leaf(16, 24)
    alive = gated_ffn(x, wg, wu, wd)

    def forward_only():
        with torch.no_grad():
            return gated_ffn(x, wg, wu, wd)

    assert torch.equal(capturing(forward_only), alive)


def test_the_stream_is_that_of_the_tensors_device(capturing, monkeypatch):
    """Tensors of a device that is not the current one: their stream is asked for with their device current."""
    import contextlib

    from pointcloudmatters_amd import _lib
    from pointcloudmatters_amd.policy import rotary_axes

    current = ["another"]

    @contextlib.contextmanager
    def on_device(device):
        before, current[0] = current[0], str(device)
        yield
        current[0] = before

    monkeypatch.setattr(_lib, "on_device", on_device)
    monkeypatch.setattr(_lib, "raw_stream", lambda: {"another": 5, "cpu": 7}[current[0]])
    x = _leaf(1, 2, 8)
    turn = lambda: rotary_axes(x, torch.zeros(1, 1), (4,))  # noqa: E731
    alive = turn()
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: current[0] == "cpu")
    turn()  # the same stream, 7
    monkeypatch.setattr(_lib, "raw_stream", lambda: {"another": 7, "cpu": 8}[current[0]])
    with pytest.raises(RuntimeError, match="eager graph"):
        turn()
    del alive
