"""rotary_axes, cross_attention and gated_ffn used together as one decoder layer over a batch of ragged clouds: against the same layer in
64 bits, forward and backward, captured and replayed, on two streams at once."""
import math

import pytest
import torch

from tests import layer_ops_ref as ref

pytestmark = pytest.mark.gpu
DEV = "cuda"
LENS, QUERIES, HEADS, KV, D, HIDDEN = [70, 5, 131], 12, 4, 2, 32, 90
E = HEADS * D
SECTIONS = (6, 5, 5)


def _problem(seed=0):
    g = torch.Generator().manual_seed(seed)
    n = lambda *s, scale=1.0: (torch.randn(*s, generator=g) * scale).bfloat16()  # noqa: E731
    b, t = len(LENS), sum(LENS)
    state = dict(x=n(b, QUERIES, E), memory=n(t, E), wq=n(E, E, scale=E ** -0.5), wk=n(KV * D, E, scale=E ** -0.5), wv=n(KV * D, E, scale=E ** -0.5),
                 wg=n(HIDDEN, E, scale=E ** -0.5), wu=n(HIDDEN, E, scale=E ** -0.5), wd=n(E, HIDDEN, scale=HIDDEN ** -0.5))
    where = dict(offset=torch.tensor(LENS).cumsum(0).to(torch.int32), q_coords=torch.rand(b, QUERIES, 3, generator=g) * 30,
                 coords=torch.randint(0, 160, (t, 3), generator=g, dtype=torch.int32))
    return state, where, n(b, QUERIES, E)


def _layer(s, w):
    """One pass on the device: rotary positions on queries and keys, attention over the packed clouds, the gated block, two residuals."""
    from pointcloudmatters_amd.policy import cross_attention, gated_ffn, rotary_axes

    q = rotary_axes((s["x"] @ s["wq"].t()).unflatten(-1, (HEADS, D)), w["q_coords"], SECTIONS)
    k = rotary_axes((s["memory"] @ s["wk"].t()).unflatten(-1, (KV, D)), w["coords"], SECTIONS)
    v = (s["memory"] @ s["wv"].t()).unflatten(-1, (KV, D))
    x = s["x"] + cross_attention(q, k, v, kv_offset=w["offset"]).flatten(-2)
    return x + gated_ffn(x, s["wg"], s["wu"], s["wd"])


def _turn(t, coords):
    half = sum(SECTIONS)
    a = torch.cat([coords[..., i, None].double() * torch.exp(-torch.arange(n).double() / n * math.log(10000.0)) for i, n in enumerate(SECTIONS)], -1)[..., None, :]
    u, v = t[..., :half], t[..., half:2 * half]
    return torch.cat([u * a.cos() - v * a.sin(), u * a.sin() + v * a.cos()], -1)


def _layer64(s, w):
    q = _turn((s["x"] @ s["wq"].t()).unflatten(-1, (HEADS, D)), w["q_coords"])
    k = _turn((s["memory"] @ s["wk"].t()).unflatten(-1, (KV, D)), w["coords"])
    v = (s["memory"] @ s["wv"].t()).unflatten(-1, (KV, D))
    rows, lo = [], 0
    for b, n in enumerate(LENS):
        kk, vv = (t[lo:lo + n].repeat_interleave(HEADS // KV, 1) for t in (k, v))
        p = torch.softmax(torch.einsum("lhd,shd->hls", q[b], kk) / math.sqrt(D), -1)
        rows.append(torch.einsum("hls,shd->lhd", p, vv).flatten(-2))
        lo += n
    x = s["x"] + torch.stack(rows)
    a, u = x @ s["wg"].t(), x @ s["wu"].t()
    return x + (a * torch.sigmoid(a) * u) @ s["wd"].t()


def test_together_against_64_bits():
    """Eight bf16 roundings lie between the inputs and the output (projection, turn, weights, attention, sum, gate, hidden, product), about
    as many again between the output and a gradient: 16 half steps in the 2-norm, far more than independent roundings add up to."""
    s, w, dy = _problem()
    d = {n: t.to(DEV).requires_grad_() for n, t in s.items()}
    y = _layer(d, {n: t.to(DEV) for n, t in w.items()})
    grads = torch.autograd.grad(y, list(d.values()), dy.to(DEV))
    e = {n: t.double().requires_grad_() for n, t in s.items()}
    y64 = _layer64(e, w)
    want = torch.autograd.grad(y64, list(e.values()), dy.double())
    for name, got, r in zip(("y", *s), (y, *grads), (y64, *want)):
        off = float((got.detach().double().cpu() - r.detach()).norm() / r.detach().norm())
        assert off <= 16 * ref.HALF, (name, off)


def test_second_derivatives_of_attention_and_block_are_refused():
    from pointcloudmatters_amd.policy import cross_attention, gated_ffn

    n = lambda *s: torch.randn(*s).bfloat16().to(DEV).requires_grad_()  # noqa: E731
    q, k, x, w, wd = n(1, 3, 2, 32), n(1, 9, 2, 32), n(4, 16), n(24, 16), n(16, 24)
    for leaf, f in ((q, lambda: cross_attention(q, k, k)), (x, lambda: gated_ffn(x, w, w, wd))):
        plain = torch.autograd.grad(f().float().pow(2).sum(), leaf)[0]
        (g,) = torch.autograd.grad(f().float().pow(2).sum(), leaf, create_graph=True)
        assert torch.equal(g, plain)
        with pytest.raises(RuntimeError, match="once_differentiable"):
            g.float().sum().backward()


def test_forward_and_backward_captured():
    from pointcloudmatters_amd import _graphs

    s, w, dy = _problem(1)
    d = {n: t.to(DEV).requires_grad_() for n, t in s.items()}
    wd, dy = {n: t.to(DEV) for n, t in w.items()}, dy.to(DEV)

    def step():
        y = _layer(d, wd)
        return y.detach(), torch.autograd.grad(y, list(d.values()), dy)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph, (y, grads) = _graphs.captured(step)
    for i in range(3):
        fresh, _, g = _problem(10 + i)
        with torch.no_grad():
            for n in d:
                d[n].copy_(fresh[n])
            dy.copy_(g)
        graph.replay()
        torch.cuda.synchronize()
        now = {n: t.detach().clone().requires_grad_() for n, t in d.items()}
        want = _layer(now, wd)
        assert torch.equal(y, want), i
        for a, b in zip(grads, torch.autograd.grad(want, list(now.values()), dy)):
            assert torch.equal(a, b), i


def test_a_captured_call_is_refused_while_an_eager_graph_of_its_leaves_lives():
    """The backward pass of such a capture would end the process (_graphs.guard_leaves): the forward call raises before there is one."""
    from pointcloudmatters_amd import _graphs
    from pointcloudmatters_amd.policy import cross_attention, gated_ffn, rotary_axes

    n = lambda *s: torch.randn(*s).bfloat16().to(DEV).requires_grad_()  # noqa: E731
    q, k, v, x, wg, wu, wd = n(1, 3, 2, 32), n(1, 9, 2, 32), n(1, 9, 2, 32), n(4, 16), n(24, 16), n(24, 16), n(16, 24)
    c = torch.zeros(1, 3, 1, device=DEV)
    calls = [lambda: rotary_axes(q, c, (4,)), lambda: cross_attention(q, k, v), lambda: gated_ffn(x, wg, wu, wd)]
    alive = [f() for f in calls]

    def refused():
        for f in calls:
            with pytest.raises(RuntimeError, match="eager graph"):
                f()
        return x.detach() + 1

    graph, _ = _graphs.captured(refused)
    graph.replay()
    torch.cuda.synchronize()
    for t in alive:  # the eager graphs themselves still work
        t.sum().backward()
    del alive, t
    graph, outs = _graphs.captured(lambda: [f() for f in calls])
    graph.replay()
    torch.cuda.synchronize()
    assert all(o.isfinite().all() for o in outs)


def test_a_captured_call_sees_the_leaves_behind_casts_and_views():
    from pointcloudmatters_amd import _graphs
    from pointcloudmatters_amd.policy import cross_attention, gated_ffn

    x, wg, wu, wd = (torch.randn(*s).to(DEV).requires_grad_() for s in ((4, 16), (24, 16), (24, 16), (16, 24)))
    q, k = torch.randn(1, 3, 64).bfloat16().to(DEV).requires_grad_(), torch.randn(1, 9, 64).bfloat16().to(DEV).requires_grad_()

    def cast():
        with torch.autocast("cuda", dtype=torch.bfloat16):
            return gated_ffn(x, wg, wu, wd)

    calls = [cast, lambda: cross_attention(*(t.unflatten(-1, (2, 32)) for t in (q, k, k)))]
    alive = [f() for f in calls]

    def refused():
        for f in calls:
            with pytest.raises(RuntimeError, match="eager graph"):
                f()
        return x.detach() + 1

    graph, _ = _graphs.captured(refused)
    graph.replay()
    torch.cuda.synchronize()
    for t in alive:
        t.sum().backward()


def test_two_captured_graphs_share_nothing():
    """Two graphs with workspaces of their own (split keys, padded copies), replayed one inside the other's work."""
    from pointcloudmatters_amd import _graphs
    from pointcloudmatters_amd.policy import cross_attention, gated_ffn

    g = torch.Generator().manual_seed(2)
    sets = []
    for i in range(2):
        q, k, v = ((torch.randn(1, n, 2, 64, generator=g)).bfloat16().to(DEV) for n in (3, 2000, 2000))
        x, wg, wu, wd = (torch.randn(*s, generator=g).bfloat16().to(DEV) for s in ((5, 33), (41, 33), (41, 33), (33, 41)))
        f = lambda q=q, k=k, v=v, x=x, wg=wg, wu=wu, wd=wd: (cross_attention(q, k, v), gated_ffn(x, wg, wu, wd))  # noqa: E731
        want = f()
        graph, out = _graphs.captured(f)
        sets.append((graph, out, want, f))  # f: a graph reads its inputs where they were, they have to live as long
    streams = [torch.cuda.Stream() for _ in sets]
    for _ in range(5):
        for st, (graph, *_) in zip(streams, sets):
            with torch.cuda.stream(st):
                graph.replay()
        torch.cuda.synchronize()
        for _, out, want, _ in sets:
            assert all(torch.equal(a, b) for a, b in zip(out, want))


def test_two_streams_at_once_give_what_one_gives():
    s, w, dy = _problem(3)
    d, wd = {n: t.to(DEV) for n, t in s.items()}, {n: t.to(DEV) for n, t in w.items()}
    want = _layer(d, wd)
    streams = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    outs = []
    for _ in range(4):
        for st in streams:
            with torch.cuda.stream(st):
                outs.append(_layer(d, wd))
    torch.cuda.synchronize()
    assert all(torch.equal(o, want) for o in outs)
