"""cross_attention (csrc/cross_attn.hip) against softmax(scale q k^T) v in 64 bits, with element-wise bounds (tests/layer_ops_ref.py)."""
import math

import pytest
import torch

from tests import layer_ops_ref as ref

pytestmark = pytest.mark.gpu
DEV = "cuda"


def _offset(lens):
    return torch.tensor(lens, dtype=torch.int64).cumsum(0).to(torch.int32) if lens is not None else None


def _inputs(qs, ks, hkv, d, heads, seed=0, scale_q=1.5):
    g = torch.Generator().manual_seed(seed)
    q = (torch.randn(*qs, heads, d, generator=g) * scale_q).bfloat16()
    k, v = (torch.randn(*ks, hkv, d, generator=g).bfloat16() for _ in range(2))
    dout = torch.randn(*qs, heads, d, generator=g).bfloat16()
    return q, k, v, dout


def _run(q, k, v, dout, mask, q_off, kv_off, scale=None):
    from pointcloudmatters_amd.policy import cross_attention

    put = lambda t: t.to(DEV) if t is not None else None  # noqa: E731
    leaves = [t.to(DEV).requires_grad_() for t in (q, k, v)]
    out, lse = cross_attention(*leaves, key_padding_mask=put(mask), q_offset=put(q_off), kv_offset=put(kv_off), scale=scale, return_lse=True)
    grads = torch.autograd.grad(out, leaves, put(dout))
    with torch.no_grad():
        plain = cross_attention(*leaves, key_padding_mask=put(mask), q_offset=put(q_off), kv_offset=put(kv_off), scale=scale)
    assert torch.equal(plain, out)  # with and without the statistics
    return out, lse, grads


def _check(q, k, v, dout, mask, q_lens, kv_lens, scale=None, leaves=None):
    d = q.shape[-1]
    q_off, kv_off = _offset(q_lens), _offset(kv_lens)
    b = q.shape[0] if q.dim() == 4 else len(q_lens)
    q_spans = ref.spans(q_off, 0, b, q.shape[1])
    k_spans = ref.spans(kv_off, 0, b, k.shape[1])
    want = ref.attention(q.flatten(0, -3), k.flatten(0, -3), v.flatten(0, -3), mask.flatten() if mask is not None else None, q_spans, k_spans,
                         scale or 1.0 / math.sqrt(d), dout.flatten(0, -3))
    out, lse, grads = _run(*(leaves or (q, k, v, dout)), mask, q_off, kv_off, scale)
    for name, got, (r, e) in zip(("out", "lse", "dq", "dk", "dv"), (out, lse, *grads), want):
        ref.check(got.flatten(0, -3) if name != "lse" else got.flatten(0, -2), r, e, name)
    return out, grads


@pytest.mark.parametrize("b,l,s,heads,hkv,d", [
    (1, 1, 1, 1, 1, 8), (1, 1, 65, 2, 2, 64), (2, 7, 64, 4, 2, 32), (3, 33, 63, 2, 1, 64), (1, 130, 129, 2, 2, 64), (2, 50, 200, 6, 2, 80),
    (1, 9, 70, 5, 1, 96), (1, 40, 300, 4, 4, 128), (2, 3, 5, 2, 2, 120), (1, 129, 33, 3, 3, 40)])
def test_padded_sides(b, l, s, heads, hkv, d):
    _check(*_inputs((b, l), (b, s), hkv, d, heads), None, None, None)


@pytest.mark.parametrize("d", [32, 64, 128])
def test_masks_with_holes_and_an_entry_without_keys(d):
    q, k, v, dout = _inputs((4, 21), (4, 150), 2, d, 4, seed=1)
    g = torch.Generator().manual_seed(2)
    mask = torch.rand(4, 150, generator=g) < 0.4
    mask[1] = True            # nothing to read
    mask[2, :140] = True      # two whole tiles of keys masked, a few left
    mask[3, 64:128] = True    # a whole tile between visible ones
    out, grads = _check(q, k, v, dout, mask, None, None)
    assert (out[1] == 0).all() and (grads[0][1] == 0).all()
    assert (grads[1].cpu()[mask] == 0).all() and (grads[2].cpu()[mask] == 0).all()


def test_whatever_stands_in_masked_or_absent_rows_has_no_influence():
    from pointcloudmatters_amd.policy import cross_attention

    q, k, v, dout = _inputs((2, 10), (2, 100), 2, 64, 4, seed=3)
    mask = torch.zeros(2, 100, dtype=torch.bool)
    mask[:, 70:] = True
    mask[0, 3] = True
    clean = _run(q, k, v, dout, mask, None, None)
    for junk in (float("nan"), float("inf"), -float("inf"), torch.finfo(torch.bfloat16).min):
        k2, v2 = (t.masked_fill(mask[..., None, None], junk) for t in (k, v))
        out, lse, grads = _run(q, k2, v2, dout, mask, None, None)
        assert torch.equal(out, clean[0]) and torch.equal(lse, clean[1]) and all(torch.equal(x, y) for x, y in zip(grads, clean[2])), junk
    # packed: the neighbours of a sequence are other clouds' rows, the rows behind the last one are nobody's
    kp, vp = (torch.cat([t[0], torch.full((30, 2, 64), float("nan")).bfloat16()]) for t in (k, v))
    got = cross_attention(q[:1].to(DEV), kp.to(DEV), vp.to(DEV), kv_offset=torch.tensor([100], dtype=torch.int32, device=DEV))
    want = cross_attention(q[:1].to(DEV), k[:1].to(DEV), v[:1].to(DEV))
    assert torch.equal(got, want)


def test_a_visible_not_a_number_is_not_hidden():
    from pointcloudmatters_amd.policy import cross_attention

    q, k, v, _ = _inputs((1, 5), (1, 40), 1, 64, 1, seed=4)
    q[0, 2, 0, 0] = float("nan")
    out = cross_attention(q.to(DEV), k.to(DEV), v.to(DEV)).cpu()
    assert out[0, 2].isnan().all() and out[0, [0, 1, 3, 4]].isfinite().all()


@pytest.mark.parametrize("heads,hkv,d", [(2, 2, 64), (6, 2, 32), (3, 1, 128)])
@pytest.mark.parametrize("q_lens,kv_lens", [([5, 0, 130, 1], [65, 64, 0, 200]), ([1] * 70, [3] * 69 + [150]), ([128, 128], [128, 64]), ([3], [1])])
def test_packed_sides(heads, hkv, d, q_lens, kv_lens):
    q, k, v, dout = _inputs((sum(q_lens),), (sum(kv_lens),), hkv, d, heads, seed=5)
    _check(q, k, v, dout, None, q_lens, kv_lens)


def test_padded_queries_over_packed_states_with_a_mask_and_back():
    q, k, v, dout = _inputs((3, 20), (210,), 2, 64, 4, seed=6)
    mask = torch.rand(210, generator=torch.Generator().manual_seed(7)) < 0.3
    _check(q, k, v, dout, mask, None, [100, 10, 100])
    q, k, v, dout = _inputs((75,), (3, 90), 2, 64, 4, seed=8)
    _check(q, k, v, dout, None, [40, 5, 30], None)


def test_rows_behind_the_last_sequence_are_zero():
    q, k, v, dout = _inputs((50,), (90,), 2, 64, 2, seed=9)
    out, _, grads = _run(q, k, v, dout, None, _offset([30, 7]), _offset([40, 41]))
    assert (out[37:] == 0).all() and (grads[0][37:] == 0).all() and (grads[1][81:] == 0).all() and (grads[2][81:] == 0).all()
    want, _, wg = _run(q[:37], k[:81], v[:81], dout[:37], None, _offset([30, 7]), _offset([40, 41]))
    assert torch.equal(out[:37], want) and torch.equal(grads[1][:81], wg[1])


def test_offsets_past_the_rows_are_clamped():
    """A wrong offset reads nothing outside the tensors: the sequence ends where its rows do."""
    from pointcloudmatters_amd.policy import cross_attention

    q, k, v, _ = _inputs((20,), (90,), 1, 32, 1, seed=10)
    bad = torch.tensor([10, 500], dtype=torch.int32, device=DEV)
    good = torch.tensor([10, 90], dtype=torch.int32, device=DEV)
    qo = torch.tensor([8, 20], dtype=torch.int32, device=DEV)
    a, b = (cross_attention(q.to(DEV), k.to(DEV), v.to(DEV), q_offset=qo, kv_offset=o) for o in (bad, good))
    assert torch.equal(a, b)
    falling = torch.tensor([50, -3], dtype=torch.int32, device=DEV)  # a second sequence of negative length holds no key
    out = cross_attention(q.to(DEV), k.to(DEV), v.to(DEV), q_offset=qo, kv_offset=falling)
    assert (out[8:] == 0).all() and out[:8].isfinite().all()


def test_views_of_packed_projections():
    """k | v as halves of one projection, q with heads first in memory, channel-strided and misaligned views (copied), expanded queries."""
    g = torch.Generator().manual_seed(11)
    kv = torch.randn(2, 77, 2, 3, 64, generator=g).bfloat16()
    q, _, _, dout = _inputs((2, 13), (2, 77), 3, 64, 3, seed=12)
    d = kv.to(DEV)
    leaves = (q.to(DEV).transpose(1, 2).contiguous().transpose(1, 2), d[:, :, 0], d[:, :, 1], dout)
    _check(q, kv[:, :, 0], kv[:, :, 1], dout, None, None, None, leaves=leaves)
    k = kv[:, :, 0].contiguous()
    odd = torch.cat([k.reshape(-1)[:1], k.reshape(-1)]).to(DEV)[1:].view(k.shape)
    apart = kv[:, :, 1].to(DEV).transpose(-1, -2).contiguous().transpose(-1, -2)
    _check(q, k, kv[:, :, 1], dout, None, None, None, leaves=(q.to(DEV), odd, apart, dout.transpose(0, 1).contiguous().transpose(0, 1)))
    one = q[:1].expand(2, 13, 3, 64)
    _check(one, k, kv[:, :, 1], dout, None, None, None, leaves=(q[:1].to(DEV).expand(2, 13, 3, 64), k, kv[:, :, 1], dout))


@pytest.mark.parametrize("scale", [1e-3, 0.7, 3.0])
def test_scales(scale):
    _check(*_inputs((1, 20), (1, 100), 1, 64, 1, seed=13), None, None, None, scale=scale)


def test_far_apart_scores_do_not_overflow():
    q, k, v, dout = _inputs((1, 9), (1, 130), 1, 64, 1, seed=14, scale_q=100.0)
    _check(q, (k * 8), v, dout, None, None, None)


def test_empty_sides():
    from pointcloudmatters_amd.policy import cross_attention

    for qs, ks in (((2, 0), (2, 5)), ((2, 5), (2, 0)), ((0, 5), (0, 5))):
        q, k, v, dout = (t.to(DEV) for t in _inputs(qs, ks, 1, 32, 2))
        q.requires_grad_(), k.requires_grad_(), v.requires_grad_()
        out = cross_attention(q, k, v)
        assert out.shape == q.shape and (out == 0).all()
        for got, t in zip(torch.autograd.grad(out, (q, k, v), dout), (q, k, v)):
            assert got.shape == t.shape and (got == 0).all()


def test_gradient_against_differences():
    """Directional derivatives of sum(out * dout) with steps that bf16 holds exactly."""
    from pointcloudmatters_amd.policy import cross_attention

    q, k, v, dout = _inputs((1, 6), (1, 70), 1, 32, 2, seed=15, scale_q=1.0)
    _, _, grads = _run(q, k, v, dout, None, None, None)
    spans = [(0, 6)], [(0, 70)]
    for i in range(3):
        step = torch.randn(q.shape if i == 0 else k.shape, generator=torch.Generator().manual_seed(16 + i)).double() * 1e-4
        vals = []
        for sign in (1, -1):
            t = [x.double() for x in (q, k, v)]
            t[i] = t[i] + sign * step
            o = ref.attention(*(x.flatten(0, 1) for x in t), None, *spans, 1 / math.sqrt(32))[0][0]
            vals.append(float((o * dout.double().flatten(0, 1)).sum().detach()))
        slope, grad = (vals[0] - vals[1]) / 2, float((grads[i].double().cpu() * step).sum())
        size = float((grads[i].double().cpu() * step).pow(2).sum().sqrt())
        assert abs(slope - grad) <= 8 * ref.HALF * size * math.sqrt(step.numel()) ** 0.5 + 1e-9, (i, slope, grad)


@pytest.mark.parametrize("b,l,s,heads,hkv,d,train", [(1, 1, 5000, 2, 2, 64, True), (2, 1, 3000, 8, 1, 128, True), (1, 100, 2051, 2, 2, 64, True)])
def test_keys_shared_out_over_workgroups(b, l, s, heads, hkv, d, train):
    """Few rows over long states: the sums of the key ranges are joined, also where whole ranges are masked."""
    q, k, v, dout = _inputs((b, l), (b, s), hkv, d, heads, seed=17)
    mask = torch.zeros(b, s, dtype=torch.bool)
    mask[0, s // 4: 3 * s // 4] = True
    _check(q, k, v, dout, mask, None, None)


def test_runs_repeat_bit_for_bit():
    args = _inputs((2, 70), (2, 900), 2, 64, 4, seed=18)
    a, b = _run(*args, None, None, None), _run(*args, None, None, None)
    assert torch.equal(a[0], b[0]) and all(torch.equal(x, y) for x, y in zip(a[2], b[2]))


@pytest.mark.parametrize("b,l,s,heads,hkv,d", [(1, 16, 70, 4, 2, 64), (1, 17, 70, 4, 2, 64), (1, 32, 150, 1, 1, 128), (2, 33, 150, 2, 2, 32), (1, 30, 50, 7, 1, 32),
                                               (1, 9, 70, 24, 1, 8), (2, 11, 66, 13, 1, 104)])
def test_rows_of_a_key_head_around_a_tile(b, l, s, heads, hkv, d):
    """16 x 2, 32 x 1 rows: one 32-row tile; more: several.  Groups of 7, 13 and 24 heads: rows divided by what is no power of two."""
    _check(*_inputs((b, l), (b, s), hkv, d, heads, seed=21), None, None, None)


def test_few_packed_rows():
    _check(*_inputs((16,), (214,), 2, 64, 4, seed=22), None, [3, 0, 13], [100, 50, 64])


@pytest.mark.parametrize("b,l,s,heads,hkv,d", [(1, 1200, 40, 4, 2, 64), (2, 1100, 70, 2, 1, 128), (1, 1500, 20, 1, 1, 32)])
def test_rows_shared_out_over_workgroups(b, l, s, heads, hkv, d):
    """Few keys under many rows: the dK and dV sums of the row ranges are joined."""
    mask = torch.zeros(b, s, dtype=torch.bool)
    mask[0, 3:17] = True
    _check(*_inputs((b, l), (b, s), hkv, d, heads, seed=23), mask, None, None)


def test_long_states_under_many_rows_at_size():
    """Packed sides of several thousand rows and keys: the rule that shares long states out further."""
    mask = torch.zeros(8300, dtype=torch.bool)
    mask[100:2400] = True
    _check(*_inputs((4700,), (8300,), 4, 16, 8, seed=24), mask, [2300, 2400], [4200, 4100])


def test_rows_far_apart():
    """Row strides of 2^22 values and more are copied first; just below them, rows of a tile are up to 2^30 bytes apart."""
    q, k, v, dout = _inputs((1, 3), (1, 5), 1, 32, 2, seed=25)
    want = _run(q, k, v, dout, None, None, None)
    for step in ((1 << 22) - 8, 1 << 22):
        def far(t):
            rows = torch.zeros((t.shape[1] - 1) * step + t[0, 0].numel(), dtype=t.dtype, device=DEV)
            view = rows.as_strided(t.shape, (0, step, t.shape[3], 1))
            return view.copy_(t.to(DEV))

        got = _run(*(far(t) for t in (q, k, v, dout)), None, None, None)
        assert torch.equal(got[0], want[0]) and all(torch.equal(a, b) for a, b in zip(got[2], want[2])), step


def test_rows_shared_by_all_positions():
    """A stride of zero: one key and value for every position, which average to that value."""
    q, k, v, dout = _inputs((2, 9), (2, 1), 2, 64, 4, seed=26)
    wide = lambda t: t.expand(2, 70, 2, 64)  # noqa: E731
    _check(q, wide(k), wide(v), dout, None, None, None, leaves=(q, wide(k.to(DEV)), wide(v.to(DEV)), dout))


def test_some_gradients_only():
    from pointcloudmatters_amd.policy import cross_attention

    q, k, v, dout = _inputs((2, 40), (2, 90), 2, 64, 4, seed=27)
    want = _run(q, k, v, dout, None, None, None)[2]
    for keep in ((0,), (1,), (2,), (0, 2), (1, 2)):
        leaves = [t.to(DEV).requires_grad_(i in keep) for i, t in enumerate((q, k, v))]
        got = torch.autograd.grad(cross_attention(*leaves), [leaves[i] for i in keep], dout.to(DEV))
        assert all(torch.equal(g, want[i]) for g, i in zip(got, keep)), keep
