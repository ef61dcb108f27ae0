"""CPU: every launch that gated_ffn and cross_attention make, over the whole range of sizes their entry points accept, is one that the
runtime takes: at least one workgroup, fewer than 2^32 threads.  The entry points run on the host with their launches recorded."""
import os
import random

import pytest

from tests.wavesim import build as _build

pytestmark = pytest.mark.skipif(not os.path.exists(_build.CLANG), reason="needs the ROCm clang++ as host compiler (tests/wavesim)")
P = 0x10000  # never dereferenced


@pytest.fixture(scope="module")
def host():
    from tests.wavesim.launches import Recorder

    return Recorder(["cross_attn.hip", "gated_ffn.hip"])


def _good(host, what):
    made = host.launches()
    for kernel, grid, block in made:
        assert 0 < grid and 0 < block <= 1024 and grid * block < 1 << 32, (what, kernel, grid, block)
    return made


def _ffn(host, r, e, f, bias=True):
    n = host.pcm_gated_ffn_ws_bytes(r, e, f, 0)
    b = P if bias else None
    assert host.pcm_gated_ffn_forward_hip(r, e, f, 0, P, e, P, P, P, b, b, b, P, P, P, P, P, n, None) == 0, (r, e, f)
    made = _good(host, (r, e, f, "forward"))
    n = host.pcm_gated_ffn_ws_bytes(r, e, f, 1)
    assert host.pcm_gated_ffn_backward_hip(r, e, f, 0, P, e, P, P, P, P, P, P, P, e, P, P, P, P, b, b, b, P, n, None) == 0, (r, e, f)
    return made + _good(host, (r, e, f, "backward"))


@pytest.mark.parametrize("r", [9, 64, 128, 129, 200, 256])
def test_gated_block_of_few_rows_and_any_width(host, r):
    """One row of tiles with more column tiles than whole rounds of workgroups: the hidden widths around every whole round."""
    for e in (8, 512, 520, 4608, 65536, 65544, 1 << 17, 1 << 20):
        for f in sorted({w + d for w in range(4096, 131073, 4096) for d in (-64, 0, 1, 64, 1000)} | {1 << 20}):
            if e * f <= 1 << 32:
                assert _ffn(host, r, e, f)


def test_gated_block_over_its_whole_range(host):
    rng = random.Random(5)
    log = lambda hi: int(round(2 ** rng.uniform(0, hi)))  # noqa: E731
    for _ in range(4000):
        r, e, f = log(24), log(20), log(20)
        if e * f > 1 << 32 or r * (e + 8) > 1 << 33 or r * (f + 64) > 1 << 36:
            continue  # refused
        assert _ffn(host, r, e, f, bias=rng.random() < 0.5)


def _cross(host, b, h, hkv, d, l, s, q_packed=False, kv_packed=False):
    """Forward and backward of b sequences of l rows over s keys (packed sides: l and s rows a sequence on average); () if refused."""
    head = (b, h, hkv, d, l, b * l, P if q_packed else None, s, b * s, P if kv_packed else None)
    rows = []
    for n, heads in ((l, h), (s, hkv), (s, hkv)):
        rows += [P, n * heads * d, heads * d, d]
    ws = lambda back: host.pcm_cross_attn_ws_bytes(b, h, hkv, d, l, b * l, q_packed, s, b * s, kv_packed, back)  # noqa: E731
    rc = host.pcm_cross_attn_forward_hip(*head, *rows, None, 0, 0.125, P, P, P, P, ws(0), None)
    made = _good(host, (head, "forward"))
    assert rc in (0, 2) and (rc == 0) == bool(made), (head, rc)
    back = host.pcm_cross_attn_backward_hip(*head, *rows, None, 0, 0.125, P, P, P, l * h * d, h * d, d, P, P, P, P, P, ws(1), None)
    assert back == rc, (head, rc, back)
    return made + _good(host, (head, "backward"))


@pytest.mark.parametrize("d", [8, 32, 64, 72, 128])
def test_attention_of_single_queries_in_very_large_batches(host, d):
    """A workgroup a (sequence, key head): up to 512 threads.  With keys the key side's limit comes first; a memory without any has none."""
    limit = 0xFFFFF000 // 512
    for pairs in (1 << 20, limit // 8 * 8, limit // 8 * 8 + 8, 8800000, 0xFFFFF000 // 256 // 8 * 8):
        for hkv in (1, 8):
            for group in (1, 4):
                assert _cross(host, pairs // hkv, hkv * group, hkv, d, 1, 0)
                assert bool(_cross(host, pairs // hkv, hkv * group, hkv, d, 1, 2)) == (pairs <= limit)
    assert not _cross(host, (1 << 32) // 256, 1, 1, d, 1, 0)  # refused
    assert any("few" in k for k, *_ in _cross(host, 1000, 8, 8, d, 1, 2))


def test_attention_over_its_whole_range(host):
    rng = random.Random(6)
    log = lambda hi: int(round(2 ** rng.uniform(0, hi)))  # noqa: E731
    for _ in range(4000):
        hkv, group = log(5), log(5)
        b, l, s = log(24), log(20), log(24)
        if b * l > 1 << 31 or b * s > 1 << 31 or l * hkv * group * 128 > 1 << 40:
            continue
        _cross(host, b, hkv * group, hkv, 8 * rng.randint(1, 16), l, s, rng.random() < 0.5, rng.random() < 0.5)
