"""Query blocks of the 4-bit attention by their rows per kv head: tiles of 16 rows on caches that are cut into
parts, the sizes on both sides of the long-block kernel, and rows without a slot in long blocks.

Tolerances as in ``test_z_gpu_kv4``, with the long-block kernel's roundings from the row on that it takes (129 per
kv head): below, keys and values are exact, a score is off by at most 2^-16 of sum |q||k| scale and with fp32
output a probability by 2^-20."""

from __future__ import annotations

import numpy as np
import pytest
import torch

from oracle import serving
from tests.test_z_gpu_kv4 import _bf16, _check, _cuda, _dev, _pool  # noqa: F401

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("seq", [33, 50, 64, 203])
def test_long_blocks_without_a_slot_are_zeros(d, seq):
    """Sequences whose slot is outside the pool or whose start is negative, beside ones that have rows: every
    output of theirs is zero, however often and on however many SMs the call runs.  8 heads of one kv head:
    264, 400, 512 and 1624 rows, the last tiles of 8, 16 and 88 rows or whole."""
    from ccut_b200.blocks.attn_kv4 import kv4_attention

    rng = np.random.default_rng(d + seq)
    pool, host = _pool(rng, 3, 1, 1, seq + 60, d)
    B = 48
    slots = np.where(np.arange(B) % 8 == 3, np.arange(B) % 3, -1).astype(np.int32)
    slots[1::8] = 3
    starts = np.full(B, 17, np.int32)
    slots[5::8], starts[5::8] = 1, -4
    q = _bf16(rng.standard_normal((B, 8, seq, d)))
    qd = _dev(q, torch.bfloat16)
    none = torch.from_numpy((slots < 0) | (slots > 2) | (starts < 0)).cuda()
    first = None
    for _ in range(20):
        got = kv4_attention(qd, pool, 0, _dev(slots), _dev(starts))
        assert int(torch.count_nonzero(got[none])) == 0
        first = got if first is None else first
        assert torch.equal(got, first)
    few = [1, 3, 5, 8]  # against the oracle, which takes a while
    _check(pool, host, 0, q[few], slots[few], starts[few], out_dtype=torch.bfloat16)


LONG = 129  # query rows per kv head from which a call runs as a long block


def _tolerance(ref, q, k, v, scale, rows, out_bf16):
    sabs = scale * (np.abs(q) @ np.abs(k).swapaxes(-1, -2)).max()
    ds, uv = (2.0 ** -11, 2.0 ** -11) if rows >= LONG else (2.0 ** -16, 0.0)
    up = 2.0 ** -11 if out_bf16 or rows >= LONG else 2.0 ** -20
    out = 2.0 ** -8 if out_bf16 else 0.0
    return out * np.abs(ref) + 2 * np.abs(v).max() * (np.expm1(2 * ds * sabs) + 2 * up + uv + 2.0 ** -16)


@pytest.mark.parametrize("dt", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("d, heads, kvh, seq, lens", [
    (128, 17, 1, 1, [8000]), (128, 34, 2, 1, [1100, 5003]), (64, 8, 1, 5, [1100, 7001, 2]), (64, 20, 2, 4, [6999]),
    (128, 8, 2, 24, [4099, 1101]), (64, 12, 1, 8, [3000]), (128, 7, 1, 9, [1500, 2900, 40, 64, 1025]),
    (64, 1, 1, 127, [1300, 200, 3003]), (128, 2, 2, 127, [2222, 5000]), (128, 2, 1, 64, [1999, 3500, 64, 1100, 2500]),
    (64, 4, 2, 64, [4444]), (64, 5, 1, 25, [2048, 2049, 2047]), (128, 3, 1, 43, [1777, 3000]), (64, 129, 1, 1, [2600, 1030]),
    (64, 80, 1, 1, [130, 5, 4000]), (128, 4, 4, 31, [31, 200, 1200]), (64, 64, 1, 2, [2, 3, 1025, 1030]),
])
def test_rows_per_kv_head(d, heads, kvh, seq, lens, dt):
    """17 to 129 rows per kv head (odd counts, tiles of 16 that end inside a query or inside a group, tiles whose
    causal limit lies before their unit's last part), ragged caches with few and with many parts to join."""
    from ccut_b200.blocks.attn_kv4 import kv4_attention

    rng = np.random.default_rng(d + heads * 7 + seq)
    B, grp = len(lens), heads // kvh
    pool, host = _pool(rng, B, 1, kvh, max(max(lens), 1100) + 30, d)
    kvals, vvals = (serving.kv4_values(*host[n])[:, 0] for n in "kv")
    slots = rng.permutation(B).astype(np.int32)
    q = _bf16(rng.standard_normal((B, heads, seq, d)))
    starts = np.array([max(0, n - seq) for n in lens], np.int32)
    for kv_len in (None, max(lens)):
        got = kv4_attention(_dev(q, torch.bfloat16), pool, 0, _dev(slots), _dev(starts), kv_len=kv_len, out_dtype=dt)
        got = got.float().cpu().numpy()
        for b in range(B):
            n = min(kv_len or pool.max_len, int(starts[b]) + seq)
            k, v = kvals[slots[b]][:, :n], vvals[slots[b]][:, :n]
            ref = serving.kv4_attention(q[b], k, v, int(starts[b]))
            tol = _tolerance(ref, q[b].reshape(kvh, grp * seq, d), k, v, d ** -0.5, grp * seq, dt == torch.bfloat16)
            off = np.abs(got[b] - ref)
            assert (off <= tol).all(), (kv_len, b, (off / tol).max())
