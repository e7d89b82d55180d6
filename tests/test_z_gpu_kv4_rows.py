"""Rows of the 4-bit attention that are easy to lose: rows without a slot in long query blocks."""

from __future__ import annotations

import numpy as np
import pytest
import torch

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
