"""Waits that run out inside the long query blocks of the 4-bit attention, without a fault: with a limit of 0
cycles an ordinary call's waits expire; it ends, says so in its status word, and the calls after it are
right."""

from __future__ import annotations

import ctypes as C

import numpy as np
import pytest
import torch

from ccut_b200 import _lib
from tests.test_z_gpu_kv4 import _bf16, _cuda, _dev, _pool  # noqa: F401

pytestmark = pytest.mark.gpu


@pytest.fixture
def budget():
    """Sets the limit of the waits; the default comes back after the test."""
    lib, was = _lib.load(), C.c_longlong()
    first = []

    def set_to(cycles):
        _lib.check(lib.ccut_debug_kv4_wait_budget(cycles, C.byref(was)), "ccut_debug_kv4_wait_budget")
        first.append(was.value)

    yield set_to
    if first:
        set_to(first[0])


@pytest.mark.parametrize("d, seq, L, dt", [(128, 40, 600, torch.bfloat16), (64, 40, 600, torch.bfloat16),
                                           (128, 33, 2700, torch.float32), (64, 70, 2700, torch.bfloat16)])
def test_a_call_whose_waits_run_out_ends(budget, d, seq, L, dt):
    from ccut_b200.blocks.attn_kv4 import kv4_attention

    rng = np.random.default_rng(d + seq)
    pool, _ = _pool(rng, 3, 1, 2, L, d)
    q = _dev(_bf16(rng.standard_normal((3, 16, seq, d))), torch.bfloat16)
    slots = _dev(np.array([2, 0, -1], np.int32))
    starts = _dev(np.array([L - seq, 17, 5], np.int32))
    want = kv4_attention(q, pool, 0, slots, starts, out_dtype=dt)
    lib = _lib.load()
    n = lib.ccut_kv4_attention_workspace_bytes(3, 16, 2, seq, L, d)
    ws, out = torch.zeros(n, dtype=torch.uint8, device="cuda"), torch.empty_like(want)
    s = torch.cuda.current_stream().cuda_stream

    def call():
        _lib.check(lib.ccut_kv4_attention(
            q.data_ptr(), *pool._pointers(0), slots.data_ptr(), starts.data_ptr(), 3, 16, 2, seq, d, L, L, pool.slot_rows,
            3, 0.0, 0.0, out.data_ptr(), _lib.OUT_BF16 if dt == torch.bfloat16 else _lib.OUT_F32, ws.data_ptr(), n, s),
            "ccut_kv4_attention")

    for _ in range(3):
        budget(0)
        call()
        assert lib.ccut_workspace_status(ws.data_ptr(), s) == _lib.ERR_TIMEOUT
        budget(2_000_000_000)
        call()
        assert lib.ccut_workspace_status(ws.data_ptr(), s) == 0
        assert torch.equal(out, want)
