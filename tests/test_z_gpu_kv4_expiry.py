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


def test_the_pool_keeps_the_status(budget):
    """The word of a pool keeps the error over later calls until it is read; wrapped pools share one; other pools
    know nothing of it."""
    from ccut_b200.blocks.attn_kv4 import Kv4Pool, kv4_attention

    rng = np.random.default_rng(1)
    wrapped, _ = _pool(rng, 2, 1, 1, 300, 64)
    own = Kv4Pool(2, 1, 1, 300, 64)
    q = _dev(_bf16(rng.standard_normal((2, 4, 50, 64))), torch.bfloat16)
    slots, starts = (_dev(np.array(a, np.int32)) for a in ([1, 0], [200, 9]))
    for pool, other in ((wrapped, own), (own, wrapped)):
        want = kv4_attention(q, pool, 0, slots, starts)
        budget(0)
        kv4_attention(q, pool, 0, slots, starts)
        budget(2_000_000_000)
        assert torch.equal(kv4_attention(q, pool, 0, slots, starts), want)
        assert other.workspace_status() == 0
        assert pool.workspace_status() == _lib.ERR_TIMEOUT and pool.workspace_status() == 0


@pytest.mark.parametrize("pool", [True, False])
def test_the_backend_raises(budget, pool):
    from ccut_b200.backend import GenericBackend
    from tests.gpu_helpers import gpu_layer
    from tests.model_helpers import make_tiny, quantized_layers
    from tests.test_z_gpu_engine import _decoder

    t = make_tiny(53, kv_heads=1, head_dim=64)
    dec = _decoder(t, [gpu_layer(ol.lw) for ol in quantized_layers(t, "awq_int4_g128", seed=53)])
    prompt = [int(x) for x in np.random.default_rng(2).integers(0, t.vocab, 200)]
    greedy = {"temperature": 0.0}
    be = GenericBackend(dec, max_seqs=2, max_len=256, pool=pool, kv_dtype="int4")
    want = be.generate_step(prompt, greedy)
    budget(0)
    with pytest.raises(TimeoutError):
        be.generate_step(prompt[:-1][::-1], greedy)
    with pytest.raises(TimeoutError):
        be.score(prompt)
    budget(2_000_000_000)
    assert be.generate_step(prompt, greedy) == want and dec.kv_status() == 0
