"""Refusals and host logic of the 4-bit kv cache, token log probabilities and adapters on the CPU:
the C ABI's argument checks (each returns before it touches a device) and the Python checks."""

from __future__ import annotations

import ctypes as C

import numpy as np
import pytest
import torch

from ccut_b200 import _lib
from oracle import serving

FAKE = C.c_void_p(4096)
ODD = C.c_void_p(4100)
NULL = None
BF, F32 = _lib.OUT_BF16, _lib.OUT_F32


@pytest.fixture(scope="module")
def lib():
    from ccut_b200 import build

    build.build()
    return _lib.load()


def test_kv4_append_and_read_checks(lib):
    def append(*, k=FAKE, kd=BF, ks=256, hs=64, v=FAKE, vd=F32, tokens=3, kvh=2, d=64, slots=FAKE, kc=FAKE, kp=FAKE,
               L=10, rows=20, n=4):
        return lib.ccut_kv4_append(k, kd, ks, hs, v, vd, 256, 64, tokens, kvh, d, slots, FAKE, kc, kp, FAKE, FAKE, L,
                                   rows, n, NULL)

    assert append(d=96) == _lib.ERR_UNSUPPORTED
    for kw in ({"tokens": -1}, {"kvh": 0}, {"L": 0}, {"rows": 19}, {"n": -1}, {"kd": 7}, {"vd": -1}, {"k": NULL},
               {"v": NULL}, {"slots": NULL}, {"kc": NULL}, {"ks": 252}, {"hs": 60}, {"k": ODD}, {"kc": ODD},
               {"kp": C.c_void_p(4098)}):
        assert append(**kw) == _lib.ERR_INVALID, kw
    assert append(tokens=0, k=NULL) == _lib.OK

    def read(*, tokens=3, d=64, out=FAKE, dt=F32, kp=FAKE, rows=20):
        return lib.ccut_kv4_read(FAKE, kp, FAKE, FAKE, FAKE, FAKE, tokens, 2, d, 10, rows, 4, out, FAKE, dt, NULL)

    assert read(d=32) == _lib.ERR_UNSUPPORTED
    for kw in ({"tokens": -1}, {"out": NULL}, {"out": ODD}, {"dt": 3}, {"kp": NULL}, {"rows": 1}):
        assert read(**kw) == _lib.ERR_INVALID, kw
    assert read(tokens=0) == _lib.OK


def test_kv4_attention_checks(lib):
    def call(*, q=FAKE, kc=FAKE, vp=FAKE, slots=FAKE, batch=2, heads=8, kvh=2, seq=1, d=64, L=5000, kv_len=5000,
             rows=10000, n=4, out=FAKE, dt=BF, ws=FAKE, nb=1 << 30):
        return lib.ccut_kv4_attention(q, kc, FAKE, FAKE, vp, slots, FAKE, batch, heads, kvh, seq, d, L, kv_len, rows,
                                      n, 0.0, 0.0, out, dt, ws, nb, NULL)

    assert call(d=96) == _lib.ERR_UNSUPPORTED
    for kw in ({"batch": -1}, {"heads": 7}, {"heads": 0}, {"kvh": 0}, {"seq": -1}, {"kv_len": 5001}, {"kv_len": -1},
               {"rows": 9999}, {"n": -1}, {"dt": 5}, {"q": NULL}, {"out": NULL}, {"slots": NULL}, {"kc": NULL},
               {"q": ODD}, {"vp": C.c_void_p(4098)}, {"out": ODD}, {"ws": ODD}):
        assert call(**kw) == _lib.ERR_INVALID, kw
    assert call(batch=0) == _lib.OK and call(seq=0) == _lib.OK
    need = lib.ccut_kv4_attention_workspace_bytes(2, 8, 2, 1, 5000, 64)
    assert need > 256
    assert call(nb=need - 1) == _lib.ERR_WORKSPACE and call(ws=NULL) == _lib.ERR_WORKSPACE
    assert lib.ccut_kv4_attention_workspace_bytes(2, 7, 2, 1, 5000, 64) == 0
    assert lib.ccut_kv4_attention_workspace_bytes(2, 8, 2, 1, 5000, 80) == 0


def test_logprobs_checks(lib):
    def call(*, x=FAKE, dt=F32, rows=2, vocab=100, ld=100, tok=FAKE, top=5, ids=FAKE, lp=FAKE):
        return lib.ccut_token_logprobs(x, dt, rows, vocab, ld, tok, top, lp, FAKE, FAKE, ids, FAKE, NULL)

    for kw in ({"dt": 9}, {"rows": -1}, {"vocab": 0}, {"ld": 99}, {"top": -1}, {"top": 101, "vocab": 100}, {"x": NULL},
               {"tok": NULL}, {"ids": NULL}, {"lp": NULL}):
        assert call(**kw) == _lib.ERR_INVALID, kw
    assert call(top=33) == _lib.ERR_UNSUPPORTED
    assert call(rows=0, x=NULL) == _lib.OK


def test_lora_checks(lib):
    w = (C.c_int * 2)(64, 8)

    def call(*, x=FAKE, a=FAKE, ids=FAKE, tokens=3, inputs=128, rank=16, n=2, slices=2, widths=w, base=FAKE, bld=72,
             out=FAKE, old=72, dt=BF, ws=FAKE, nb=1 << 30):
        return lib.ccut_lora_add(x, a, FAKE, FAKE, ids, tokens, inputs, rank, n, slices, widths, base, bld, out, old,
                                 dt, ws, nb, NULL)

    for kw in ({"tokens": -1}, {"inputs": 0}, {"inputs": 100}, {"rank": 0}, {"rank": 8}, {"n": -1}, {"slices": 0},
               {"widths": NULL}, {"widths": (C.c_int * 2)(64, 4)}, {"widths": (C.c_int * 2)(64, -8)}, {"bld": 64},
               {"old": 76}, {"dt": 2}, {"x": NULL}, {"a": NULL}, {"ids": NULL}, {"base": NULL}, {"out": NULL},
               {"x": ODD}, {"out": ODD}):
        assert call(**kw) == _lib.ERR_INVALID, kw
    assert call(rank=144) == _lib.ERR_UNSUPPORTED  # 2 * 144 > 256
    assert call(slices=5, widths=(C.c_int * 5)(8, 8, 8, 8, 8)) == _lib.ERR_UNSUPPORTED
    assert call(tokens=0, x=NULL) == _lib.OK
    assert lib.ccut_lora_workspace_bytes(256, 128, 16, 2, 2) == 0  # a decode step takes none
    need = lib.ccut_lora_workspace_bytes(300, 128, 16, 2, 2)
    assert need > 256 and call(tokens=300, nb=need - 1) == _lib.ERR_WORKSPACE
    assert call(tokens=300, ws=ODD) == _lib.ERR_WORKSPACE and call(tokens=300, ws=NULL) == _lib.ERR_WORKSPACE


def test_python_checks():
    """The shims refuse wrong shapes, types and devices before any device call."""
    from ccut_b200.adapters import LoraBank
    from ccut_b200.blocks.attn_kv4 import Kv4Cache, Kv4Pool, kv4_append, kv4_attention
    from ccut_b200.logprobs import token_logprobs

    with pytest.raises(NotImplementedError):
        Kv4Pool(1, 1, 1, 8, 96, device="cpu")
    with pytest.raises(ValueError):
        Kv4Pool(0, 1, 1, 8, 64, device="cpu")
    pool = Kv4Pool(3, 2, 2, 8, 128, device="cpu")
    assert pool.bytes_per_position() == 2 * 2 * 2 * 36 * 2
    with pytest.raises(ValueError):
        pool.cache(3)
    c = pool.cache(2)
    assert c.length == 0 and c.max_len == 8
    with pytest.raises(ValueError):
        c.truncate(1)
    own = Kv4Cache(2, 2, 8, 128, device="cpu")
    assert own.pool.slots == 1 and own.slot == 0
    with pytest.raises(ValueError):
        pool._pointers(2)
    assert pool._pointers(1)[0] - pool._pointers(0)[0] == 2 * 8 * 64
    assert pool._pointers(1)[1] - pool._pointers(0)[1] == 2 * 8 * 2 * 4
    for bad in ((pool.k[0], pool.k_par, pool.v, pool.v_par), (pool.k, pool.k_par.float(), pool.v, pool.v_par),
                (pool.k, pool.k_par, pool.v[:2], pool.v_par),
                (pool.k.transpose(2, 3), pool.k_par.transpose(2, 3), pool.v.transpose(2, 3), pool.v_par.transpose(2, 3))):
        with pytest.raises(ValueError):
            Kv4Pool.wrap(*bad)
    i = torch.zeros(2, dtype=torch.int32)
    with pytest.raises(ValueError):
        kv4_append(pool, 0, torch.zeros(2, 2, 128), torch.zeros(2, 2, 128), i, i)  # CPU tensors
    with pytest.raises(ValueError):
        kv4_attention(torch.zeros(2, 4, 1, 128, dtype=torch.bfloat16), pool, 0, i, i)
    with pytest.raises(ValueError):
        token_logprobs(torch.zeros(2, 9), i)
    a, b = torch.zeros(2, 32, 64, dtype=torch.bfloat16), torch.zeros(2, 24, 16, dtype=torch.bfloat16)
    s = torch.ones(2)
    bank = LoraBank(a, b, s, [16, 8])
    assert (bank.rank, bank.inputs, bank.outputs, bank.adapters) == (16, 64, 24, 2)
    for args in ((a.float(), b, s, [16, 8]), (a, b, s, [24]), (a, b, s, [16, 4]), (a, b, s.double(), [16, 8]),
                 (a, b, s[:1], [16, 8]), (a[:1], b, s, [16, 8]), (a, b, s, [])):
        with pytest.raises(ValueError):
            LoraBank(*args)
    with pytest.raises(NotImplementedError):
        LoraBank(torch.zeros(1, 288, 64, dtype=torch.bfloat16), torch.zeros(1, 24, 144, dtype=torch.bfloat16), s[:1],
                 [16, 8])
    x = torch.zeros(3, 64, dtype=torch.bfloat16)
    with pytest.raises(ValueError):
        bank.add(torch.zeros(3, 24), x, torch.zeros(3, dtype=torch.int32))  # CPU tensors
    with pytest.raises(ValueError):
        bank.add(torch.zeros(3, 25), x, torch.zeros(3, dtype=torch.int32))
    with pytest.raises(ValueError):
        LoraBank.from_matrices([([(np.zeros((8, 64)), np.zeros((16, 4)))], 1.0)], device="cpu")
    with pytest.raises(ValueError):
        LoraBank.from_matrices([([None], 1.0)], device="cpu")
    padded = LoraBank.from_matrices([([(np.ones((8, 64)), np.ones((16, 8)))], 2.0)], device="cpu")
    assert padded.rank == 16 and float(padded.a.sum()) == 8 * 64 and float(padded.b.sum()) == 16 * 8


def test_oracle_format_rounds_within_a_step():
    """The oracle's 4-bit format: every value within half a step (plus the roundings of the pair) of
    its input, ends of the range included."""
    rng = np.random.default_rng(0)
    x = (rng.standard_normal((50, 128)) * np.exp(rng.uniform(-3, 3, (50, 1)))).astype(np.float32)
    c, p = serving.kv4_quantize(x)
    s = p[..., 0].astype(np.float64).repeat(64, -1)
    m = np.abs(p[..., 1].astype(np.float64)).repeat(64, -1)
    # half a step; the top end may be cut by 15 half-ulps of s, the bottom by half an ulp of m
    assert (np.abs(serving.kv4_values(c, p) - x) <= s * (0.5 + 15 * 2.0 ** -11) + m * 2.0 ** -11).all()


def test_wait_budget_checks():
    import ctypes as C

    from ccut_b200 import _lib, build

    build.build()
    lib, was = _lib.load(), C.c_longlong(-1)
    assert lib.ccut_debug_kv4_wait_budget(-1, C.byref(was)) == _lib.ERR_INVALID
    assert lib.ccut_debug_kv4_wait_budget(1 << 40, C.byref(was)) == _lib.ERR_INVALID  # above the kernels' own limit
    assert lib.ccut_debug_kv4_wait_budget(0, None) == _lib.ERR_INVALID and was.value == -1
    assert lib.ccut_debug_kv4_wait_budget(5, C.byref(was)) == 0 and was.value > 5
    default = was.value
    assert lib.ccut_debug_kv4_wait_budget(default, C.byref(was)) == 0 and was.value == 5


def test_status_word_checks(lib):
    def call(status, q=FAKE, batch=2):
        return lib.ccut_kv4_attention_reported(q, FAKE, FAKE, FAKE, FAKE, FAKE, FAKE, batch, 8, 2, 1, 64, 50, 50, 100, 4, 0.0,
                                               0.0, FAKE, BF, FAKE, 1 << 20, status, NULL)

    assert call(C.c_void_p(4098)) == _lib.ERR_INVALID
    assert call(FAKE, q=NULL) == _lib.ERR_INVALID
    assert call(NULL, batch=0) == _lib.OK and call(FAKE, batch=0) == _lib.OK


def test_positions_that_pass_31_bits(lib):
    """What a query may see, kv_len + seq, is an int in the kernels: a call past it is refused."""
    most = 2 ** 31 - 1

    def call(kv_len, seq):
        return lib.ccut_kv4_attention(FAKE, FAKE, FAKE, FAKE, FAKE, FAKE, FAKE, 1, 2, 1, seq, 64, most, kv_len, most, 1,
                                      0.0, 0.0, FAKE, BF, FAKE, 1 << 40, NULL)

    for kv_len, seq in ((most, 1), (most - 100, 64), (most - 4096 - 63, 64)):
        assert call(kv_len, seq) == _lib.ERR_UNSUPPORTED
