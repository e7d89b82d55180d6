"""Decoder and engine backend on the CPU with 4-bit caches, per-request adapters and log probabilities:
the host logic (which rows a step writes, which calls it makes, which caches it may reuse, what it
refuses), with stand-ins for the device calls."""

from __future__ import annotations

import numpy as np
import pytest
import torch

from tests.model_helpers import make_tiny
from tests.serving_helpers import banks, use_standins
from tests.test_model_cpu import _build, _build_mla, _rel, torch_ops  # noqa: F401
from tests.model_helpers import MLA_TINY


@pytest.fixture
def ops(torch_ops, monkeypatch):  # noqa: F811
    use_standins(monkeypatch)
    return torch_ops


# The same token in calls of different numbers of rows: a bf16 projection may be summed in another order and round
# to the neighbouring value, a step of 2^-7 of it, and with it a code of the cache; each of the two layers
# averages such steps over its 256 features, so the logits move by less than one step per layer.
SHAPE = 2 * 2.0 ** -7


def _prompts(t, lens, seed=0):
    rng = np.random.default_rng(seed)
    return [[int(x) for x in rng.integers(0, t.vocab, n)] for n in lens]


def test_int4_cache_steps_agree(ops):
    """Chunked prefill, single steps, batches of equal and unequal lengths, pooled and separate caches give
    the same logits; a truncated cache recomputes its tail; the logits stay near the bf16 caches'."""
    t = make_tiny(3, kv_heads=2)
    dec = _build(ops, t)
    a, b, c = _prompts(t, (9, 7, 7))
    ref = []
    for p in (a, b, c):
        cache = dec.new_cache(16, "int4")
        ref.append(dec.forward(p, cache, all_logits=True))
        assert cache.length == len(p)
        near = dec.forward(p, dec.new_cache(16), all_logits=True)
        assert _rel(ref[-1], near) < 0.25 and not torch.equal(ref[-1], near)
    pool = dec.new_pool(3, 16, "int4")
    ca, cb, cc = pool.cache(2), pool.cache(0), pool.cache(1)
    got = dec.forward_batch([(a[:4], ca, None), (b[:3], cb, None), (c[:3], cc, None)], all_logits=True)
    for g, r, n in zip(got, ref, (4, 3, 3)):
        assert _rel(g, r[:n]) < SHAPE
    got = dec.forward_batch([(b[3:5], cb, None), (c[3:5], cc, None)], all_logits=True)
    assert _rel(got[0], ref[1][3:5]) < SHAPE and _rel(got[1], ref[2][3:5]) < SHAPE
    for i in range(4, 9):
        assert _rel(dec.forward([a[i]], ca), ref[0][i]) < SHAPE
    ca.truncate(5)
    assert _rel(dec.forward(a[5:], ca), ref[0][-1]) < SHAPE
    lone = dec.new_cache(16, "int4")  # a cache of its own beside a pooled one
    lg = dec.forward_batch([(a, lone, None), (b[5:], cb, None)])
    assert _rel(lg[0], ref[0][-1]) < SHAPE and _rel(lg[1], ref[1][-1]) < SHAPE


def test_step_calls(ops, monkeypatch):
    """One append for a pool's spans; one attention call when they run the same number of tokens, with
    the longest length, else one per span."""
    t = make_tiny(4, layers=1)
    dec = _build(ops, t)
    pool = dec.new_pool(3, 20, "int4")
    calls = []
    app, att = ops.kv4_append, ops.kv4_attention
    monkeypatch.setattr(ops, "kv4_append", lambda *a, **k: (calls.append(("w", a[2].shape[0])), app(*a, **k))[1])
    monkeypatch.setattr(ops, "kv4_attention",
                        lambda *a, **k: (calls.append(("r", tuple(a[0].shape[::2]), k["kv_len"])), att(*a, **k))[1])
    cs = [pool.cache(i) for i in range(3)]
    p = _prompts(t, (6, 2, 2))
    dec.forward_batch([(x, c, None) for x, c in zip(p, cs)])
    assert calls == [("w", 10), ("r", (1, 6), 6), ("r", (1, 2), 2), ("r", (1, 2), 2)]
    calls.clear()
    dec.forward_batch([([1], c, None) for c in cs])
    assert calls == [("w", 3), ("r", (3, 1), 7)]


def test_refusals(ops):
    t = make_tiny(5, kv_heads=2)
    dec = _build(ops, t)
    with pytest.raises(ValueError):
        dec.new_cache(8, "fp8")
    with pytest.raises(ValueError):
        dec.forward_batch([([1], dec.new_cache(8), None), ([1], dec.new_cache(8, "int4"), None)])
    pool = dec.new_pool(2, 8, "int4")
    with pytest.raises(ValueError):
        dec.forward_batch([([1], pool.cache(1), None), ([1], pool.cache(1), None)])
    with pytest.raises(ValueError):
        dec.forward([1] * 9, pool.cache(0))
    with pytest.raises(ValueError):
        dec.forward([1], pool.cache(0), adapter=0)  # no banks
    bk = banks(t, 2, 8, 0, "cpu")
    with pytest.raises(ValueError):
        dec.set_adapters(bk[:1])
    with pytest.raises(ValueError):
        dec.set_adapters([{"ffn": bk[0]["o"]}, None])
    with pytest.raises(ValueError):
        dec.set_adapters([{"qkv": bk[0]["o"]}, None])
    with pytest.raises(ValueError):
        dec.set_adapters([bk[0], banks(t, 3, 8, 0, "cpu")[1]])
    assert dec.num_adapters == 0 and dec.layers[0].adapters == {}
    dec.set_adapters(bk)
    for bad in (2, -1, "0", True, 0.0):
        with pytest.raises(ValueError):
            dec.forward([1], pool.cache(0), adapter=bad)
    mla = _build_mla(ops, make_tiny(6, mla=MLA_TINY))
    with pytest.raises(NotImplementedError):
        mla.new_pool(1, 8, "int4")
    with pytest.raises(NotImplementedError):
        mla.set_adapters([None, None])
    from ccut_b200.backend import GenericBackend

    be = GenericBackend(dec, max_seqs=2, max_len=8)
    with pytest.raises(ValueError):
        be.generate_batch([([1, 2], {"adapter": 7})])
    assert not be._seqs  # refused before any cache was taken
    with pytest.raises(ValueError):
        GenericBackend(dec, kv_dtype="int8", pool=True)


def test_adapters_of_a_batch(ops):
    """Each sequence of a batch gets its own adapter; the answers are those of the sequences alone; an
    adapter changes them; none leaves the base model's."""
    t = make_tiny(7, kv_heads=2)
    dec = _build(ops, t)
    p = _prompts(t, (5, 5, 5))
    base = dec.forward(p[0], dec.new_cache(8), all_logits=True)
    dec.set_adapters(banks(t, 2, 8, 1, "cpu"))
    assert dec.num_adapters == 2
    assert torch.equal(dec.forward(p[0], dec.new_cache(8), all_logits=True), base)
    alone = [dec.forward(x, dec.new_cache(8), adapter=a, all_logits=True) for x, a in zip(p, (1, None, 0))]
    got = dec.forward_batch([(x, dec.new_cache(8), None, a) for x, a in zip(p, (1, None, 0))], all_logits=True)
    for g, r in zip(got, alone):
        assert _rel(g, r) < SHAPE
    assert _rel(alone[0], dec.forward(p[0], dec.new_cache(8), adapter=0, all_logits=True)) > 4 * SHAPE


def test_backend_keeps_adapters_apart(ops):
    """A cache serves only requests of the adapter it was computed with; prefix reuse within one adapter
    still works; log probabilities and scores answer the decoder's logits."""
    from ccut_b200.backend import GenericBackend

    t = make_tiny(8, kv_heads=2)
    dec = _build(ops, t)
    dec.set_adapters(banks(t, 2, 8, 2, "cpu"))
    prompt = _prompts(t, (6,))[0]
    for kw in ({"pool": True, "kv_dtype": "int4"}, {"kv_dtype": "int4"}, {}):
        be = GenericBackend(dec, max_seqs=3, max_len=16, **kw)
        greedy = [{"temperature": 0.0, "adapter": a} for a in (None, 0, 1)]
        first = [t_ for t_, _ in be.generate_batch([(prompt, g) for g in greedy], logprobs=3)]
        assert be.tokens_run == 18
        again = [be.generate_step(prompt + [tok], g, logprobs=2) for tok, g in zip(first, greedy)]
        assert be.tokens_run == 21  # one position each: the adapter's own cache was found
        for (tok, info), g, f in zip(again, greedy, first):
            lone = GenericBackend(dec, max_seqs=1, max_len=16, **({"kv_dtype": "int4"} if kw else {}))
            want = lone.logits_for(prompt + [f], g["adapter"]).double()
            lp = torch.log_softmax(want, 0)
            assert tok == int(lp.argmax()) and info["rank"] == 1 and info["top"][0][0] == tok and len(info["top"]) == 2
            near = 2 * SHAPE * float(want.abs().max())  # log Z and the logit move by at most that each
            assert abs(info["logprob"] - float(lp[tok])) < near
            assert abs(info["entropy"] + float((lp.exp() * lp).sum())) < 4 * near
    be = GenericBackend(dec, max_seqs=2, max_len=16, prefill_chunk=4)
    sc = be.score(prompt, top_n=1, adapter=1)
    lp = torch.log_softmax(dec.forward(prompt, dec.new_cache(8), adapter=1, all_logits=True).double(), 1)
    assert len(sc) == 5 and not be._seqs
    near = 2 * SHAPE * float(dec.forward(prompt, dec.new_cache(8), adapter=1, all_logits=True).abs().max())
    for i, s in enumerate(sc):
        assert abs(s["logprob"] - float(lp[i, prompt[i + 1]])) < near and 0 <= s["top"][0][0] < t.vocab
    assert be.score(prompt[:1]) == []


def test_alternatives_are_checked_before_anything_runs(ops):
    """A number of alternatives that no answer can hold is refused with no position computed, no cache taken."""
    from ccut_b200.backend import GenericBackend

    t = make_tiny(8, kv_heads=2)
    be = GenericBackend(_build(ops, t), max_seqs=2, max_len=16)
    prompt = _prompts(t, (6,))[0]
    for n, err in ((-1, ValueError), (1.5, ValueError), (True, ValueError), ("2", ValueError), (t.vocab + 1, ValueError),
                   (33, NotImplementedError)):
        if n == 33 and t.vocab < 33:
            err = ValueError
        for call in (lambda: be.generate_step(prompt, {"temperature": 0.0}, logprobs=n),
                     lambda: be.generate_batch([(prompt, None)], logprobs=n), lambda: be.score(prompt, top_n=n)):
            with pytest.raises(err):
                call()
    assert be.tokens_run == 0 and not be._seqs
    with pytest.raises(ValueError):
        be.score(prompt, adapter=0)
    assert be.tokens_run == 0


def test_new_adapters_take_no_old_cache(ops):
    """After ``set_adapters`` a cache of the old bank's adapter is not reused; one without an adapter is."""
    from ccut_b200.backend import GenericBackend

    t = make_tiny(8, kv_heads=2)
    dec = _build(ops, t)
    dec.set_adapters(banks(t, 2, 8, 2, "cpu"))
    prompt = _prompts(t, (6,))[0]
    be = GenericBackend(dec, max_seqs=3, max_len=16)
    for a in (None, 0):
        be.logits_for(prompt, a)
    assert be.tokens_run == 12
    dec.set_adapters(banks(t, 2, 8, 3, "cpu"))
    got = be.logits_for(prompt, 0)
    assert be.tokens_run == 18 and torch.equal(got, GenericBackend(dec, max_seqs=1, max_len=16).logits_for(prompt, 0))
    be.logits_for(prompt)
    assert be.tokens_run == 19


def test_config_kv_cache_dtype():
    from ccut_b200 import config
    from tests.test_config import AWQ

    assert config.quant_settings({"quant": {"kv_cache_dtype": "int4"}}, AWQ)["kv_cache_dtype"] == "int4"


def test_an_expired_wait_reaches_the_caller(ops, monkeypatch):
    """A status in the caches' word (as the attention leaves it when a bounded wait ran out) ends the step with
    TimeoutError, whichever call the step is; the caches are not reused, and the next call answers as a
    new backend does.  The bf16 caches have no such word."""
    from ccut_b200 import _lib
    from ccut_b200.backend import GenericBackend

    t = make_tiny(9, kv_heads=2)
    dec = _build(ops, t)
    prompt = _prompts(t, (6,))[0]
    assert dec.kv_status() == 0
    attend, stall = ops.kv4_attention, []

    def stalled(q, pool, *a, **k):
        if stall:
            pool.status.fill_(_lib.ERR_TIMEOUT)
        return attend(q, pool, *a, **k)

    monkeypatch.setattr(ops, "kv4_attention", stalled)
    greedy = {"temperature": 0.0}
    for pool in (True, False):
        be = GenericBackend(dec, max_seqs=3, max_len=16, pool=pool, kv_dtype="int4")
        want = be.generate_step(prompt, greedy)
        calls = [lambda: be.generate_step(prompt, greedy), lambda: be.generate_step(prompt, greedy, logprobs=1),
                 lambda: be.generate_batch([(prompt, greedy), (prompt[:4], None)]), lambda: be.logits_for(prompt),
                 lambda: be.score(prompt), lambda: be.forward_step(prompt), lambda: be.generate(prompt, 2)]
        for call in calls:
            stall.append(1)
            with pytest.raises(TimeoutError):
                call()
            stall.clear()
            assert all(s.ids == [] and s.cache.length == 0 for s in be._seqs) and dec.kv_status() == 0
            ran = be.tokens_run
            assert be.generate_step(prompt, greedy) == want and be.tokens_run == ran + len(prompt)
        _, past = be.forward_step(prompt[:3])
        stall.append(1)
        with pytest.raises(TimeoutError):
            be.forward_step(prompt, past)
        stall.clear()
        assert past.length == 3
        again = be.forward_step(prompt, be.forward_step(prompt[:3])[1])[0]
        assert torch.equal(be.forward_step(prompt, past)[0], again)


def test_status_words():
    from ccut_b200 import _lib
    from ccut_b200.blocks.attn_kv4 import Kv4Cache, Kv4Pool

    a, b = Kv4Pool(1, 1, 1, 8, 64, device="cpu"), Kv4Pool(1, 1, 1, 8, 64, device="cpu")
    a.status.fill_(_lib.ERR_TIMEOUT)
    assert b.workspace_status() == 0 and a.workspace_status() == _lib.ERR_TIMEOUT and a.workspace_status() == 0
    own = torch.zeros(1, dtype=torch.int32)
    assert Kv4Cache(1, 1, 8, 64, "cpu", own).pool.status is own
    assert Kv4Pool.wrap(a.k, a.k_par, a.v, a.v_par, own).status is own
    assert Kv4Pool.wrap(a.k, a.k_par, a.v, a.v_par).status is Kv4Pool.wrap(b.k, b.k_par, b.v, b.v_par).status
    for bad in (torch.zeros(2, dtype=torch.int32), torch.zeros(1), torch.zeros((), dtype=torch.int32)):
        with pytest.raises(ValueError):
            Kv4Pool.wrap(a.k, a.k_par, a.v, a.v_par, bad)
