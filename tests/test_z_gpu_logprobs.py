"""Token log probabilities on the GPU (``ccut_token_logprobs``) against the oracle in 64 bits.

Tolerances: a term e^(x - m) in fp32 is off by a few 2^-24 of itself (the exponential) plus
2^-24 |x - m| (the rounding of the difference), the sums by less than 2^-18 of theirs (fp32 partial
sums of at most a few thousand positive terms), so log Z is off by less than 2^-16 and a log
probability lp by less than 2^-16 + 2^-23 |lp|; the entropy is a difference of log Z and a mean of
x - m whose size is at most the largest |lp| that carries probability, off by less than 2^-16 of it."""

from __future__ import annotations

import numpy as np
import pytest
import torch

from oracle import formats, serving

pytestmark = pytest.mark.gpu

EPS = 2.0 ** -16


@pytest.fixture(scope="module", autouse=True)
def _cuda():
    if not torch.cuda.is_available():
        pytest.skip("needs a CUDA device")
    from ccut_b200 import build
    build.build()


def _check(x, tokens, top, dtype=torch.float32, ld=None):
    from ccut_b200.logprobs import token_logprobs

    if dtype == torch.bfloat16:
        x = formats.bf16_bits_to_f32(formats.bf16_bits_from_f32(x))
    t = torch.from_numpy(x).cuda().to(dtype)
    if ld:
        buf = torch.full((x.shape[0], ld), float("nan"), dtype=dtype, device="cuda")
        buf[:, : x.shape[1]] = t
        t = buf[:, : x.shape[1]]
    r = token_logprobs(t, torch.from_numpy(np.asarray(tokens, np.int32)).cuda(), top_n=top)
    lp, ent, rank, ids, tlp = serving.token_logprobs(x, tokens, top)
    np.testing.assert_array_equal(r.rank.cpu().numpy(), rank)
    np.testing.assert_array_equal(r.top_ids.cpu().numpy(), ids)
    got = r.logprob.cpu().numpy()
    assert (np.isnan(got) == np.isnan(lp)).all()
    fin = np.isfinite(lp)
    assert (got[~fin & ~np.isnan(lp)] == -np.inf).all()
    assert (np.abs(got[fin] - lp[fin]) <= EPS + 2.0 ** -23 * np.abs(lp[fin])).all()
    assert (np.abs(r.entropy.cpu().numpy() - ent) <= EPS * (1 + np.abs(ent) + np.log(x.shape[1]))).all()
    tg = r.top_logprobs.cpu().numpy()
    f2 = np.isfinite(tlp)
    assert (tg[~f2] == -np.inf).all()
    assert (np.abs(tg[f2] - tlp[f2]) <= EPS + 2.0 ** -23 * np.abs(tlp[f2])).all()


@pytest.mark.parametrize("rows, vocab, top, dtype", [
    (1, 1, 1, torch.float32), (3, 2, 2, torch.bfloat16), (2, 31, 5, torch.float32), (5, 33, 32, torch.float32),
    (1, 1023, 20, torch.bfloat16), (7, 1025, 0, torch.float32), (1, 151936, 20, torch.float32),
    (8, 151936, 5, torch.float32), (33, 32003, 32, torch.bfloat16), (200, 5001, 7, torch.float32),
    (3, 102400, 32, torch.bfloat16), (700, 4097, 1, torch.float32),
])
def test_matches_oracle(rows, vocab, top, dtype):
    rng = np.random.default_rng(rows * 1000 + vocab)
    x = (rng.standard_normal((rows, vocab)) * rng.uniform(0.5, 6, (rows, 1))).astype(np.float32)
    tok = rng.integers(0, vocab, rows)
    tok[0] = vocab - 1
    if rows > 2:
        tok[1], tok[2] = int(x[1].argmax()), 0
    _check(x, tok, top, dtype)


@pytest.mark.parametrize("vocab", [700, 20000])
def test_ties_masks_and_orders(vocab):
    """Equal logits (the order falls back on the index), rows sorted up and down, a row with few
    finite logits, logits at the type's lowest value, zeros of both signs, far tokens, sharp rows,
    tokens outside the vocabulary."""
    rng = np.random.default_rng(vocab)
    x = rng.standard_normal((12, vocab)).astype(np.float32)
    x[0] = 0.25
    x[1] = np.sort(x[1])
    x[2] = -np.sort(x[2])
    x[3] = -np.inf
    x[3, [5, 600, 17]] = [1.0, 2.0, 1.0]
    x[4] = np.finfo(np.float32).min
    x[4, 77] = 0.0
    x[5] = np.where(np.arange(vocab) % 2, -0.0, 0.0)
    x[6] = rng.integers(-3, 3, vocab)
    x[7] *= 1000
    x[8] += 1e6
    x[9, ::3] = -1e30
    tok = [vocab - 1, 0, vocab - 1, 17, 3, 9, 250, int(x[7].argmin()), 1, 0, -1, vocab]
    _check(x, tok, 32)
    _check(x[:3], [1, 2, 699], 3, ld=vocab + 5)  # rows at odd addresses, the rest of the buffer NaN


def test_rows_that_have_no_distribution():
    """NaN, +inf or only -inf in a row: NaN probabilities for that row alone; ids stay in range, NaN last."""
    from ccut_b200.logprobs import token_logprobs

    x = torch.randn((5, 3000), device="cuda")
    want = token_logprobs(x, torch.arange(5, dtype=torch.int32, device="cuda"), top_n=4)
    y = x.clone()
    y[1, 7], y[2, 9], y[3] = float("nan"), float("inf"), -float("inf")
    r = token_logprobs(y, torch.arange(5, dtype=torch.int32, device="cuda"), top_n=4)
    for f in ("logprob", "entropy"):
        assert torch.isnan(getattr(r, f)[1:4]).all()
        assert torch.equal(getattr(r, f)[[0, 4]], getattr(want, f)[[0, 4]])
    assert torch.isnan(r.top_logprobs[1:4]).all()
    assert torch.equal(r.top_ids[[0, 1, 4]], want.top_ids[[0, 1, 4]])
    assert int(r.top_ids[2, 0]) == 9 and r.top_ids[3].tolist() == [0, 1, 2, 3]
    z = torch.full((1, 40), float("nan"), device="cuda")
    z[0, 11], z[0, 30] = -float("inf"), 2.0
    r = token_logprobs(z, torch.tensor([11], dtype=torch.int32, device="cuda"), top_n=5)
    assert r.top_ids[0].tolist() == [30, 11, 0, 1, 2] and int(r.rank) == 2


def test_captured_and_repeated_calls_agree():
    from ccut_b200.logprobs import token_logprobs

    x = torch.randn((4, 50000), device="cuda")
    tok = torch.tensor([1, 2, 3, 4], dtype=torch.int32, device="cuda")
    token_logprobs(x, tok, top_n=8)
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        out = token_logprobs(x, tok, top_n=8)
    for _ in range(2):
        x.copy_(torch.randn_like(x))
        tok.add_(100)
        g.replay()
        g.replay()
        for a, b in zip(out, token_logprobs(x, tok, top_n=8)):
            assert torch.equal(a, b)


@pytest.mark.parametrize("rows, vocab, top, dtype", [
    (2400, 8192, 20, torch.float32), (1200, 8200, 20, torch.float32), (40, 100001, 8, torch.float32),
    (4, 100000, 32, torch.bfloat16), (300, 50000, 32, torch.float32), (5000, 2500, 20, torch.bfloat16),
])
def test_runs_of_nan_are_last_in_the_order(rows, vocab, top, dtype):
    """NaN in whole stretches of a row, at its begin, in its middle, at its end, or nearly everywhere: the
    alternatives and the rank are the first of the rest, the same in every call."""
    from ccut_b200.logprobs import token_logprobs

    rng = np.random.default_rng(rows + vocab)
    x = rng.standard_normal((rows, vocab)).astype(np.float32)
    x = np.sort(x, 1) if rows == 1200 else x  # the best come last
    if dtype == torch.bfloat16:
        x = formats.bf16_bits_to_f32(formats.bf16_bits_from_f32(x))
    for r in range(rows):
        kind = r % 6
        if kind < 4:
            n = (600, vocab // 2, vocab // 8, vocab - 10)[kind]
            at = (0, 0, vocab // 8 * 3, 7)[kind]
            x[r, at: at + n] = np.nan
        elif kind == 4:
            x[r, vocab // 4:] = np.nan
    tok = rng.integers(0, vocab, rows).astype(np.int32)
    xd, td = torch.from_numpy(x).cuda().to(dtype), torch.from_numpy(tok).cuda()
    order = np.lexsort((np.broadcast_to(np.arange(vocab), x.shape), -x, np.isnan(x)))  # NaN last, then by value, then by index
    rank = np.argsort(order, 1)[np.arange(rows), tok] + 1
    for _ in range(5):
        r = token_logprobs(xd, td, top_n=top)
        np.testing.assert_array_equal(r.top_ids.cpu().numpy(), order[:, :top])
        np.testing.assert_array_equal(r.rank.cpu().numpy(), rank)
        nan = torch.from_numpy(np.isnan(x).any(1)).cuda()
        assert torch.equal(torch.isnan(r.logprob), nan) and torch.equal(torch.isnan(r.entropy), nan)
