"""The 4-bit kv cache on the GPU (``ccut_kv4_append`` / ``_read`` / ``_attention``) against the
oracle's definitions: the format bit for bit, attention in 64 bits.

Tolerance of attention (``_tol``), from the roundings the kernels make.  Scores: a short query
block multiplies the exact codes by q rounded to 11 bits of its largest element's scale and sums
in fp32 (below 2^-16 of sum |q||k|); a long one reads k^ rounded to fp16 (2^-11 of each).  A score
error e changes a probability by a factor within e^{+-2 e} (its own and the sum's).  Probabilities
enter the second product as fp16 (2^-11) or, with fp32 output in a short block, as two fp16 parts
(2^-20); v^ is exact in a short block and fp16 (2^-11) in a long one.  An output is a convex
combination of values of size at most max|v|, so each of these costs at most twice its factor
times max|v|; the last rounding to bf16 costs 2^-8 of the value."""

from __future__ import annotations

import numpy as np
import pytest
import torch

from oracle import formats, serving

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module", autouse=True)
def _cuda():
    if not torch.cuda.is_available():
        pytest.skip("needs a CUDA device")
    from ccut_b200 import build
    build.build()


def _bf16(a):
    return formats.bf16_bits_to_f32(formats.bf16_bits_from_f32(np.asarray(a, np.float32)))


def _dev(a, dtype=None):
    t = torch.from_numpy(np.ascontiguousarray(a)).cuda()
    return t if dtype is None else t.to(dtype)


def _pool(rng, slots, layers, kvh, L, d, spread=1.0):
    from ccut_b200.blocks.attn_kv4 import Kv4Pool

    host = {}
    for n in "kv":
        x = rng.standard_normal((slots, layers, kvh, L, d)).astype(np.float32) * spread
        x += rng.standard_normal((1, layers, kvh, 1, d)).astype(np.float32)
        host[n] = serving.kv4_quantize(x)
    return Kv4Pool.wrap(*(_dev(a) for n in "kv" for a in host[n])), host


def _tol(ref, q, k, v, scale, seq_rows, out_bf16):
    long_block = seq_rows > 32  # more query rows per kv head than the short-block kernel takes
    sabs = scale * (np.abs(q) @ np.abs(k).swapaxes(-1, -2)).max()
    ds = sabs * (2.0 ** -11 if long_block else 2.0 ** -16)
    up = 2.0 ** -11 if out_bf16 or long_block else 2.0 ** -20
    uv = 2.0 ** -11 if long_block else 0.0
    vmax = np.abs(v).max()
    return (2.0 ** -8 if out_bf16 else 0.0) * np.abs(ref) + 2 * vmax * (np.expm1(2 * ds) + 2 * up + uv + 2.0 ** -16)


def _check(pool, host, layer, qh, slots, starts, kv_len=None, softcap=None, scale=None, out_dtype=torch.float32):
    from ccut_b200.blocks.attn_kv4 import kv4_attention

    kvals, vvals = (serving.kv4_values(*host[n])[:, layer] for n in "kv")
    got = kv4_attention(_dev(qh, torch.bfloat16), pool, layer, _dev(np.asarray(slots, np.int32)),
                        _dev(np.asarray(starts, np.int32)), kv_len=kv_len, softcap=softcap, scale=scale,
                        out_dtype=out_dtype)
    assert got.dtype == out_dtype and tuple(got.shape) == qh.shape
    got = got.float().cpu().numpy()
    B, H, S, d = qh.shape
    grp = H // pool.kv_heads
    L = pool.max_len if kv_len is None else kv_len
    for b in range(B):
        if not (0 <= slots[b] < pool.slots and starts[b] >= 0) or L == 0:
            assert np.count_nonzero(got[b]) == 0
            continue
        n = min(L, starts[b] + S)
        k, v = kvals[slots[b]][:, :n], vvals[slots[b]][:, :n]
        ref = serving.kv4_attention(qh[b], k, v, starts[b], scale, softcap)
        tol = _tol(ref, qh[b].reshape(pool.kv_heads, grp * S, d), k, v, scale or d ** -0.5, grp * S,
                   out_dtype == torch.bfloat16)
        bad = np.abs(got[b] - ref) - tol
        assert not (bad > 0).any() and np.isfinite(got[b]).all(), (b, bad.max(), np.abs(got[b] - ref).max())


@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_append_and_read_are_the_format(d, dtype):
    """Codes and params of random, constant, tiny, huge, one-sided and non-finite groups, from strided
    rows at scattered places; rows not named stay as they were."""
    from ccut_b200.blocks.attn_kv4 import Kv4Pool, kv4_append, kv4_read

    rng = np.random.default_rng(d)
    slots, layers, kvh, L, n = 3, 2, 3, 40, 37
    x = rng.standard_normal((2, n, kvh, d)).astype(np.float32)
    x[:, 1] = 0.0
    x[:, 2] = 3.14159
    x[:, 3] *= 1e-9
    x[:, 4] *= 3e4
    x[:, 5] = 1e5 * np.sign(x[:, 5])
    x[:, 6] = 100 + 0.01 * x[:, 6]
    x[:, 7] = np.arange(d) % 16  # exact codes
    x[:, 8] = (np.arange(d) % 31) * 0.5  # halves: ties of the rounding
    x[:, 9, 0, 3], x[:, 10, 1, d - 1], x[:, 11, 2, 0] = np.nan, np.inf, -np.inf
    x[:, 12] = np.where(np.arange(d) == 5, 1.0, 0.0)
    if dtype == torch.bfloat16:
        x = formats.bf16_bits_to_f32(formats.bf16_bits_from_f32(x))
    pool = Kv4Pool(slots, layers, kvh, L, d)
    for t in (pool.k, pool.v):
        t.fill_(0xA5)
    where = rng.permutation(slots * L)[:n]
    sl, pos = (where // L).astype(np.int32), (where % L).astype(np.int32)
    sl[20], pos[21], sl[22], pos[23] = -1, L, slots, -5  # skipped
    k = torch.empty((kvh, n, d + 8), dtype=dtype, device="cuda")[:, :, :d].transpose(0, 1)  # strided rows
    k.copy_(_dev(x[0]))
    v = _dev(x[1], dtype)
    before = [t.clone() for t in (pool.k, pool.k_par, pool.v, pool.v_par)]
    kv4_append(pool, 1, k, v, _dev(sl), _dev(pos))
    rk, rv = kv4_read(pool, 1, _dev(sl), _dev(pos))
    bk, _ = kv4_read(pool, 1, _dev(sl), _dev(pos), torch.bfloat16)
    for name, codes, par, back, xs in (("k", pool.k, pool.k_par, rk, x[0]), ("v", pool.v, pool.v_par, rv, x[1])):
        want_c, want_p = (before[0] if name == "k" else before[2]).cpu().numpy().copy(), None
        want_p = (before[1] if name == "k" else before[3]).cpu().numpy().copy()
        c, p = serving.kv4_quantize(xs)
        vals = serving.kv4_values(c, p)
        for t in range(n):
            if 0 <= sl[t] < slots and 0 <= pos[t] < L:
                want_c[sl[t], 1, :, pos[t]], want_p[sl[t], 1, :, pos[t]] = c[t], p[t]
            else:
                vals[t] = 0
        np.testing.assert_array_equal(codes.cpu().numpy(), want_c)
        np.testing.assert_array_equal(par.cpu().numpy(), want_p)  # NaN equal to NaN
        np.testing.assert_array_equal(back.cpu().numpy(), vals.astype(np.float32))
    np.testing.assert_array_equal(bk.float().cpu().numpy(), rk.to(torch.bfloat16).float().cpu().numpy())


@pytest.mark.parametrize("d, heads, kvh, seq, lens, dt", [
    (128, 32, 4, 1, [1, 2, 15, 16, 17, 63, 64, 65, 255, 257, 600], torch.bfloat16),
    (128, 8, 4, 1, [700, 33, 5], torch.float32),
    (64, 16, 2, 1, [1, 31, 32, 33, 900], torch.float32),
    (64, 7, 1, 1, [129, 40], torch.bfloat16),
    (64, 5, 5, 3, [3, 70, 300], torch.float32),
    (128, 16, 2, 2, [2, 3, 128, 513], torch.bfloat16),
    (128, 24, 1, 1, [77, 1000], torch.float32),
    (64, 32, 2, 2, [50, 1001], torch.bfloat16),
    (128, 4, 4, 31, [31, 200], torch.float32),
    (128, 32, 4, 33, [33, 34, 161, 290], torch.bfloat16),
    (64, 8, 2, 70, [70, 127, 400], torch.bfloat16),
    (128, 6, 2, 129, [129, 300], torch.float32),
    (64, 3, 3, 200, [200, 329], torch.float32),
    (128, 80, 1, 1, [130, 5], torch.bfloat16),
])
def test_attention_matches_oracle(d, heads, kvh, seq, lens, dt):
    """Lengths around every tile edge, group sizes from 1 to 80, decode rows, short and long blocks,
    slots in another order than the rows, one of two layers."""
    rng = np.random.default_rng(d + heads + seq)
    B, L = len(lens), max(lens) + 9
    pool, host = _pool(rng, B + 1, 2, kvh, L, d)
    slots = rng.permutation(B + 1)[:B]
    qh = _bf16(rng.standard_normal((B, heads, seq, d)))
    starts = [n - seq for n in lens]
    _check(pool, host, 1, qh, slots, starts, out_dtype=dt)
    _check(pool, host, 0, qh, slots, starts, kv_len=max(lens), out_dtype=dt)


@pytest.mark.parametrize("seq", [1, 2, 40])
def test_attention_edges(seq):
    """Slots outside the pool and negative starts give zero rows; starts past the cache see all of it;
    kv_len cuts what a row sees, kv_len 0 leaves nothing; scale and soft cap; sharp scores."""
    rng = np.random.default_rng(seq)
    pool, host = _pool(rng, 3, 2, 2, 150, 64)
    qh = _bf16(rng.standard_normal((6, 8, seq, 64)) * 6)
    slots, starts = [2, 0, -1, 3, 1, 1], [100, 2 ** 31 - 1, 5, 5, -1, 0]
    for kw in ({}, {"kv_len": 90}, {"kv_len": 0}, {"softcap": 5.0}, {"scale": 0.3}, {"out_dtype": torch.bfloat16}):
        _check(pool, host, 1, qh, slots, starts, **kw)


@pytest.mark.parametrize("seq", [1, 3, 70])
def test_what_is_not_seen_never_reaches_a_row(seq):
    """NaN and infinite values in positions past a row's last, in other slots and in other layers
    leave its output as it is; a NaN that a row sees makes that row NaN and no other."""
    from ccut_b200.blocks.attn_kv4 import kv4_attention

    rng = np.random.default_rng(seq + 5)
    n = 100 + seq
    pool, host = _pool(rng, 2, 2, 1, 300, 128)
    q = _dev(_bf16(rng.standard_normal((1, 4, seq, 128))), torch.bfloat16)
    one = (torch.tensor([1], dtype=torch.int32, device="cuda"), torch.tensor([n - seq], dtype=torch.int32, device="cuda"))
    clean = kv4_attention(q, pool, 1, *one)
    for par in (pool.k_par, pool.v_par):
        par[0] = float("nan")
        par[:, 0] = float("inf")
        par[1, 1, :, n:] = float("nan")
    assert torch.equal(kv4_attention(q, pool, 1, *one), clean)
    if seq > 1:
        for par in (pool.k_par, pool.v_par):
            keep = par.clone()
            par[1, 1, :, n - 1, 0] = float("nan")
            got = kv4_attention(q, pool, 1, *one)
            assert torch.equal(got[:, :, :-1], clean[:, :, :-1])
            assert torch.isnan(got[:, :, -1]).any(-1).all()
            par.copy_(keep)


def test_scales_of_very_different_size():
    """Value scales that span fp16's range within one row's positions."""
    rng = np.random.default_rng(3)
    from ccut_b200.blocks.attn_kv4 import Kv4Pool

    for d, seq in ((128, 1), (64, 2), (64, 40)):
        L = 400
        x = rng.standard_normal((2, 1, 1, 1, L, d)).astype(np.float32)
        x[1] *= np.exp(rng.uniform(-12, 9, (1, 1, 1, L, 1))).astype(np.float32)
        host = {n: serving.kv4_quantize(x[i]) for i, n in enumerate("kv")}
        pool = Kv4Pool.wrap(*(_dev(a) for n in "kv" for a in host[n]))
        qh = _bf16(rng.standard_normal((1, 4, seq, d)))
        _check(pool, host, 0, qh, [0], [L - seq], out_dtype=torch.bfloat16)


def test_offsets_past_32_bits():
    """Rows whose code offset passes 2^32 bytes: a pool of 66 slots of 2^20 positions (4.4 GB of k)."""
    from ccut_b200.blocks.attn_kv4 import Kv4Pool, kv4_append, kv4_attention, kv4_read

    L, slots, d = 1 << 20, 66, 128
    pool = Kv4Pool.wrap(*(torch.empty(s, dtype=t, device="cuda") for t, s in
                          ((torch.uint8, (slots, 1, 1, L, d // 2)), (torch.float16, (slots, 1, 1, L, 2, 2))) * 2))
    rng = np.random.default_rng(0)
    x = rng.standard_normal((2, 50, 1, d)).astype(np.float32)
    sl = torch.full((50,), slots - 1, dtype=torch.int32, device="cuda")
    pos = torch.arange(50, dtype=torch.int32, device="cuda")
    kv4_append(pool, 0, _dev(x[0]), _dev(x[1]), sl, pos)
    rk, rv = kv4_read(pool, 0, sl, pos)
    vals = [serving.kv4_values(*serving.kv4_quantize(a)) for a in x]
    np.testing.assert_array_equal(rk.cpu().numpy(), vals[0].astype(np.float32))
    np.testing.assert_array_equal(rv.cpu().numpy(), vals[1].astype(np.float32))
    for seq in (1, 50):
        qh = _bf16(rng.standard_normal((1, 4, seq, d)))
        got = kv4_attention(_dev(qh, torch.bfloat16), pool, 0, sl[:1], torch.full_like(sl[:1], 50 - seq), kv_len=50)
        k, v = vals[0].transpose(1, 0, 2), vals[1].transpose(1, 0, 2)
        ref = serving.kv4_attention(qh[0], k, v, 50 - seq)
        tol = _tol(ref, qh[0].reshape(1, -1, d), k, v, d ** -0.5, 4 * seq, True)
        assert (np.abs(got[0].float().cpu().numpy() - ref) <= tol).all()


@pytest.mark.parametrize("seq", [1, 64])
def test_captured_call_replays_on_new_inputs(seq):
    """A captured step (append, then attention) replayed after its inputs changed gives the eager
    answer, twice the same bits; two streams with calls of their own do not disturb each other."""
    from ccut_b200.blocks.attn_kv4 import kv4_append, kv4_attention

    rng = np.random.default_rng(seq)
    pool, _ = _pool(rng, 2, 1, 2, 500, 128)
    q = _dev(_bf16(rng.standard_normal((2, 16, seq, 128))), torch.bfloat16)
    kv = torch.randn((2, 2 * seq, 2, 128), device="cuda")
    slots = torch.tensor([1, 0], dtype=torch.int32, device="cuda")
    starts = torch.tensor([200, 333], dtype=torch.int32, device="cuda")
    sl = slots.repeat_interleave(seq).contiguous()

    def step():
        pos = (starts[:, None] + torch.arange(seq, dtype=torch.int32, device="cuda")).reshape(-1)
        kv4_append(pool, 0, kv[0], kv[1], sl, pos)
        return kv4_attention(q, pool, 0, slots, starts)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        out = step()
    for _ in range(2):
        q.copy_(torch.randn_like(q, dtype=torch.float32))
        kv.copy_(torch.randn_like(kv))
        starts.add_(1)
        g.replay()
        first = out.clone()
        g.replay()
        assert torch.equal(out, first)
        assert torch.equal(first, step())
    other, _ = _pool(rng, 2, 1, 2, 500, 128)
    want = [kv4_attention(q, p, 0, slots, starts) for p in (pool, other)]
    torch.cuda.synchronize()
    with torch.cuda.stream(side):
        a = [kv4_attention(q, pool, 0, slots, starts) for _ in range(20)]
    b = [kv4_attention(q, other, 0, slots, starts) for _ in range(20)]
    torch.cuda.synchronize()
    assert all(torch.equal(x, want[0]) for x in a) and all(torch.equal(x, want[1]) for x in b)


@pytest.mark.parametrize("seq", [1, 3, 70])
def test_values_at_the_top_of_the_range(seq):
    """A group of +-1e5 is held as +-65504, its top up to half a step of fp16 more.  The row that
    sees it gets it; the rows before it, whose mask hides it, keep their bits."""
    from ccut_b200.blocks.attn_kv4 import kv4_append, kv4_attention

    rng = np.random.default_rng(seq + 50)
    n, d = 100 + seq, 128
    pool, host = _pool(rng, 1, 1, 1, 200, d)
    q = _bf16(rng.standard_normal((1, 4, seq, d)))
    at = (torch.zeros(1, dtype=torch.int32, device="cuda"), torch.full((1,), n - seq, dtype=torch.int32, device="cuda"))
    clean = kv4_attention(_dev(q, torch.bfloat16), pool, 0, *at)
    k = host["k"]
    row = serving.kv4_values(*k)[0, 0, :, n - 1][None].astype(np.float32)
    big = np.where(np.arange(d) % 3 == 0, -1e5, 1e5).astype(np.float32)[None, None]
    kv4_append(pool, 0, _dev(row), _dev(big), at[0], torch.full_like(at[0], n - 1))
    host["k"], host["v"] = ((pool.k.cpu().numpy(), pool.k_par.cpu().numpy()), (pool.v.cpu().numpy(), pool.v_par.cpu().numpy()))
    got = kv4_attention(_dev(q, torch.bfloat16), pool, 0, *at)
    assert torch.equal(got[:, :, :-1], clean[:, :, :-1])
    assert np.abs(serving.kv4_values(*host["v"])[0, 0, 0, n - 1]).max() >= 65504
    _check(pool, host, 0, q, [0], [n - seq])


@pytest.mark.parametrize("d, heads, kvh, seq, lens, dt", [
    (128, 32, 4, 1, [1, 1025, 3000, 64, 1, 2047], torch.bfloat16),
    (128, 8, 1, 1, [1100] * 40, torch.float32),
    (128, 4, 2, 5, [5, 1300, 2500], torch.float32),
    (64, 16, 2, 2, [1500, 40, 2001], torch.bfloat16),
    (64, 8, 1, 1, [20011], torch.bfloat16),
    (64, 12, 1, 1, [9000, 3], torch.float32),
    (128, 16, 2, 40, [1401, 2600], torch.bfloat16),
    (64, 16, 1, 20, [6007], torch.float32),
])
def test_long_caches(d, heads, kvh, seq, lens, dt):
    """Lengths at which a sequence is cut into parts that are joined, beside ones that are not; with
    the pool's length as the bound and with the longest sequence's."""
    rng = np.random.default_rng(d + heads + seq + 1)
    B, L = len(lens), max(max(lens), 1100) + 70
    pool, host = _pool(rng, B, 1, kvh, L, d)
    slots = rng.permutation(B)
    qh = _bf16(rng.standard_normal((B, heads, seq, d)))
    starts = [n - seq for n in lens]
    _check(pool, host, 0, qh, slots, starts, out_dtype=dt)
    _check(pool, host, 0, qh, slots, starts, kv_len=max(lens), out_dtype=dt, softcap=20.0)


@pytest.mark.parametrize("d, seq, dt", [(128, 40, torch.bfloat16), (64, 33, torch.float32), (64, 1, torch.float32)])
def test_short_rows_beside_long_ones(d, seq, dt):
    """In a call whose positions are split over several CTAs: rows that see one tile, rows of no slot and rows
    with a negative start."""
    rng = np.random.default_rng(d + seq)
    pool, host = _pool(rng, 4, 1, 2, 2700, d)
    qh = _bf16(rng.standard_normal((6, 16, seq, d)))
    _check(pool, host, 0, qh, [2, 0, 4, 1, 3, -1], [0, 2600, 7, 100, -3, 50], out_dtype=dt)
