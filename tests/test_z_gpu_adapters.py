"""Low-rank adapters on the GPU (``ccut_lora_add``, ``LoraBank``) against the oracle in 64 bits.

Tolerance: products of bf16 values are exact in fp32; a sum of n of them is off by at most n 2^-24
of the sum of their sizes, so h is off by inputs 2^-24 |x||A| and the output by that through |B|,
plus rank 2^-24 and the part of h that the second product drops (2^-24 with fp32 output, 2^-16 with
bf16) of |B||h|; adding the base rounds by half a step of the output type (2^-24 or 2^-8)."""

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


def _inputs(rng, tokens, inputs, rank, widths, adapters, dtype):
    x = _bf16(rng.standard_normal((tokens, inputs)))
    a = _bf16(rng.standard_normal((adapters, rank * len(widths), inputs)) * inputs ** -0.5)
    b = _bf16(rng.standard_normal((adapters, sum(widths), rank)))
    s = rng.uniform(0.25, 2, adapters).astype(np.float32)
    base = rng.standard_normal((tokens, sum(widths))).astype(np.float32)
    if dtype == torch.bfloat16:
        base = _bf16(base)
    return x, a, b, s, base


def _bank(a, b, s, widths):
    from ccut_b200.adapters import LoraBank

    return LoraBank(torch.from_numpy(a).cuda().bfloat16(), torch.from_numpy(b).cuda().bfloat16(),
                    torch.from_numpy(s).cuda(), widths)


def _tol(ref, x, a, b, s, ids, widths, dtype):
    r = b.shape[2]
    zero = np.zeros_like(ref)
    size = serving.lora_add(zero, np.abs(x), np.abs(a), np.abs(b), s, ids, widths)
    drop = 2.0 ** -16 if dtype == torch.bfloat16 else 2.0 ** -24
    half = 2.0 ** -8 if dtype == torch.bfloat16 else 2.0 ** -24
    return size * ((x.shape[1] + r + 8) * 2.0 ** -24 + drop) + half * np.abs(ref)


@pytest.mark.parametrize("tokens, inputs, rank, widths, adapters, dtype", [
    (1, 64, 16, [8], 1, torch.float32), (1, 2048, 16, [256, 64, 64], 5, torch.bfloat16),
    (5, 72, 32, [40], 3, torch.float32), (16, 256, 48, [264, 8, 80], 4, torch.bfloat16),
    (17, 1384, 64, [520, 264, 72], 9, torch.float32), (64, 512, 16, [512, 128, 128], 40, torch.float32),
    (130, 2048, 64, [1024], 2, torch.bfloat16), (257, 136, 256, [304], 3, torch.float32),
    (1000, 264, 16, [136, 136, 8, 24], 6, torch.bfloat16),
])
def test_matches_oracle(tokens, inputs, rank, widths, adapters, dtype):
    """Mixed adapters in every tile, runs of one, rows without one (ids below and above the bank's)."""
    rng = np.random.default_rng(tokens + inputs)
    x, a, b, s, base = _inputs(rng, tokens, inputs, rank, widths, adapters, dtype)
    bank = _bank(a, b, s, widths)
    for kind in ("mixed", "runs"):
        ids = rng.integers(-1, adapters + 1, tokens).astype(np.int32)
        if kind == "runs":
            ids = np.sort(ids)[::-1].copy()
        ids[rng.integers(0, tokens)] = adapters - 1
        ref = serving.lora_add(base, x, a, b, s, ids, widths)
        dev = torch.from_numpy(base).cuda().to(dtype)
        got = bank.add(dev, torch.from_numpy(x).cuda().bfloat16(), torch.from_numpy(ids).cuda())
        err = np.abs(got.float().cpu().numpy() - ref) - _tol(ref, x, a, b, s, ids, widths, dtype)
        assert not (err > 0).any(), (kind, err.max())
        none = (ids < 0) | (ids >= adapters)
        assert torch.equal(got[torch.from_numpy(none).cuda()], dev[torch.from_numpy(none).cuda()])
        again = dev.clone()
        bank.add(again, torch.from_numpy(x).cuda().bfloat16(), torch.from_numpy(ids).cuda(), out=again)
        assert torch.equal(again, got)


def test_rows_do_not_reach_each_other():
    """NaN and infinite weights of one adapter, and infinite inputs of one row, stay in their rows;
    a row's result does not depend on which rows are beside it."""
    rng = np.random.default_rng(1)
    widths = [64, 24]
    x, a, b, s, base = _inputs(rng, 40, 128, 32, widths, 4, torch.float32)
    ids = rng.integers(-1, 4, 40).astype(np.int32)
    ids[:4] = [0, 1, 2, 3]
    t = [torch.from_numpy(v).cuda() for v in (base, x, ids)]
    want = _bank(a, b, s, widths).add(t[0], t[1].bfloat16(), t[2])
    a2, b2, x2 = a.copy(), b.copy(), x.copy()
    a2[1, 3], b2[2, 5] = np.nan, np.inf
    x2[0] = np.inf
    got = _bank(a2, b2, s, widths).add(t[0], torch.from_numpy(x2).cuda().bfloat16(), t[2])
    same = torch.from_numpy(~np.isin(ids, [1, 2])).cuda()
    same[0] = False
    assert torch.equal(got[same], want[same])
    assert torch.isnan(got[1, :64]).all()  # rank row 3 is part 0's
    for r in (0, 3, 21):
        alone = _bank(a, b, s, widths).add(t[0][r: r + 1].clone(), t[1][r: r + 1].bfloat16(), t[2][r: r + 1].clone())
        np.testing.assert_allclose(alone[0].cpu().numpy(), want[r].cpu().numpy(), rtol=1e-5, atol=1e-5)


def test_strided_bases_and_no_tokens():
    """A column block of a wider buffer is read and written in place, the columns beside it kept."""
    rng = np.random.default_rng(2)
    x, a, b, s, base = _inputs(rng, 33, 256, 16, [64], 2, torch.bfloat16)
    bank = _bank(a, b, s, [64])
    ids = torch.from_numpy((np.arange(33) % 3 - 1).astype(np.int32)).cuda()
    xd, dev = torch.from_numpy(x).cuda().bfloat16(), torch.from_numpy(base).cuda().bfloat16()
    want = bank.add(dev, xd, ids)
    wide = torch.full((33, 136), 7.0, device="cuda", dtype=torch.bfloat16)
    wide[:, 8:72] = dev
    view = wide[:, 8:72]
    assert bank.add(view, xd, ids, out=view) is view
    assert torch.equal(view, want) and bool((wide[:, :8] == 7).all()) and bool((wide[:, 72:] == 7).all())
    assert torch.equal(bank.add(wide[:, 8:72].t().contiguous().t(), xd, ids),
                       bank.add(want, xd, ids))  # any base strides
    assert bank.add(dev[:0], xd[:0], ids[:0]).shape == (0, 64)


def test_bank_from_checkpoint_matrices():
    """Ranks of 8 and 24 padded to 32, a part that one adapter lacks, alpha / r scales."""
    from ccut_b200.adapters import LoraBank

    rng = np.random.default_rng(4)
    inputs, widths = 256, [48, 16]
    mats = []
    for r in (8, 24):
        mats.append([(_bf16(rng.standard_normal((r, inputs)) / 16), _bf16(rng.standard_normal((w, r)))) for w in widths])
    mats[1][1] = None
    bank = LoraBank.from_matrices([(mats[0], 2.0), (mats[1], 0.5)])
    assert bank.rank == 32 and bank.widths == widths
    x, base = _bf16(rng.standard_normal((3, inputs))), rng.standard_normal((3, 64)).astype(np.float32)
    got = bank.add(torch.from_numpy(base).cuda(), torch.from_numpy(x).cuda().bfloat16(),
                   torch.tensor([1, -1, 0], dtype=torch.int32, device="cuda")).cpu().numpy()
    ref = base.astype(np.float64)
    for t, (i, scale) in ((0, (1, 0.5)), (2, (0, 2.0))):
        for j, at in ((0, 0), (1, 48)):
            if mats[i][j] is not None:
                A, B = (m.astype(np.float64) for m in mats[i][j])
                ref[t, at: at + widths[j]] += scale * (B @ (A @ x[t]))
    np.testing.assert_allclose(got, ref, rtol=1e-5, atol=1e-4)


@pytest.mark.parametrize("tokens, inputs, rank, widths, adapters, dtype", [
    (300, 200, 64, [264, 72], 3, torch.float32), (513, 128, 32, [136, 40, 88], 4, torch.bfloat16),
    (700, 512, 64, [520], 2, torch.bfloat16), (259, 64, 96, [200, 8], 2, torch.float32),
    (321, 1032, 32, [8, 24, 16, 200], 1, torch.float32), (400, 256, 64, [24, 104, 8, 248], 5, torch.bfloat16),
])
def test_prompts_match_oracle(tokens, inputs, rank, widths, adapters, dtype):
    """More tokens than a decode step: every rank class, blocks of outputs that hold several parts."""
    rng = np.random.default_rng(tokens + rank)
    x, a, b, s, base = _inputs(rng, tokens, inputs, rank, widths, adapters, dtype)
    bank = _bank(a, b, s, widths)
    xd, bd = torch.from_numpy(x).cuda().bfloat16(), torch.from_numpy(base).cuda().to(dtype)
    for ids in (rng.integers(-1, adapters, tokens), np.sort(rng.integers(0, adapters, tokens)), np.full(tokens, -1)):
        ids = ids.astype(np.int32)
        ref = serving.lora_add(base, x, a, b, s, ids, widths)
        got = bank.add(bd, xd, torch.from_numpy(ids).cuda()).float().cpu().numpy()
        assert (np.abs(got - ref) <= _tol(ref, x, a, b, s, ids, widths, dtype)).all()


def test_misaligned_inputs():
    """Contiguous tensors that begin off a 16-byte boundary are taken all the same."""
    rng = np.random.default_rng(8)
    x, a, b, s, base = _inputs(rng, 5, 64, 16, [24], 2, torch.bfloat16)
    bank, ids = _bank(a, b, s, [24]), torch.tensor([0, 1, -1, 1, 0], dtype=torch.int32, device="cuda")
    xd, bd = torch.from_numpy(x).cuda().bfloat16(), torch.from_numpy(base).cuda().bfloat16()

    def shifted(t):
        flat = torch.zeros(t.numel() + 8, dtype=t.dtype, device="cuda")
        flat[1: 1 + t.numel()] = t.reshape(-1)
        return flat[1: 1 + t.numel()].view(t.shape)

    assert torch.equal(bank.add(shifted(bd), shifted(xd), shifted(ids)), bank.add(bd, xd, ids))
    with pytest.raises(ValueError):
        bank.add(bd, xd, ids, out=shifted(bd))


@pytest.mark.parametrize("tokens", [37, 300])
def test_captured_calls_and_two_streams(tokens):
    """A captured call replayed after its inputs changed gives the eager answer, the same bits twice; calls on
    two streams at once do not disturb each other."""
    rng = np.random.default_rng(tokens + 9)
    x, a, b, s, base = _inputs(rng, tokens, 520, 32, [72, 16], 5, torch.bfloat16)
    bank = _bank(a, b, s, [72, 16])
    xd, bd = torch.from_numpy(x).cuda().bfloat16(), torch.from_numpy(base).cuda().bfloat16()
    ids = [torch.from_numpy(rng.integers(-1, 5, tokens).astype(np.int32)).cuda() for _ in range(3)]
    want = [bank.add(bd, xd, i) for i in ids]
    held = ids[0].clone()
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        bank.add(bd, xd, held)
    torch.cuda.current_stream().wait_stream(stream)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = bank.add(bd, xd, held)
    for i, w in zip(ids + ids, want + want):
        held.copy_(i)
        graph.replay()
        assert torch.equal(out, w)
    streams = [torch.cuda.Stream() for _ in ids]
    for st in streams:
        st.wait_stream(torch.cuda.current_stream())
    got = [[] for _ in ids]
    for _ in range(4):
        for st, i, g in zip(streams, ids, got):
            with torch.cuda.stream(st):
                g.append(bank.add(bd, xd, i))
    torch.cuda.synchronize()
    for g, w in zip(got, want):
        assert all(torch.equal(y, w) for y in g)
