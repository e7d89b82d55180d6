"""4-bit attention where one position takes nearly all of the probability and what is left decides the output:
a sink, whose values are zeros.

Tolerance per output, with p_j = e^(x_j - max x) and l their sum.  A score is off by at most ds = e sum |q||k| scale,
e = 2^-16 for a short query block and 2^-11 (keys as fp16) for a long one, which changes p_j / l by a factor
within e^(+-2 ds).  Probabilities enter the second product as fp16, at most half a step off: 2^-11 of p_j, or half of
the least step 2^-24 where p_j is so small.  The kernels scale them by a power of two so that the largest
is in [2^10, 2^15]: the least step then costs 2^-35 of a probability of 1.  In a short block it is p_j s_j that is
rounded, scaled by the largest s of the row's positions, and multiplies codes of at most 15 (fp32 output keeps a
second part, 2^-20); a long one rounds the values to fp16 as well.  fp32 sums cost less than 2^-16 of the sum of
absolute terms, the output's type 2^-8 (bf16) of the value."""

from __future__ import annotations

import numpy as np
import pytest
import torch

from oracle import serving
from tests.test_z_gpu_kv4 import _bf16, _cuda, _dev  # noqa: F401

pytestmark = pytest.mark.gpu

LONG = 129  # query rows per kv head from which a call runs as a long block


def _sink_case(rng, d, L, at, nats, grp, seq):
    """q [grp, seq, d]; k, v codes and params [1, 1, 1, L, ..] with the sink at `at`, whose score is about nats[h]
    above the others' for head h."""
    u = rng.choice([-1.0, 1.0], d).astype(np.float32)
    k = 0.3 * rng.standard_normal((L, d)).astype(np.float32)
    k[at] = 2 * u
    v = 1 + 0.5 * rng.standard_normal((L, d)).astype(np.float32)
    v[at] = 0
    q = np.asarray(nats, np.float32)[:, None, None] * u / (2 * d ** 0.5) + 0.2 * rng.standard_normal((grp, seq, d))
    return _bf16(q), serving.kv4_quantize(k[None, None, None]), serving.kv4_quantize(v[None, None, None])


def _reference(q, k, v, sv, lim, seq_rows, out_bf16):
    """One row: (output, tolerance) from its query q [d], values k, v [n, d], value scales sv [n, d / 64]."""
    d = q.shape[0]
    long_block = seq_rows >= LONG
    k, v, sv = k[: lim + 1], v[: lim + 1], sv[: lim + 1]
    x = k @ q * d ** -0.5
    p = np.exp(x - x.max())
    l = p.sum()
    ref = p @ v / l
    ds = (2.0 ** -11 if long_block else 2.0 ** -16) * (np.abs(k) @ np.abs(q)).max() * d ** -0.5
    up, least = (2.0 ** -20 if not (out_bf16 or long_block) else 2.0 ** -11), 2.0 ** -35
    tol = p @ np.abs(v) / l * (np.expm1(2 * ds) + up + 2.0 ** -16)
    if long_block:
        tol += (p @ np.abs(v) * 2.0 ** -11 + least * np.abs(v).sum(0)) / l
    else:
        s = np.repeat(sv, 64, 1)
        tol += 15 * (up * (p @ s) + least * len(p) * sv.max() + 2.0 ** -16 * (p @ s)) / l
    return ref, tol + (2.0 ** -8 * np.abs(ref) if out_bf16 else 0)


@pytest.mark.parametrize("dt", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("d, grp, seq, L, kv_len", [
    (128, 8, 1, 8192, 8192), (64, 8, 1, 3001, 3001), (128, 8, 1, 700, 700), (64, 16, 1, 1000, 1000), (128, 16, 2, 4100, 4100),
    (64, 12, 5, 2100, 2100), (128, 8, 40, 2600, 2600), (64, 8, 40, 2600, 2600), (128, 8, 40, 400, 400), (64, 8, 70, 450, 450),
])
def test_what_a_sink_leaves(d, grp, seq, L, kv_len, dt):
    """Sinks 8 to 18 nats above thousands of positions, one scale of probabilities a head, at the begin, inside and
    near the end of the cache: short blocks whole and cut, long blocks whole and split."""
    from ccut_b200.blocks.attn_kv4 import Kv4Pool, kv4_attention

    rng = np.random.default_rng(d + grp + seq)
    nats = np.linspace(8, 18, grp)
    for at in (0, L // 2 + 3, L - seq - 2):
        q, k, v = _sink_case(rng, d, L, at, nats, grp, seq)
        pool = Kv4Pool.wrap(*(_dev(a) for pair in (k, v) for a in pair))
        i32 = [torch.tensor([n], dtype=torch.int32, device="cuda") for n in (0, L - seq)]
        got = kv4_attention(_dev(q[None], torch.bfloat16), pool, 0, *i32, kv_len=kv_len, out_dtype=dt)[0].float().cpu().numpy()
        kv, vv = (serving.kv4_values(*p)[0, 0, 0] for p in (k, v))
        sv = v[1][0, 0, 0, :, :, 0].astype(np.float64)
        for h in range(grp):
            for i in range(0, seq, 13):
                ref, tol = _reference(q[h, i].astype(np.float64), kv, vv, sv, L - seq + i, grp * seq, dt == torch.bfloat16)
                off = np.abs(got[h, i] - ref)
                assert (off <= tol).all(), (at, h, i, (off / tol).max(), np.linalg.norm(off) / np.linalg.norm(ref))
