"""CPU restatement (numpy) of the 4-bit kv cache, token log probabilities and low-rank adapters.

Test infrastructure only.  These operators have no counterpart in the reference; the functions
here state their definitions (the cache format in the fp32 steps that fix it, everything else
in 64 bits) apart from the CUDA code.
"""

from __future__ import annotations

import numpy as np

__all__ = ["kv4_attention", "kv4_quantize", "kv4_values", "lora_add", "token_logprobs"]

GROUP = 64


def kv4_quantize(x: np.ndarray) -> tuple:
    """fp32 ``[..., d]`` -> codes uint8 ``[..., d / 2]`` and (scale, minimum) fp16 ``[..., d / 64, 2]``."""
    x = np.asarray(x, np.float32)
    g = x.reshape(x.shape[:-1] + (-1, GROUP))
    bad = ~np.isfinite(g).all(-1)
    c = np.clip(np.where(np.isfinite(g), g, 0), -65504, 65504).astype(np.float32)
    m = c.min(-1).astype(np.float16)
    s = np.maximum((c.max(-1) - m.astype(np.float32)) * np.float32(1.0 / 15.0), 0).astype(np.float16)
    sf, mf = s.astype(np.float32)[..., None], m.astype(np.float32)[..., None]
    with np.errstate(divide="ignore", invalid="ignore", over="ignore"):
        q = np.where((sf > 0) & ~bad[..., None], np.clip(np.rint((np.where(np.isfinite(g), g, 0) - mf) / sf), 0, 15), 0)
    q = q.astype(np.uint8).reshape(x.shape)
    par = np.stack([s, m], -1)
    par[bad] = np.float16(np.nan)
    return q[..., 0::2] | (q[..., 1::2] << 4), par


def kv4_values(codes: np.ndarray, par: np.ndarray) -> np.ndarray:
    """The values that codes and params stand for, in 64 bits."""
    q = np.stack([codes & 15, codes >> 4], -1).reshape(codes.shape[:-1] + (-1, GROUP)).astype(np.float64)
    p = par.astype(np.float64)
    return (q * p[..., 0:1] + p[..., 1:2]).reshape(codes.shape[:-1] + (codes.shape[-1] * 2,))


def kv4_attention(q, k, v, start: int, scale: float | None = None, softcap: float | None = None) -> np.ndarray:
    """One sequence: q ``[heads, seq, d]``, k / v values ``[kv_heads, n, d]``; query i sees positions
    ``<= start + i``.  64 bits; a query that sees nothing gives zeros."""
    q, k, v = (np.asarray(a, np.float64) for a in (q, k, v))
    h, s, d = q.shape
    out = np.zeros((h, s, d))
    for j in range(h):
        kk, vv = k[j * k.shape[0] // h], v[j * k.shape[0] // h]
        for i in range(s):
            n = min(k.shape[1], start + i + 1)
            if n <= 0:
                continue
            x = kk[:n] @ q[j, i] * (scale or d ** -0.5)
            if softcap:
                x = np.tanh(x / softcap) * softcap
            p = np.exp(x - x.max())
            out[j, i] = p @ vv[:n] / p.sum()
    return out


def token_logprobs(x, tokens, top_n: int) -> tuple:
    """(logprob, entropy, rank, top_ids, top_logprobs) of rows x (finite or -inf logits), 64 bits."""
    x = np.asarray(x, np.float64)
    rows, vocab = x.shape
    m = x.max(1, keepdims=True)
    lp = x - m - np.log(np.exp(x - m).sum(1, keepdims=True))
    p = np.exp(lp)
    ent = -np.where(p > 0, p * np.where(p > 0, lp, 0), 0).sum(1)
    order = np.argsort(-x, axis=1, kind="stable")
    got = np.full(rows, np.nan)
    rank = np.zeros(rows, np.int32)
    for r, t in enumerate(tokens):
        if 0 <= t < vocab:
            got[r] = lp[r, t]
            rank[r] = 1 + int(np.nonzero(order[r] == t)[0][0])
    ids = order[:, :top_n].astype(np.int32)
    return got, ent, rank, ids, np.take_along_axis(lp, ids, 1)


def lora_add(base, x, a, b, scales, ids, widths) -> np.ndarray:
    """base + scale B A x per token, 64 bits (shapes as ``ccut_lora_add``)."""
    y = np.asarray(base, np.float64).copy()
    r = b.shape[2]
    for t, i in enumerate(ids):
        if not 0 <= i < a.shape[0]:
            continue
        h = a[i].astype(np.float64) @ x[t].astype(np.float64)
        at = 0
        for j, w in enumerate(widths):
            y[t, at: at + w] += float(scales[i]) * (b[i, at: at + w].astype(np.float64) @ h[j * r: (j + 1) * r])
            at += w
    return y
