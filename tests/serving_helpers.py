"""Torch / numpy stand-ins for the 4-bit cache, adapter and log-probability calls (any device), built on
``oracle.serving``: what the decoder and backend tests put in place of the CUDA calls."""

from __future__ import annotations

import numpy as np
import torch

from ccut_b200.logprobs import TokenLogprobs
from oracle import serving


def _np(t):
    return t.detach().float().cpu().numpy() if t.is_floating_point() else t.detach().cpu().numpy()


def kv4_append(pool, layer, k, v, slots, positions):
    for x, codes, par in ((k, pool.k, pool.k_par), (v, pool.v, pool.v_par)):
        c, p = serving.kv4_quantize(_np(x))
        for t, (s, pos) in enumerate(zip(_np(slots), _np(positions))):
            if 0 <= s < pool.slots and 0 <= pos < pool.max_len:
                codes[s, layer, :, pos] = torch.from_numpy(c[t]).to(codes.device)
                par[s, layer, :, pos] = torch.from_numpy(p[t]).to(par.device)


def kv4_attention(q, pool, layer, slots, starts, kv_len=None, scale=None, softcap=None, out_dtype=torch.bfloat16):
    n = pool.max_len if kv_len is None else kv_len
    out = np.zeros(tuple(q.shape))
    for b, (s, st) in enumerate(zip(_np(slots), _np(starts))):
        if 0 <= s < pool.slots and st >= 0:
            k = serving.kv4_values(_np(pool.k[s, layer]), pool.k_par[s, layer].cpu().numpy())[:, :n]
            v = serving.kv4_values(_np(pool.v[s, layer]), pool.v_par[s, layer].cpu().numpy())[:, :n]
            out[b] = serving.kv4_attention(_np(q[b]), k, v, int(st), scale, softcap)
    return torch.from_numpy(out).to(device=q.device, dtype=out_dtype)


def lora_add(bank, base, x, ids, out=None):
    y = serving.lora_add(_np(base), _np(x), _np(bank.a), _np(bank.b), _np(bank.scales), _np(ids), bank.widths)
    y = torch.from_numpy(y).to(device=base.device, dtype=base.dtype)
    if out is None:
        return y
    out.copy_(y)
    return out


def token_logprobs(logits, tokens, top_n=0):
    lp, ent, rank, ids, tlp = serving.token_logprobs(_np(logits), _np(tokens), top_n)
    f = [torch.from_numpy(np.asarray(a, np.float32)) for a in (lp, ent, tlp)]
    return TokenLogprobs(f[0], f[1], torch.from_numpy(rank), torch.from_numpy(ids), f[2])


def use_standins(monkeypatch):
    import ccut_b200.backend as backend
    import ccut_b200.model as m
    from ccut_b200.adapters import LoraBank

    monkeypatch.setattr(m, "kv4_append", kv4_append)
    monkeypatch.setattr(m, "kv4_attention", kv4_attention)
    monkeypatch.setattr(LoraBank, "add", lora_add)
    monkeypatch.setattr(backend, "token_logprobs", token_logprobs)


def banks(t, adapters: int, rank: int, seed: int, device, scale: float = 1.0) -> list:
    """Per layer of the tiny model ``t``: random adapters for its q / k / v and output projections."""
    from ccut_b200.adapters import LoraBank

    rng = np.random.default_rng(seed)
    q, kv = t.heads * t.head_dim, t.kv_heads * t.head_dim
    out = []
    for _ in range(t.layers):
        layer = {}
        for name, n_in, widths in (("qkv", t.hidden, [q, kv, kv]), ("o", q, [t.hidden])):
            mats = [([(rng.standard_normal((rank, n_in)) * n_in ** -0.5, rng.standard_normal((w, rank)) * rank ** -0.5)
                      for w in widths], scale) for _ in range(adapters)]
            layer[name] = LoraBank.from_matrices(mats, device=device)
        out.append(layer)
    return out
