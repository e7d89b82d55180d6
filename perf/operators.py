"""The serving operators of this package as measured calls, each beside a plain form of the same
mathematics in elementary torch operations.

Operators (``kind`` of a case):

``append``    k / v rows of new tokens quantized to 4 bits (groups of 64 features, fp16 scale and
              minimum) into a cache pool, and the rows read back as the values they stand for
``attend``    grouped-query attention over such a cache: decode steps and prompt chunks
``logprobs``  log probability, entropy and rank of given tokens and the top alternatives
``lora``      low-rank adapters of many requests added beside a shared projection

``own`` selects the package's calls; otherwise ``run`` computes the plain forms.
"""

from __future__ import annotations

import math

import numpy as np
import torch

own = False

GROUP = 64  # features that share one (scale, minimum) pair of the 4-bit cache


# ---- cases ---------------------------------------------------------------------------------------
def listed():
    return [
        # one decode step of 64 requests: every request's new k / v row of one layer
        {"name": "append step of 64", "kind": "append", "tokens": 64, "kv_heads": 4, "head_dim": 128, "slots": 64,
         "max_len": 640, "dtype": "bf16"},
        # a long prompt chunk, fp32 rows as the rotary embedding gives them
        {"name": "append prompt 8190", "kind": "append", "tokens": 8190, "kv_heads": 4, "head_dim": 128, "slots": 2,
         "max_len": 8192, "dtype": "fp32"},
        # a single request shortly after a short prompt: latency
        {"name": "decode 1 x 513", "kind": "attend", "batch": 1, "heads": 32, "kv_heads": 4, "head_dim": 128, "seq": 1,
         "len_min": 513, "len_max": 513, "max_len": 1024},
        # eight requests of the engine's decode workload (prompts of 512 and what followed)
        {"name": "decode 8 x 600", "kind": "attend", "batch": 8, "heads": 32, "kv_heads": 4, "head_dim": 128, "seq": 1,
         "len_min": 512, "len_max": 690, "max_len": 1024},
        # a full batch of long, uneven requests: the cache exceeds the L2
        {"name": "decode 64 ragged 8k", "kind": "attend", "batch": 64, "heads": 32, "kv_heads": 4, "head_dim": 128,
         "seq": 1, "len_min": 3001, "len_max": 8191, "max_len": 8192},
        # one very long request: the long axis is all there is to split
        {"name": "decode 1 x 131071", "kind": "attend", "batch": 1, "heads": 16, "kv_heads": 2, "head_dim": 64,
         "seq": 1, "len_min": 131071, "len_max": 131071, "max_len": 131072},
        # the prefill chunk of the engine workload's shape: 4096 tokens from position 0
        {"name": "prefill 4096", "kind": "attend", "batch": 1, "heads": 32, "kv_heads": 4, "head_dim": 128,
         "seq": 4096, "len_min": 4096, "len_max": 4096, "max_len": 8192},
        # odd chunks of two requests deep in their prompts, head dim 64
        {"name": "chunk 2 x 509 at 6k", "kind": "attend", "batch": 2, "heads": 16, "kv_heads": 4, "head_dim": 64,
         "seq": 509, "len_min": 5501, "len_max": 6997, "max_len": 7168},
        # log probabilities of one decode step's tokens with five alternatives
        {"name": "logprobs 8 x 151936", "kind": "logprobs", "rows": 8, "vocab": 151936, "top": 5, "dtype": "fp32"},
        # a scored prompt
        {"name": "logprobs 2047 x 102400", "kind": "logprobs", "rows": 2047, "vocab": 102400, "top": 20,
         "dtype": "fp32"},
        # q / k / v projection of a decode batch in which 16 adapters (and some requests without one) mix
        {"name": "lora qkv step of 64", "kind": "lora", "tokens": 64, "adapters": 16, "rank": 16, "inputs": 2048,
         "widths": "4096,512,512", "requests": 64, "dtype": "fp32"},
        # output projection of three prompts' tokens
        {"name": "lora o prompt 4093", "kind": "lora", "tokens": 4093, "adapters": 8, "rank": 64, "inputs": 4096,
         "widths": "2048", "requests": 3, "dtype": "bf16"},
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    kind = rng.choice(["append", "attend", "attend", "logprobs", "lora"])
    if kind == "append":
        tokens = _log_int(rng, 1, 8190)
        slots = rng.randint(1, 16)
        return {"kind": kind, "tokens": tokens, "kv_heads": rng.choice([1, 2, 3, 4, 8]) if tokens < 4000 else 4,
                "head_dim": rng.choice([64, 128]), "slots": slots, "max_len": -(-tokens // slots) + rng.randint(0, 500),
                "dtype": rng.choice(["bf16", "fp32"])}
    if kind == "attend":
        kv_heads = rng.choice([1, 2, 4, 8])
        heads = kv_heads * rng.choice([1, 2, 4, 7, 8, 16])
        d = rng.choice([64, 128])
        if rng.random() < 0.6:
            batch = _log_int(rng, 1, 64)
            most = max(64, min(131072, 64 * 8192 * 4 // (2 * batch * kv_heads)))
            hi = _log_int(rng, 1, most)
            seq = rng.choice([1, 1, 1, 2, 3]) if hi > 8 else 1
        else:
            batch = rng.choice([1, 1, 2, 3])
            seq = _log_int(rng, 4, 2048)
            hi = seq + rng.choice([0, rng.randint(1, 4096)])
            heads = min(heads, kv_heads * 8, 32)
            heads -= heads % kv_heads
        lo = max(seq, hi - rng.randint(0, hi // 2))
        return {"kind": kind, "batch": batch, "heads": heads, "kv_heads": kv_heads, "head_dim": d, "seq": seq,
                "len_min": lo, "len_max": max(lo, hi), "max_len": max(lo, hi) + rng.randint(0, 300)}
    if kind == "logprobs":
        vocab = _log_int(rng, 1000, 151936)
        rows = _log_int(rng, 1, max(1, min(4096, 2047 * 102400 // vocab)))
        return {"kind": kind, "rows": rows, "vocab": vocab, "top": rng.choice([0, 1, 5, 20]),
                "dtype": rng.choice(["fp32", "fp32", "bf16"])}
    tokens = _log_int(rng, 1, 4093)
    widths = rng.choice(["4096,512,512", "2048", "1536", "1024,1024", "520,264,72"])
    return {"kind": "lora", "tokens": tokens, "adapters": rng.randint(1, 32), "rank": rng.choice([16, 32, 64]),
            "inputs": rng.choice([512, 2048, 4096, 1384]), "widths": widths,
            "requests": min(tokens, _log_int(rng, 1, 64)), "dtype": rng.choice(["fp32", "bf16"])}


# ---- what a case holds, from its numbers alone -----------------------------------------------------
def _lens(c):
    """Cached positions of every batch row, this call's tokens included: evenly spread, shuffled."""
    b = c["batch"]
    lens = np.linspace(c["len_min"], c["len_max"], b).round().astype(np.int64)
    return lens[np.random.RandomState(b).permutation(b)]


def _ids(c):
    """Adapter of every token: each request has one (or none: -1), its tokens are adjacent."""
    r = np.random.RandomState(c["tokens"] + 7 * c["adapters"])
    per = r.randint(-1, c["adapters"], c["requests"]) if c["requests"] > 3 else np.arange(c["requests"]) % c["adapters"]
    cut = np.sort(r.permutation(c["tokens"] - 1)[: c["requests"] - 1] + 1) if c["tokens"] > 1 else np.zeros(0, np.int64)
    return per[np.searchsorted(cut, np.arange(c["tokens"]), side="right")].astype(np.int32)


def _widths(c):
    return [int(w) for w in c["widths"].split(",")]


def work(case):
    c = case
    if c["kind"] == "append":
        n = c["tokens"] * c["kv_heads"] * c["head_dim"] * 2
        return {"bytes": n * (4 if c["dtype"] == "fp32" else 2) + n * 36 / 64 + 4 * n, "flops": 8 * n}
    if c["kind"] == "attend":
        lens = _lens(c)
        rows = c["heads"] * c["head_dim"] * c["seq"] * c["batch"] * 2
        cache = float(lens.sum()) * c["kv_heads"] * c["head_dim"] * 2 * 36 / 64
        seen = float(sum(c["seq"] * (n - c["seq"]) + c["seq"] * (c["seq"] + 1) / 2 for n in lens.tolist()))
        return {"bytes": cache + 2 * rows, "flops": 4 * seen * c["heads"] * c["head_dim"]}
    if c["kind"] == "logprobs":
        n = c["rows"] * c["vocab"]
        return {"bytes": n * (4 if c["dtype"] == "fp32" else 2) + c["rows"] * (16 + 8 * c["top"]), "flops": 6 * n}
    ids, w = _ids(c), _widths(c)
    e = 4 if c["dtype"] == "fp32" else 2
    used = len(set(ids[ids >= 0].tolist()))
    weights = used * c["rank"] * (len(w) * c["inputs"] + sum(w)) * 2
    some = int((ids >= 0).sum())
    return {"bytes": weights + some * c["inputs"] * 2 + c["tokens"] * sum(w) * 2 * e,
            "flops": 2 * some * c["rank"] * (len(w) * c["inputs"] + sum(w))}


# ---- inputs ------------------------------------------------------------------------------------------
def _quantized(x):
    """fp32 rows [..., d] -> (codes uint8 [..., d / 2], scale and minimum fp16 [..., d / 64, 2])."""
    g = x.unflatten(-1, (x.shape[-1] // GROUP, GROUP))
    lo, hi = g.amin(-1).clamp(-65504.0, 65504.0), g.amax(-1).clamp(-65504.0, 65504.0)
    m = lo.half()
    s = ((hi - m.float()) * (1.0 / 15.0)).clamp(min=0.0).half()
    sf = s.float().unsqueeze(-1)
    q = ((g - m.float().unsqueeze(-1)) / torch.where(sf > 0, sf, torch.ones_like(sf))).round().clamp(0, 15)
    q = torch.where(sf > 0, q, torch.zeros_like(q)).to(torch.uint8).flatten(-2)
    return q[..., 0::2] | (q[..., 1::2] << 4), torch.stack([s, m], -1)


def _values(codes, par):
    """The fp32 values that codes [..., d / 2] and (scale, minimum) pairs [..., d / 64, 2] stand for."""
    q = torch.stack([codes & 15, codes >> 4], -1).flatten(-2).float()
    q = q.unflatten(-1, (q.shape[-1] // GROUP, GROUP))
    return (q * par[..., 0:1].float() + par[..., 1:2].float()).flatten(-2)


def prepare(case, seed):
    c = case
    dev = torch.device("cuda")
    g = torch.Generator(device=dev)
    g.manual_seed(seed)

    def normal(*shape):
        return torch.randn(shape, generator=g, device=dev)

    st = {"case": c}
    if c["kind"] == "append":
        n, h, d = c["tokens"], c["kv_heads"], c["head_dim"]
        dt = torch.float32 if c["dtype"] == "fp32" else torch.bfloat16
        bias = normal(1, h, d)  # channels of k have means of their own
        st["k"], st["v"] = (normal(n, h, d) + 2 * bias).to(dt), (normal(n, h, d) * 0.5).to(dt)
        each = -(-n // c["slots"])
        at = torch.arange(n, device=dev)
        st["slots"] = (at // each).to(torch.int32)
        st["positions"] = (at % each + (c["max_len"] - each)).to(torch.int32)
        rows = (c["slots"], 1, h, c["max_len"])
        for name in ("k", "v"):
            st["codes_" + name] = torch.zeros(rows + (d // 2,), dtype=torch.uint8, device=dev)
            st["par_" + name] = torch.zeros(rows + (d // GROUP, 2), dtype=torch.float16, device=dev)
        return st
    if c["kind"] == "attend":
        b, h, d, n = c["batch"], c["kv_heads"], c["head_dim"], c["max_len"]
        lens = torch.from_numpy(_lens(c)).to(dev)
        st["slots"] = torch.from_numpy(np.random.RandomState(b + 1).permutation(b).astype(np.int32)).to(dev)
        st["starts"] = (lens - c["seq"]).to(torch.int32)
        st["q"] = normal(b, c["heads"], c["seq"], d).to(torch.bfloat16)
        for name in ("k", "v"):
            mean = normal(1, 1, h, 1, d)
            codes = torch.empty((b, 1, h, n, d // 2), dtype=torch.uint8, device=dev)
            par = torch.empty((b, 1, h, n, d // GROUP, 2), dtype=torch.float16, device=dev)
            step = max(1, (1 << 25) // (h * n * d))
            for at in range(0, b, step):
                x = normal(min(step, b - at), 1, h, n, d)
                x = (x + mean) if name == "k" else x * 0.5
                codes[at: at + step], par[at: at + step] = _quantized(x)
            st["codes_" + name], st["par_" + name] = codes, par
        return st
    if c["kind"] == "logprobs":
        dt = torch.float32 if c["dtype"] == "fp32" else torch.bfloat16
        sharp = 1.0 + 2.0 * torch.rand((c["rows"], 1), generator=g, device=dev)
        x = normal(c["rows"], c["vocab"]) * sharp
        st["logits"] = x.to(dt)
        near = torch.argmax(x[:, : c["vocab"] // 2], dim=1)  # a likely token in every second row
        any_ = torch.randint(0, c["vocab"], (c["rows"],), generator=g, device=dev)
        even = torch.arange(c["rows"], device=dev) % 2 == 0
        st["tokens"] = torch.where(even, near, any_).to(torch.int32)
        return st
    w, n, r = _widths(c), c["adapters"], c["rank"]
    dt = torch.float32 if c["dtype"] == "fp32" else torch.bfloat16
    st["x"] = normal(c["tokens"], c["inputs"]).to(torch.bfloat16)
    st["a"] = (normal(n, len(w) * r, c["inputs"]) * c["inputs"] ** -0.5).to(torch.bfloat16)
    st["b"] = (normal(n, sum(w), r) * r ** -0.5).to(torch.bfloat16)
    st["scales"] = 0.5 + torch.rand((n,), generator=g, device=dev)
    st["ids"] = torch.from_numpy(_ids(c)).to(dev)
    st["base"] = normal(c["tokens"], sum(w)).to(dt)
    return st


# ---- the operators -----------------------------------------------------------------------------------
def run(state):
    return {"append": _append, "attend": _attend, "logprobs": _logprobs, "lora": _lora}[state["case"]["kind"]](state)


def _append(st):
    if own:
        from ccut_b200.blocks.attn_kv4 import Kv4Pool, kv4_append, kv4_read

        pool = Kv4Pool.wrap(st["codes_k"], st["par_k"], st["codes_v"], st["par_v"])
        kv4_append(pool, 0, st["k"], st["v"], st["slots"], st["positions"])
        return kv4_read(pool, 0, st["slots"], st["positions"])
    slots, pos = st["slots"].long(), st["positions"].long()
    out = []
    out += [_plain_append(st["k"], st["codes_k"], st["par_k"], slots, pos)]
    out += [_plain_append(st["v"], st["codes_v"], st["par_v"], slots, pos)]
    return tuple(out)


def _plain_append(x, codes, par, slots, pos):
    q, p = _quantized(x.float())
    codes[slots, 0, :, pos], par[slots, 0, :, pos] = q, p
    return _values(codes[slots, 0, :, pos], par[slots, 0, :, pos])


def _attend(st):
    c = st["case"]
    if own:
        from ccut_b200.blocks.attn_kv4 import Kv4Pool, kv4_attention

        pool = Kv4Pool.wrap(st["codes_k"], st["par_k"], st["codes_v"], st["par_v"])
        return kv4_attention(st["q"], pool, 0, st["slots"], st["starts"], kv_len=c["len_max"])
    n, s = c["len_max"], c["seq"]
    slots = st["slots"].long()
    k = _values(st["codes_k"][slots, 0, :, :n], st["par_k"][slots, 0, :, :n])
    v = _values(st["codes_v"][slots, 0, :, :n], st["par_v"][slots, 0, :, :n])
    q = st["q"].float().unflatten(1, (c["kv_heads"], c["heads"] // c["kv_heads"])).flatten(2, 3)
    x = (q @ k.transpose(2, 3)) * c["head_dim"] ** -0.5  # [batch, kv_heads, group * seq, n]
    x = x.unflatten(2, (c["heads"] // c["kv_heads"], s))
    last = st["starts"].long()[:, None] + torch.arange(s, device=q.device)
    hide = torch.arange(n, device=q.device) > last[:, None, None, :, None]
    x = x.masked_fill_(hide, -math.inf)
    x = x - x.amax(-1, keepdim=True)
    p = torch.exp_(x)
    p = p / p.sum(-1, keepdim=True)
    o = p.flatten(2, 3) @ v
    return o.unflatten(2, (c["heads"] // c["kv_heads"], s)).flatten(1, 2).to(torch.bfloat16)


def _logprobs(st):
    c = st["case"]
    if own:
        from ccut_b200.logprobs import token_logprobs

        r = token_logprobs(st["logits"], st["tokens"], top_n=c["top"])
        return {"logprob": r.logprob, "entropy": r.entropy, "rank": r.rank, "top_ids": r.top_ids,
                "top_logprobs": r.top_logprobs}
    x = st["logits"].float()
    tok = st["tokens"].long()[:, None]
    at = torch.arange(c["vocab"], device=x.device)
    mine = x.gather(1, tok)
    rank = 1 + (x > mine).sum(1) + ((x == mine) & (at < tok)).sum(1)
    m = x.amax(1, keepdim=True)
    e = torch.exp(x - m)
    z = e.sum(1, keepdim=True, dtype=torch.float64)
    logz = torch.log(z)
    mean = (e * (x - m)).sum(1, keepdim=True, dtype=torch.float64) / z
    bits = (x + 0.0).view(torch.int32)
    key = torch.where(bits < 0, bits ^ 0x7FFFFFFF, bits).long() * (1 << 32) + (c["vocab"] - 1 - at)
    top = torch.topk(key, c["top"], dim=1).values
    ids = c["vocab"] - 1 - (top & 0xFFFFFFFF)
    return {"logprob": ((mine - m).double() - logz)[:, 0].float(), "entropy": (logz - mean)[:, 0].float(),
            "rank": rank.to(torch.int32), "top_ids": ids.to(torch.int32),
            "top_logprobs": ((x.gather(1, ids) - m).double() - logz).float()}


def _lora(st):
    c, w = st["case"], _widths(st["case"])
    if own:
        from ccut_b200.adapters import LoraBank

        return LoraBank(st["a"], st["b"], st["scales"], w).add(st["base"], st["x"], st["ids"])
    n, r, t = c["adapters"], c["rank"], c["tokens"]
    mine = (st["ids"][:, None] == torch.arange(n, device=st["ids"].device)).float() * st["scales"]
    h = (st["x"].float() @ st["a"].float().flatten(0, 1).t()).view(t, n, len(w), r) * mine[:, :, None, None]
    b = st["b"].float().split(w, dim=1)
    parts = [h[:, :, j].reshape(t, n * r) @ b[j].transpose(0, 1).reshape(w[j], n * r).t() for j in range(len(w))]
    return (st["base"].float() + torch.cat(parts, 1)).to(st["base"].dtype)


# ---- the same from the definitions, in 64 bits --------------------------------------------------------
def exact(case, seed):
    st, c = prepare(case, seed), case
    if c["kind"] == "append":
        return tuple(_exact_rows(st[name].float().cpu().numpy()) for name in ("k", "v"))
    if c["kind"] == "attend":
        return _exact_attend(st, c)
    if c["kind"] == "logprobs":
        return _exact_logprobs(st, c)
    x, a, b = st["x"].double(), st["a"].double(), st["b"].double()
    y = st["base"].double()
    r = c["rank"]
    for i in range(c["adapters"]):
        rows = torch.nonzero(st["ids"] == i)[:, 0]
        if rows.numel() == 0:
            continue
        h = x[rows] @ a[i].t()
        at = 0
        for j, w in enumerate(_widths(c)):
            y[rows, at: at + w] += float(st["scales"][i]) * (h[:, j * r: (j + 1) * r] @ b[i, at: at + w].t())
            at += w
    return y


def _exact_rows(x):
    """The stored values of rows x: the format fixes its scale and code as fp32 expressions (fp16
    minimum m, fp16 scale fl((max - m) * fl(1/15)), code fl((x - m) / s) to the nearest, ties to even);
    the value they stand for is code * s + m."""
    g = x.reshape(x.shape[:-1] + (-1, GROUP))
    m = g.min(-1).astype(np.float16)
    s = np.maximum((g.max(-1) - m.astype(np.float32)) * np.float32(1.0 / 15.0), 0).astype(np.float16)
    sf, mf = s.astype(np.float32)[..., None], m.astype(np.float32)[..., None]
    with np.errstate(divide="ignore", invalid="ignore"):
        q = np.where(sf > 0, np.clip(np.rint((g - mf) / sf), 0, 15), 0)
    return (q.astype(np.float64) * sf.astype(np.float64) + mf.astype(np.float64)).reshape(x.shape)


def _exact_attend(st, c):
    b, hk, d, s = c["batch"], c["kv_heads"], c["head_dim"], c["seq"]
    grp = c["heads"] // hk
    out = torch.zeros((b, c["heads"], s, d), dtype=torch.float64, device="cuda")
    for row in range(b):
        slot, start = int(st["slots"][row]), int(st["starts"][row])
        n = start + s
        for h in range(hk):
            kv = []
            for name in ("k", "v"):
                codes, par = st["codes_" + name][slot, 0, h, :n], st["par_" + name][slot, 0, h, :n].double()
                val = torch.empty((n, d), dtype=torch.float64, device="cuda")
                val[:, 0::2], val[:, 1::2] = (codes % 16).double(), (codes // 16).double()
                kv.append(val * par[:, :, 0].repeat_interleave(GROUP, 1) + par[:, :, 1].repeat_interleave(GROUP, 1))
            for j in range(grp):
                x = st["q"][row, h * grp + j].double() @ kv[0].t() / math.sqrt(d)
                x += torch.full((s, n), -math.inf, dtype=torch.float64, device="cuda").triu(start + 1)
                out[row, h * grp + j] = torch.softmax(x, -1) @ kv[1]
    return out


def _exact_logprobs(st, c):
    lp, ent, top = [], [], []
    for at in range(0, c["rows"], 64):
        x = st["logits"][at: at + 64].double()
        q = x - torch.logsumexp(x, 1, keepdim=True)
        lp.append(q.gather(1, st["tokens"][at: at + 64].long()[:, None])[:, 0])
        ent.append(-(q.exp() * q).sum(1))
        top.append(torch.topk(q, c["top"], dim=1).values)
    return {"logprob": torch.cat(lp), "entropy": torch.cat(ent), "rank": None, "top_ids": None,
            "top_logprobs": torch.cat(top)}
