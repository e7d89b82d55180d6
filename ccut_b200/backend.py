"""Engine backend over ``MoeDecoder``: the served path of the reference's ``Engine`` reaches the
GPU decoder through it.

``Engine._backend_step`` (``ccut/engine.py:305-333``) calls, for every scheduled request,
``backend.generate_step(prompt[:prefill_consumed] + generated, sampling_params=...)`` and takes
one token id back (errors evict that request).  ``GenericBackend`` answers that call:

* it keeps up to ``max_seqs`` sequence caches (``KvCache``, bf16 k / v in HBM) keyed by the
  token ids they hold.  A call reuses the cache with the longest common prefix of its ids (at
  least one token is always recomputed, for its logits), truncates it there and runs the rest
  as prefill chunks of at most ``prefill_chunk`` tokens.  A request that grows by one token per
  step therefore runs one token per step; chunked prefill runs each new chunk once; a request
  that diverges from a cached one (a shared prompt, a retried step) keeps the shared part.
  With all slots held, the least recently used cache is taken;
* it samples the next token from the last position's logits on the device
  (``ccut_b200.sampling.sample``: greedy at ``temperature <= 0``, else the reference's
  temperature / top-k / min-p / top-p transform and one draw from a seeded generator).

``generate_batch([(input_ids, sampling_params), ...])`` answers a whole engine step at once
(the loop of ``_backend_step`` as one call): the requests' new ids run through one decoder
pass per prefill chunk, so their MoE blocks see all the step's tokens together.

``sampling_params["adapter"]`` names the request's low-rank adapter (an index into the layers' banks; None or
absent: none); a cache serves only requests of the adapter it was computed with.  ``generate_step`` and
``generate_batch`` with ``logprobs=n`` also answer each token's log probability, its rank, the entropy and the
``n`` best alternatives (``ccut_b200.logprobs``, on the logits before temperature and filters); ``score``
answers them for the tokens of a given text.

Over 4-bit caches a step whose attention ran out of one of its bounded waits raises ``TimeoutError``
(the reference's class for a stalled wait, ccut/experts/reader.py:327); the caches are emptied, so the next
call of the request computes its prompt again.

``generate`` and ``forward_step`` give the interface of the reference's fallback backend
(``L1Backend``, ``ccut/models/backend_transformers.py:31-124``), which the engine uses when a
backend has no ``generate_step``: ``forward_step(input_ids, past)`` returns the logits of the
last id and the cache to pass back, ``generate`` loops it with a ``sampling(logits, position)``
callable (greedy by default) and stops at ``eos_token_id``.
"""

from __future__ import annotations

from typing import Any, Callable

import numpy as np
import torch

from ccut_b200 import _lib
from ccut_b200.logprobs import MAX_TOP, token_logprobs
from ccut_b200.model import KvCache, MoeDecoder
from ccut_b200.sampling import sample

__all__ = ["GenericBackend", "common_prefix"]


def common_prefix(a: list[int], b: list[int]) -> int:
    """Length of the longest common prefix of two id lists."""
    n = min(len(a), len(b))
    if a[:n] == b[:n]:
        return n
    x = np.asarray(a[:n], dtype=np.int64)
    y = np.asarray(b[:n], dtype=np.int64)
    return int(np.argmax(x != y))


class _Seq:
    def __init__(self, cache: KvCache):
        self.cache = cache
        self.ids: list[int] = []
        self.adapter = None  # what the cached positions were computed with: (adapter, of which set), None for none


class GenericBackend:
    """``generate_step`` backend for the reference's ``Engine`` over a ``MoeDecoder``."""

    tier = "L0"

    def __init__(self, model: MoeDecoder, max_seqs: int = 4, max_len: int = 4096, prefill_chunk: int = 4096,
                 seed: int = 0, eos_token_id: int | None = None, pool: bool = False, kv_dtype: str | None = None):
        """``pool``: keep the sequence caches in one ``KvPool``, so that a decode step of several
        requests (``generate_batch``) runs one attention launch per layer.  ``kv_dtype``: ``"bf16"``,
        ``"int4"`` (4-bit caches, ``blocks.attn_kv4``) or None (the model's ``kv_dtype``)."""
        if max_seqs < 1 or max_len < 1 or prefill_chunk < 1:
            raise ValueError("max_seqs, max_len and prefill_chunk must be positive")
        self.model = model
        self._cache_args = {} if kv_dtype is None else {"kv_dtype": kv_dtype}
        self._pool = model.new_pool(max_seqs, max_len, **self._cache_args) if pool else None
        self.max_seqs, self.max_len, self.prefill_chunk = int(max_seqs), int(max_len), int(prefill_chunk)
        self.eos_token_id = eos_token_id
        self._seqs: list[_Seq] = []  # least recently used first
        self._gen = torch.Generator(device=model.device)
        self._gen.manual_seed(int(seed))
        self.tokens_run = 0  # positions the decoder computed (prefix reuse skips the rest)

    # ---- sequence caches ---------------------------------------------------------------
    def _acquire(self, ids: list[int], taken: list, adapter: int | None = None) -> tuple[_Seq, int]:
        """The cache to run ``ids`` in (not one of ``taken``) and how many of its positions stay: those
        of a common prefix computed with the same adapter."""
        best, best_p = None, 0
        key = None if adapter is None else (adapter, self.model.adapters_set)
        for s in self._seqs:
            if any(s is t for t in taken) or s.adapter != key:
                continue
            p = common_prefix(s.ids, ids)
            if p > best_p:
                best, best_p = s, p
        reuse = min(best_p, len(ids) - 1)
        if best is None or reuse == 0:
            reuse = 0
            if len(self._seqs) < self.max_seqs:
                cache = (self._pool.cache(len(self._seqs)) if self._pool is not None
                         else self.model.new_cache(self.max_len, **self._cache_args))
                best = _Seq(cache)
            else:
                free = [s for s in self._seqs if not any(s is t for t in taken)]
                if not free:
                    raise ValueError(f"a batch of more than max_seqs={self.max_seqs} sequences")
                best = free[0]  # least recently used
        if any(best is s for s in self._seqs):
            self._seqs.remove(best)
        self._seqs.append(best)
        best.adapter = key
        return best, reuse

    def _check(self, input_ids) -> list[int]:
        ids = [int(t) for t in input_ids]
        if not ids:
            raise ValueError("generate_step needs at least one input id")
        if len(ids) > self.max_len:
            raise ValueError(f"{len(ids)} ids exceed the backend's max_len of {self.max_len}")
        return ids

    def _check_waits(self) -> None:
        """Raises when a bounded wait of the attention over 4-bit caches ran out since the last check; no
        cache is reused then."""
        code = self.model.kv_status()
        if code:
            for s in self._seqs:
                s.cache.truncate(0)
                s.ids = []
            _lib.check(code, "attention over 4-bit caches")

    def logits_batch(self, id_lists, adapters=None) -> list:
        """fp32 logits ``[vocab]`` of the last id of every list, the lists run together: each
        call of the decoder takes the next ``prefill_chunk`` ids (at most) of every list that
        has ids left, so decoding sequences share their MoE passes.  ``adapters``: the adapter of
        every list (or None), default none."""
        out = self._logits(id_lists, adapters)
        self._check_waits()
        return out

    def _logits(self, id_lists, adapters) -> list:
        lists = [self._check(ids) for ids in id_lists]
        adapters = [None] * len(lists) if adapters is None else list(adapters)
        if len(adapters) != len(lists):
            raise ValueError(f"{len(adapters)} adapters for {len(lists)} id lists")
        for a in adapters:
            if a is not None:
                self.model._adapter(a)  # refused before any cache is taken
        seqs: list[_Seq] = []
        pos: list[int] = []
        for ids, adapter in zip(lists, adapters):
            seq, reuse = self._acquire(ids, seqs, adapter)
            seq.cache.truncate(min(reuse, seq.cache.length))
            seq.ids = ids[: seq.cache.length]
            seqs.append(seq)
            pos.append(reuse)
        out: list = [None] * len(lists)
        while True:
            todo = [j for j in range(len(lists)) if pos[j] < len(lists[j])]
            if not todo:
                return out
            ends = [min(len(lists[j]), pos[j] + self.prefill_chunk) for j in todo]
            logits = self.model.forward_batch(
                [(lists[j][pos[j]: e], seqs[j].cache, pos[j]) + (() if adapters[j] is None else (adapters[j],))
                 for j, e in zip(todo, ends)])
            for j, e, lg in zip(todo, ends, logits):
                self.tokens_run += e - pos[j]
                seqs[j].ids = lists[j][:e]
                pos[j] = e
                if e == len(lists[j]):
                    out[j] = lg

    def logits_for(self, input_ids, adapter: int | None = None) -> torch.Tensor:
        """fp32 logits ``[vocab]`` of the last of ``input_ids`` (runs what no cache holds)."""
        return self.logits_batch([input_ids], [adapter])[0]

    # ---- Engine interface ----------------------------------------------------------------
    def generate_step(self, input_ids, sampling_params: dict | None = None, logprobs: int | None = None):
        """The next token id; with ``logprobs`` = n, ``(id, answer)`` as ``generate_batch``."""
        if logprobs is not None:
            return self.generate_batch([(input_ids, sampling_params)], logprobs)[0]
        return self.generate_batch([(input_ids, sampling_params)])[0]

    def generate_batch(self, requests, logprobs: int | None = None) -> list:
        """``requests`` = ``[(input_ids, sampling_params), ...]``, one per scheduled request of an
        engine step (at most ``max_seqs``): the next token of each, from one batched pass.  With
        ``logprobs`` = n, ``(token, answer)`` of each, ``answer`` a dict of the token's ``logprob``
        and ``rank``, the distribution's ``entropy`` (nats) and the n best ``top`` as ``(id,
        logprob)``, from the logits before temperature and filters."""
        requests = list(requests)
        top_n = None if logprobs is None else self._alternatives(logprobs)
        logits = self._logits([r[0] for r in requests], [(r[1] or {}).get("adapter") for r in requests])
        tokens = [sample(lg, r[1], self._gen) for lg, r in zip(logits, requests)]
        self._check_waits()  # the tokens were waited for
        if logprobs is None:
            return tokens
        if not requests:
            return []
        return list(zip(tokens, self._answers(torch.stack([lg.reshape(-1) for lg in logits]), tokens, top_n)))

    def _alternatives(self, n) -> int:  # refused before anything runs
        if isinstance(n, bool) or not isinstance(n, (int, np.integer)) or not 0 <= n <= self.model.vocab:
            raise ValueError(f"alternatives must be an int in [0, {self.model.vocab}], got {n!r}")
        if n > MAX_TOP:
            raise NotImplementedError(f"{n} alternatives (have up to {MAX_TOP})")
        return int(n)

    @staticmethod
    def _answers(logits: torch.Tensor, tokens, top_n: int) -> list:
        r = token_logprobs(logits, torch.as_tensor(tokens, dtype=torch.int32).to(logits.device), top_n)
        lp, ent, rank = r.logprob.tolist(), r.entropy.tolist(), r.rank.tolist()
        ids, tops = r.top_ids.tolist(), r.top_logprobs.tolist()
        return [{"logprob": lp[i], "rank": rank[i], "entropy": ent[i], "top": list(zip(ids[i], tops[i]))}
                for i in range(len(lp))]

    def score(self, input_ids, top_n: int = 0, adapter: int | None = None) -> list:
        """The answers (as ``generate_batch``) for ``input_ids[1:]``, each given the ids before it.  Runs in
        a cache of its own, ``min(prefill_chunk, 1024)`` positions at a time (the logits of one chunk are
        held at once)."""
        ids, top_n = self._check(input_ids), self._alternatives(top_n)
        out: list = []
        if len(ids) < 2:
            return out
        cache = self.model.new_cache(len(ids) - 1, **self._cache_args)
        step = min(self.prefill_chunk, 1024)
        for c0 in range(0, len(ids) - 1, step):
            c1 = min(len(ids) - 1, c0 + step)
            extra = {} if adapter is None else {"adapter": adapter}
            logits = self.model.forward(ids[c0:c1], cache, c0, all_logits=True, **extra)
            self.tokens_run += c1 - c0
            out += self._answers(logits, ids[c0 + 1: c1 + 1], top_n)
            self._check_waits()
        return out

    # ---- L1Backend interface -------------------------------------------------------------
    def forward_step(self, input_ids, past: Any = None) -> tuple[torch.Tensor, KvCache]:
        """``input_ids`` the whole sequence so far; ``past`` the cache a previous call returned
        (its positions must be a prefix of ``input_ids``) or None.  Returns ``(logits [1, vocab],
        cache)``."""
        ids = [int(t) for t in input_ids]
        if not ids:
            raise ValueError("forward_step needs at least one input id")
        cache = past if past is not None else self.model.new_cache(self.max_len, **self._cache_args)
        if len(ids) > cache.max_len:
            raise ValueError(f"{len(ids)} ids exceed the cache's max_len of {cache.max_len}")
        start = min(cache.length, len(ids) - 1)
        cache.truncate(start)
        logits = None
        for c0 in range(start, len(ids), self.prefill_chunk):
            c1 = min(len(ids), c0 + self.prefill_chunk)
            logits = self.model.forward(ids[c0:c1], cache, c0)
            self.tokens_run += c1 - c0
        try:
            self._check_waits()
        except TimeoutError:
            cache.truncate(start)
            raise
        return logits.reshape(1, -1), cache

    def generate(self, token_ids, max_tokens: int, on_token: Callable[[int], None] | None = None,
                 sampling: Callable[[Any, int], int] | None = None) -> list[int]:
        if sampling is None:
            def sampling(logits, pos):
                return int(torch.argmax(logits.reshape(-1)).item())
        past = None
        current = [int(t) for t in token_ids]
        out: list[int] = []
        for _ in range(int(max_tokens)):
            logits, past = self.forward_step(current, past)
            tok = int(sampling(logits, len(out)))
            out.append(tok)
            if on_token is not None:
                on_token(tok)
            current.append(tok)
            if self.eos_token_id is not None and tok == self.eos_token_id:
                break
        return out
