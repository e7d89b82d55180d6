"""Log probabilities of given tokens, their entropy and rank, and the top alternatives
(``ccut_token_logprobs``): what an engine answers besides the sampled ids, and what scoring a
prompt needs.  One pass over the logits; the reference has no counterpart (its engine answers
with token ids only, ``ccut/engine.py:335-352``)."""

from __future__ import annotations

from typing import NamedTuple

import torch

from ccut_b200 import _lib
from ccut_b200.layer import _run

__all__ = ["MAX_TOP", "TokenLogprobs", "token_logprobs"]

MAX_TOP = 32

_DTYPES = {torch.bfloat16: _lib.OUT_BF16, torch.float32: _lib.OUT_F32}


class TokenLogprobs(NamedTuple):
    logprob: torch.Tensor  # fp32 [rows]: log softmax(row)[token]
    entropy: torch.Tensor  # fp32 [rows], in nats
    rank: torch.Tensor  # int32 [rows], 1 = the first in the order (value descending, index ascending)
    top_ids: torch.Tensor  # int32 [rows, top_n], the first top_n of that order
    top_logprobs: torch.Tensor  # fp32 [rows, top_n]


def token_logprobs(logits: torch.Tensor, tokens: torch.Tensor, top_n: int = 0) -> TokenLogprobs:
    """``logits [rows, vocab]`` (bf16 or fp32, unit stride along the vocabulary), ``tokens`` int32
    ``[rows]``, all on one CUDA device.  A token outside the vocabulary has logprob NaN and rank
    0; logits of ``-inf`` have probability 0; a row with NaN, ``+inf`` or nothing but ``-inf`` has
    NaN log probabilities.  ``top_n`` <= 32."""
    if logits.dim() != 2 or logits.dtype not in _DTYPES or not logits.is_cuda:
        raise ValueError("logits must be bf16 or fp32 [rows, vocab] on a CUDA device")
    rows, vocab = logits.shape
    if tokens.dtype != torch.int32 or tokens.dim() != 1 or tokens.shape[0] != rows or tokens.device != logits.device:
        raise ValueError(f"tokens must be int32 [{rows}] on {logits.device}")
    if vocab == 0 or not 0 <= top_n <= vocab:
        raise ValueError(f"top_n = {top_n} of a vocabulary of {vocab}")
    if top_n > MAX_TOP:
        raise NotImplementedError(f"top_n = {top_n} (have up to {MAX_TOP})")
    if logits.stride(1) != 1 or (rows > 1 and logits.stride(0) < vocab):
        logits = logits.contiguous()
    tokens = tokens if tokens.is_contiguous() else tokens.contiguous()
    dev = logits.device
    logprob = torch.empty(rows, dtype=torch.float32, device=dev)
    entropy, rank = torch.empty_like(logprob), torch.empty_like(tokens)
    ids = torch.empty((rows, top_n), dtype=torch.int32, device=dev)
    top = torch.empty((rows, top_n), dtype=torch.float32, device=dev)
    _run(dev, "ccut_token_logprobs", logits.data_ptr(), _DTYPES[logits.dtype], rows, vocab,
         logits.stride(0) if rows > 1 else vocab, tokens.data_ptr(), top_n, logprob.data_ptr(), entropy.data_ptr(),
         rank.data_ptr(), ids.data_ptr(), top.data_ptr())
    return TokenLogprobs(logprob, entropy, rank, ids, top)
