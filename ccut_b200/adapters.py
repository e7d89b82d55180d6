"""Low-rank adapters of many requests at once beside a shared projection (``ccut_lora_add``).

A ``LoraBank`` holds the adapters of one projection: ``out[t] = base[t] + scales[i] * B_i A_i
x[t]`` with ``i = ids[t]``, each token with its own adapter or none (-1).  A fused projection
(q, k and v side by side) is one bank with a width per part.  ``DecoderLayer(..., adapters=
{"qkv": bank, "o": bank})`` adds them to a decoder layer's projections; ``MoeDecoder.forward``
and ``GenericBackend`` (``sampling_params["adapter"]``) take an adapter per request.  The
reference has no counterpart."""

from __future__ import annotations

import ctypes as C

import numpy as np
import torch

from ccut_b200 import _lib
from ccut_b200.layer import _run

__all__ = ["LoraBank"]

_DTYPES = {torch.bfloat16: _lib.OUT_BF16, torch.float32: _lib.OUT_F32}
MAX_SLICES, MAX_RANKS = 4, 256


class LoraBank:
    """``a`` bf16 ``[adapters, parts * rank, inputs]``, ``b`` bf16 ``[adapters, sum(widths), rank]``,
    ``scales`` fp32 ``[adapters]`` on one CUDA device; ``widths`` the output features of each
    part (multiples of 8); part j's outputs take rank rows ``j * rank ..`` of ``a``.  ``rank`` is a
    multiple of 16 with ``parts * rank <= 256``, ``inputs`` a multiple of 8 (``from_matrices``
    pads other ranks with zeros)."""

    def __init__(self, a: torch.Tensor, b: torch.Tensor, scales: torch.Tensor, widths):
        widths = [int(w) for w in widths]
        if a.dim() != 3 or b.dim() != 3 or a.dtype != torch.bfloat16 or b.dtype != torch.bfloat16:
            raise ValueError("a and b must be bf16 [adapters, parts * rank, inputs] and [adapters, outputs, rank]")
        n, ranks, inputs = a.shape
        outputs, rank = b.shape[1], b.shape[2]
        parts = len(widths)
        if b.shape[0] != n or ranks != parts * rank or outputs != sum(widths) or parts == 0:
            raise ValueError(f"a {tuple(a.shape)} and b {tuple(b.shape)} do not fit widths {widths}")
        if rank == 0 or rank % 16 or inputs == 0 or inputs % 8 or any(w <= 0 or w % 8 for w in widths):
            raise ValueError("rank must be a positive multiple of 16, inputs and widths of 8")
        if parts > MAX_SLICES or ranks > MAX_RANKS:
            raise NotImplementedError(f"{parts} parts of rank {rank} (have up to {MAX_SLICES} parts, {MAX_RANKS} ranks)")
        if scales.dtype != torch.float32 or scales.dim() != 1 or scales.shape[0] != n:
            raise ValueError(f"scales must be fp32 [{n}]")
        if not a.device == b.device == scales.device:
            raise ValueError("a, b and scales must be on one device")
        self.a, self.b, self.scales = (t if t.is_contiguous() else t.contiguous() for t in (a, b, scales))
        self.adapters, self.rank, self.inputs, self.outputs, self.widths = n, rank, inputs, outputs, widths
        self.device = a.device
        self._widths = (C.c_int * parts)(*widths)

    @classmethod
    def from_matrices(cls, adapters: list, device="cuda") -> "LoraBank":
        """From per-adapter matrices as checkpoints hold them: ``adapters[i]`` = ``(parts, scale)``
        with ``parts`` a list of ``(A [r, inputs], B [width, r])``, one per part of the projection;
        ``scale`` is ``alpha / r``.  A part may be None (not adapted: zeros).  Ranks may differ;
        all are padded with zero rows to the next multiple of 16 of the largest."""
        if not adapters:
            raise ValueError("a bank needs at least one adapter")
        mats = [[None if m is None else tuple(_matrix(x) for x in m) for m in parts] for parts, _ in adapters]
        count = len(mats[0])
        if count == 0 or any(len(m) != count for m in mats):
            raise ValueError("every adapter needs the same parts")
        widths, inputs, rank = [], None, 1
        for j in range(count):
            have = [m[j] for m in mats if m[j] is not None]
            if not have:
                raise ValueError(f"no adapter has part {j}: its width is unknown")
            widths.append(have[0][1].shape[0])
            for A, B in have:
                if A.dim() != 2 or B.dim() != 2 or A.shape[0] != B.shape[1] or B.shape[0] != widths[j]:
                    raise ValueError(f"part {j}: A {tuple(A.shape)} and B {tuple(B.shape)} do not fit")
                inputs = A.shape[1] if inputs is None else inputs
                if A.shape[1] != inputs:
                    raise ValueError(f"part {j}: A has {A.shape[1]} inputs, others {inputs}")
                rank = max(rank, A.shape[0])
        rank = (rank + 15) // 16 * 16
        a = torch.zeros((len(mats), count * rank, inputs), dtype=torch.bfloat16)
        b = torch.zeros((len(mats), sum(widths), rank), dtype=torch.bfloat16)
        for i, m in enumerate(mats):
            at = 0
            for j in range(count):
                if m[j] is not None:
                    A, B = m[j]
                    a[i, j * rank: j * rank + A.shape[0]] = A
                    b[i, at: at + widths[j], : B.shape[1]] = B
                at += widths[j]
        scales = torch.tensor([float(s) for _, s in adapters], dtype=torch.float32)
        return cls(a.to(device), b.to(device), scales.to(device), widths)

    def add(self, base: torch.Tensor, x: torch.Tensor, ids: torch.Tensor, out: torch.Tensor | None = None) -> torch.Tensor:
        """``base [tokens, outputs]`` (bf16 or fp32) plus the adapters' products with ``x [tokens,
        inputs]`` bf16; ``ids`` int32 ``[tokens]``, -1 (or any id outside the bank) for none.
        Returns ``out`` (new by default; ``out=base`` adds in place)."""
        if base.dim() != 2 or base.shape[1] != self.outputs or base.dtype not in _DTYPES:
            raise ValueError(f"base must be bf16 or fp32 [tokens, {self.outputs}]")
        n = base.shape[0]
        if x.dtype != torch.bfloat16 or x.dim() != 2 or tuple(x.shape) != (n, self.inputs):
            raise ValueError(f"x must be bf16 [{n}, {self.inputs}]")
        if ids.dtype != torch.int32 or ids.dim() != 1 or ids.shape[0] != n:
            raise ValueError(f"ids must be int32 [{n}]")
        if not self.a.is_cuda:
            raise ValueError("adapters run on CUDA tensors only")
        if not base.device == x.device == ids.device == self.device:
            raise ValueError(f"base, x and ids must be on {self.device}")
        if out is None:
            out = torch.empty_like(base, memory_format=torch.contiguous_format)
        elif out.dtype != base.dtype or out.shape != base.shape or out.device != base.device or not _rows_ok(out):
            raise ValueError("out must be like base, its rows contiguous and 16-byte aligned")
        base = base if _rows_ok(base) else base.clone(memory_format=torch.contiguous_format)
        x = x if x.is_contiguous() and x.data_ptr() % 16 == 0 else x.clone(memory_format=torch.contiguous_format)
        ids = ids if ids.is_contiguous() else ids.contiguous()
        nbytes = _lib.load().ccut_lora_workspace_bytes(n, self.inputs, self.rank, len(self.widths), self.adapters)
        ws = torch.empty(nbytes, dtype=torch.uint8, device=self.device) if nbytes else None
        _run(self.device, "ccut_lora_add", x.data_ptr(), self.a.data_ptr(), self.b.data_ptr(), self.scales.data_ptr(),
             ids.data_ptr(), n, self.inputs, self.rank, self.adapters, len(self.widths), self._widths, base.data_ptr(),
             base.stride(0), out.data_ptr(), out.stride(0), _DTYPES[base.dtype], ws.data_ptr() if nbytes else None, nbytes)
        return out


def _matrix(x) -> torch.Tensor:
    return x.detach().cpu() if isinstance(x, torch.Tensor) else torch.from_numpy(np.asarray(x, dtype=np.float32))


def _rows_ok(t: torch.Tensor) -> bool:
    """Rows that the kernel reads in place: unit stride, 16-byte aligned starts."""
    return t.stride(1) == 1 and t.stride(0) % 8 == 0 and t.stride(0) >= t.shape[1] and t.data_ptr() % 16 == 0
