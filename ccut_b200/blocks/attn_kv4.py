"""4-bit kv caches and the attention that reads them (``ccut_kv4_*``).

A cache row (one position of one kv head) keeps 4-bit codes with one fp16 pair (scale, minimum)
per 64 features: 36 bytes per 64 features where the bf16 caches keep 128.  ``Kv4Pool`` /
``Kv4Cache`` stand where ``model.KvPool`` / ``model.KvCache`` do (``MoeDecoder.new_pool(...,
kv_dtype="int4")``, ``GenericBackend(..., kv_dtype="int4")``, ``[quant] kv_cache_dtype =
"int4"``).  The reference keeps fp32 arrays (``ccut/models/generic.py:304-345``); there is no
reference counterpart of the format.

- ``kv4_append(pool, layer, k, v, slots, positions)`` quantizes new rows into the pool;
- ``kv4_attention(q, pool, layer, slots, starts)`` attends over it, a batch of sequences of
  different lengths in one call (decode steps and prompt chunks);
- ``kv4_read(pool, layer, slots, positions)`` gives rows back as the values they stand for.

The tensors are on one CUDA device; the calls run on that device's current stream.  Head dims
64 and 128.
"""

from __future__ import annotations

import torch

from ccut_b200 import _lib
from ccut_b200.layer import _run

__all__ = ["GROUP", "Kv4Cache", "Kv4Pool", "kv4_append", "kv4_attention", "kv4_read"]

GROUP = 64  # features per (scale, minimum) pair

_DTYPES = {torch.bfloat16: _lib.OUT_BF16, torch.float32: _lib.OUT_F32}
_words: dict = {}  # device -> the status word of its wrapped pools, and its address


def _device_word(device: torch.device) -> tuple:
    """One status word for all wrapped pools of a device that were given none: wrapping launches nothing."""
    word = _words.get(device)
    if word is None:
        t = torch.zeros(1, dtype=torch.int32, device=device)
        word = (t, t.data_ptr())
        if device.type != "cuda" or not torch.cuda.is_current_stream_capturing():  # a graph's memory is the graph's
            _words[device] = word
    return word


def read_status(word: torch.Tensor) -> int:
    """The code in a status word (0 = ok), which is cleared; waits for the current stream."""
    if word.device.type != "cuda":
        code = int(word)
        word.zero_()
        return code
    with torch.cuda.device(word.device):
        return _lib.load().ccut_workspace_status(word.data_ptr(), torch.cuda.current_stream().cuda_stream)


class Kv4Pool:
    """The 4-bit caches of up to ``slots`` sequences in one allocation: ``k`` / ``v`` codes
    ``[slots, layers, kv_heads, max_len, head_dim / 2]`` uint8 and ``k_par`` / ``v_par``
    ``[slots, layers, kv_heads, max_len, head_dim / 64, 2]`` fp16.  ``status`` (int32 ``[1]``, by default one of
    its own; pools may share one) keeps the error of an attention call whose bounded waits ran out
    until ``workspace_status`` reads it."""

    def __init__(self, slots: int, layers: int, kv_heads: int, max_len: int, head_dim: int, device="cuda",
                 status: torch.Tensor | None = None):
        if slots <= 0 or layers <= 0 or kv_heads <= 0 or max_len <= 0:
            raise ValueError("slots, layers, kv_heads and max_len must be positive")
        if head_dim not in (64, 128):
            raise NotImplementedError(f"head dim {head_dim} (have 64, 128)")
        rows = (slots, layers, kv_heads, max_len)
        self.k = torch.zeros(rows + (head_dim // 2,), dtype=torch.uint8, device=device)
        self.v = torch.zeros_like(self.k)
        self.k_par = torch.zeros(rows + (head_dim // GROUP, 2), dtype=torch.float16, device=device)
        self.v_par = torch.zeros_like(self.k_par)
        self._shape()
        self._report_to(torch.zeros(1, dtype=torch.int32, device=device) if status is None else status)

    @classmethod
    def wrap(cls, k: torch.Tensor, k_par: torch.Tensor, v: torch.Tensor, v_par: torch.Tensor,
             status: torch.Tensor | None = None) -> "Kv4Pool":
        """A pool over existing tensors of the layout above (contiguous, nothing copied); without a
        ``status`` of its own it shares one with the device's other such pools."""
        shape = tuple(k.shape)
        if len(shape) != 5 or k.dtype != torch.uint8 or shape[4] not in (32, 64):
            raise ValueError("k must be uint8 [slots, layers, kv_heads, max_len, 32 or 64]")
        par = shape[:4] + (shape[4] // 32, 2)
        if v.dtype != torch.uint8 or v.shape != shape or k_par.shape != par or v_par.shape != par:
            raise ValueError("k, v, k_par and v_par must share slots, layers, kv_heads, max_len and head_dim")
        if k_par.dtype != torch.float16 or v_par.dtype != torch.float16:
            raise ValueError("k_par and v_par must be fp16")
        if not (k.is_contiguous() and v.is_contiguous() and k_par.is_contiguous() and v_par.is_contiguous()):
            raise ValueError("the pool's tensors must be contiguous")
        if not k.device == v.device == k_par.device == v_par.device:
            raise ValueError("the pool's tensors must be on one device")
        p = cls.__new__(cls)
        p.k, p.k_par, p.v, p.v_par = k, k_par, v, v_par
        p._shape()
        if status is None:
            p.status, p._status = _device_word(p.device)
        else:
            p._report_to(status)
        return p

    def workspace_status(self) -> int:
        """Device status word of the attention calls over this pool (0 = ok); clears it."""
        return read_status(self.status)

    def _report_to(self, status: torch.Tensor) -> None:
        if status.dtype != torch.int32 or status.shape != (1,) or status.device != self.device:
            raise ValueError(f"status must be int32 [1] on {self.device}")
        self.status, self._status = status, status.data_ptr()

    def _shape(self) -> None:
        self.slots, self.layers, self.kv_heads, self.max_len, half = self.k.shape
        self.head_dim = 2 * half
        self.device = self.k.device
        self.slot_rows = self.layers * self.kv_heads * self.max_len
        self._base = (self.k.data_ptr(), self.k_par.data_ptr(), self.v.data_ptr(), self.v_par.data_ptr())

    def _pointers(self, layer: int):
        """Device addresses of layer ``layer`` of slot 0: k codes, k params, v codes, v params."""
        if not 0 <= layer < self.layers:
            raise ValueError(f"layer {layer} outside the pool's {self.layers}")
        rows = layer * self.kv_heads * self.max_len
        c, p = rows * (self.head_dim // 2), rows * (self.head_dim // GROUP) * 4
        k, kp, v, vp = self._base
        return k + c, kp + p, v + c, vp + p

    def cache(self, slot: int) -> "Kv4Cache":
        return Kv4Cache.in_pool(self, slot)

    def bytes_per_position(self) -> int:
        return self.layers * self.kv_heads * self.head_dim // GROUP * 36 * 2


class Kv4Cache:
    """One sequence's 4-bit cache: slot ``slot`` of ``pool`` (a pool of one slot of its own when
    made directly), ``length`` positions valid."""

    def __init__(self, layers: int, kv_heads: int, max_len: int, head_dim: int, device="cuda",
                 status: torch.Tensor | None = None):
        self._take(Kv4Pool(1, layers, kv_heads, max_len, head_dim, device, status), 0)

    @classmethod
    def in_pool(cls, pool: Kv4Pool, slot: int) -> "Kv4Cache":
        if not 0 <= slot < pool.slots:
            raise ValueError(f"slot {slot} outside the pool's {pool.slots}")
        c = cls.__new__(cls)
        c._take(pool, slot)
        return c

    def _take(self, pool: Kv4Pool, slot: int) -> None:
        self.pool, self.slot, self.max_len, self.length = pool, int(slot), pool.max_len, 0

    def truncate(self, n: int) -> None:
        """Keep the first ``n`` positions (later ones are overwritten by the next forward)."""
        if not 0 <= n <= self.length:
            raise ValueError(f"cannot truncate {self.length} cached positions to {n}")
        self.length = int(n)


def _check_pool(pool, device) -> None:
    if not isinstance(pool, Kv4Pool):
        raise ValueError("pool must be a Kv4Pool")
    if device != pool.device:
        raise ValueError(f"tensors on {device} for a pool on {pool.device}")
    if device.type != "cuda":
        raise ValueError("the 4-bit cache runs on CUDA tensors only")


def _index(t: torch.Tensor, n: int, pool: Kv4Pool, name: str) -> torch.Tensor:
    if t.dtype != torch.int32 or t.shape != (n,) or t.device != pool.device:
        raise ValueError(f"{name} must be int32 [{n}] on {pool.device}")
    return t if t.is_contiguous() else t.contiguous()


def _rows(x: torch.Tensor, pool: Kv4Pool, name: str) -> tuple:
    """x ``[tokens, kv_heads, head_dim]`` bf16 or fp32 with strides the kernel reads in place: (x, tokens,
    address, dtype code, token stride, head stride)."""
    shape, dt = x.shape, _DTYPES.get(x.dtype)
    if len(shape) != 3 or shape[1] != pool.kv_heads or shape[2] != pool.head_dim:
        raise ValueError(f"{name} must be [tokens, {pool.kv_heads}, {pool.head_dim}], got {tuple(shape)}")
    if dt is None:
        raise ValueError(f"{name} must be bf16 or fp32")
    (st, sh, sd), p = x.stride(), x.data_ptr()
    if sd != 1 or (st | sh) % 8 or p % 16:
        x = x.clone(memory_format=torch.contiguous_format)
        (st, sh, _), p = x.stride(), x.data_ptr()
    return x, shape[0], p, dt, st, sh


def kv4_append(pool: Kv4Pool, layer: int, k: torch.Tensor, v: torch.Tensor, slots: torch.Tensor,
               positions: torch.Tensor) -> None:
    """Quantize ``k`` / ``v`` ``[tokens, kv_heads, head_dim]`` (bf16 or fp32, any strides) into rows
    ``(slots[t], positions[t])`` (int32) of ``layer``.  Pairs outside the pool are skipped; the
    pairs of one call must differ."""
    _check_pool(pool, k.device)
    k, n, kx, k_dt, k_st, k_sh = _rows(k, pool, "k")
    v, nv, vx, v_dt, v_st, v_sh = _rows(v, pool, "v")
    if nv != n or v.device != pool.device:
        raise ValueError("k and v must have the same tokens on the same device")
    slots, positions = _index(slots, n, pool, "slots"), _index(positions, n, pool, "positions")
    kc, kp, vc, vp = pool._pointers(layer)
    _run(pool.device, "ccut_kv4_append", kx, k_dt, k_st, k_sh, vx, v_dt, v_st, v_sh, n, pool.kv_heads, pool.head_dim,
         slots.data_ptr(), positions.data_ptr(), kc, kp, vc, vp, pool.max_len, pool.slot_rows, pool.slots)


def kv4_read(pool: Kv4Pool, layer: int, slots: torch.Tensor, positions: torch.Tensor,
             out_dtype: torch.dtype = torch.float32) -> tuple:
    """``(k, v)`` ``[tokens, kv_heads, head_dim]`` (fp32 or bf16): the values that rows
    ``(slots[t], positions[t])`` (int32) of ``layer`` stand for, zeros for pairs outside the pool."""
    _check_pool(pool, slots.device)
    n = slots.shape[0] if slots.dim() else 0
    slots, positions = _index(slots, n, pool, "slots"), _index(positions, n, pool, "positions")
    if out_dtype not in _DTYPES:
        raise ValueError("out_dtype must be bf16 or fp32")
    k = torch.empty((n, pool.kv_heads, pool.head_dim), dtype=out_dtype, device=pool.device)
    v = torch.empty_like(k)
    kc, kp, vc, vp = pool._pointers(layer)
    _run(pool.device, "ccut_kv4_read", kc, kp, vc, vp, slots.data_ptr(), positions.data_ptr(), n, pool.kv_heads,
         pool.head_dim, pool.max_len, pool.slot_rows, pool.slots, k.data_ptr(), v.data_ptr(), _DTYPES[out_dtype])
    return k, v


def kv4_attention(q: torch.Tensor, pool: Kv4Pool, layer: int, slots: torch.Tensor, starts: torch.Tensor,
                  kv_len: int | None = None, scale: float | None = None, softcap: float | None = None,
                  out_dtype: torch.dtype = torch.bfloat16) -> torch.Tensor:
    """q ``[batch, heads, seq, head_dim]`` bf16; batch row b attends over slot ``slots[b]`` of
    ``layer``, its query i over positions ``<= starts[b] + i`` (int32) -> ``[batch, heads, seq,
    head_dim]`` (bf16 or fp32).  ``kv_len``: an upper bound of ``starts[b] + seq`` when the host
    knows one (positions at or past it are not read); default: the pool's ``max_len``.  ``scale``: None (or 0) for
    ``head_dim ** -0.5``.  Up to 128 query rows per kv head (``heads / kv_heads * seq``) the codes themselves
    are multiplied, and fp32 output is off by about 1e-6 of the largest value; more rows round k, v and the
    probabilities to fp16 (11 bits), whatever ``out_dtype``.  A call whose
    bounded waits ran out leaves zero rows and an error for ``pool.workspace_status()``."""
    _check_pool(pool, q.device)
    shape = q.shape
    if q.dtype != torch.bfloat16 or len(shape) != 4 or shape[3] != pool.head_dim:
        raise ValueError(f"q must be bf16 [batch, heads, seq, {pool.head_dim}]")
    b, h, s, d = shape
    if h == 0 or h % pool.kv_heads:
        raise ValueError(f"heads ({h}) must be a positive multiple of kv_heads ({pool.kv_heads})")
    if out_dtype not in _DTYPES:
        raise ValueError("out_dtype must be bf16 or fp32")
    n = pool.max_len if kv_len is None else int(kv_len)
    if not 0 <= n <= pool.max_len:
        raise ValueError(f"kv_len {n} outside [0, {pool.max_len}]")
    slots, starts = _index(slots, b, pool, "slots"), _index(starts, b, pool, "starts")
    q = q if q.is_contiguous() else q.contiguous()
    if q.data_ptr() % 16:
        q = q.clone()
    out = torch.empty_like(q) if out_dtype == torch.bfloat16 else torch.empty_like(q, dtype=out_dtype)
    kc, kp, vc, vp = pool._pointers(layer)
    nbytes = _lib.load().ccut_kv4_attention_workspace_bytes(b, h, pool.kv_heads, s, n, d)
    ws = torch.empty(nbytes, dtype=torch.uint8, device=q.device) if nbytes > 256 else None  # 256: none is used
    _run(pool.device, "ccut_kv4_attention_reported", q.data_ptr(), kc, kp, vc, vp, slots.data_ptr(), starts.data_ptr(), b, h,
         pool.kv_heads, s, d, pool.max_len, n, pool.slot_rows, pool.slots, float(scale or 0.0), float(softcap or 0.0),
         out.data_ptr(), _DTYPES[out_dtype], ws.data_ptr() if ws is not None else None, nbytes, pool._status)
    return out
