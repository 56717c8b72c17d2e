"""A KV cache held in 4 or 8 bits.

``QuantizedKV`` owns (or wraps) one layer's buffers in the layout of
``core_kvq_t`` (include/core_b200.h) and keeps each sequence's token count on
the device; ``append`` quantises rows into it as they come, ``read`` gives them
back in the model's dtype and ``attend`` runs attention straight on the codes.
The kernels are reached through ``ops.kv_quantize``, ``ops.kv_dequantize`` and
``ops.attention_quantized``, which take the cache and explicit places.
"""

from __future__ import annotations

import ctypes

import torch

from . import _lib, ops

CAPACITY_STEP = 128


def _normal_tensors():
    """A cache outlives the forward that creates it: its tensors are changed in place
    later, which those made under inference_mode do not allow outside of it."""
    return torch.inference_mode(False)


class QuantizedKV:
    """One layer's K and V in 4 or 8 bits.

    k_codes, v_codes : (B, Hkv, capacity, 16 * bits) uint8
    k_meta, v_meta   : (B, Hkv, capacity, 128 / group, 2) float16, (scale, zero)
    lengths          : (B,) int32 on the device, tokens of each sequence
    max_length       : host-side bound of ``lengths``
    """

    __slots__ = ("k_codes", "k_meta", "v_codes", "v_meta", "bits", "group", "batch", "n_kv_heads",
                 "capacity", "index", "handle", "_lengths", "max_length")

    def __init__(self, k_codes: torch.Tensor, k_meta: torch.Tensor, v_codes: torch.Tensor,
                 v_meta: torch.Tensor):
        """Wraps existing buffers (their rows are the caller's; lengths start at 0)."""
        shape, meta_shape = k_codes.shape, k_meta.shape
        if len(shape) != 4 or len(meta_shape) != 5:
            raise ValueError("codes must be (B, Hkv, capacity, 16 * bits), meta "
                             "(B, Hkv, capacity, 128 / group, 2)")
        B, H, cap, width = shape
        groups = meta_shape[3]
        if width not in (64, 128) or groups not in (1, 2, 4):
            raise ValueError("a row takes 64 (4 bits) or 128 (8 bits) bytes and 1, 2 or 4 groups")
        if B <= 0 or H <= 0 or cap <= 0 or cap % CAPACITY_STEP:
            raise ValueError(f"capacity must be a positive multiple of {CAPACITY_STEP}")
        at = k_codes.get_device()
        if at < 0 or k_meta.get_device() != at or v_codes.get_device() != at or v_meta.get_device() != at:
            raise ValueError("core_b200 operates on CUDA tensors only, all on one device")
        if (v_codes.shape != shape or k_codes.dtype is not torch.uint8 or v_codes.dtype is not torch.uint8
                or not k_codes.is_contiguous() or not v_codes.is_contiguous()):
            raise ValueError("codes must be contiguous uint8 tensors of one shape")
        if (meta_shape != (B, H, cap, groups, 2) or v_meta.shape != meta_shape
                or k_meta.dtype is not torch.float16 or v_meta.dtype is not torch.float16
                or not k_meta.is_contiguous() or not v_meta.is_contiguous()):
            raise ValueError("meta must be contiguous float16 tensors (B, Hkv, capacity, groups, 2)")
        self.k_codes, self.k_meta, self.v_codes, self.v_meta = k_codes, k_meta, v_codes, v_meta
        self.bits, self.group = width // 16, 128 // groups
        self.batch, self.n_kv_heads, self.capacity = B, H, cap
        self.index = at
        # the core_kvq_t that the C-ABI takes
        self.handle = ctypes.byref(_lib.CoreKvq(
            k_codes.data_ptr(), k_meta.data_ptr(), v_codes.data_ptr(), v_meta.data_ptr(), B, H, cap,
            self.bits, self.group))
        self._lengths = None
        self.max_length = 0

    @classmethod
    def empty(cls, batch: int, n_kv_heads: int, capacity: int, *, bits: int = 4, group: int = 64,
              device="cuda") -> "QuantizedKV":
        """An empty cache with room for ``capacity`` tokens a sequence (rounded up to 128)."""
        if bits not in (4, 8) or group not in (32, 64, 128):
            raise ValueError("bits must be 4 or 8 and group 32, 64 or 128")
        if batch <= 0 or n_kv_heads <= 0 or capacity <= 0:
            raise ValueError("batch, n_kv_heads and capacity must be positive")
        cap = -(-int(capacity) // CAPACITY_STEP) * CAPACITY_STEP
        codes = (batch, n_kv_heads, cap, 16 * bits)
        meta = (batch, n_kv_heads, cap, 128 // group, 2)
        with _normal_tensors():
            return cls(torch.empty(codes, dtype=torch.uint8, device=device),
                       torch.empty(meta, dtype=torch.float16, device=device),
                       torch.empty(codes, dtype=torch.uint8, device=device),
                       torch.empty(meta, dtype=torch.float16, device=device))

    @property
    def lengths(self) -> torch.Tensor:
        if self._lengths is None:
            with _normal_tensors():
                self._lengths = torch.zeros(self.batch, dtype=torch.int32, device=self.device)
        return self._lengths

    @property
    def device(self) -> torch.device:
        return self.k_codes.device

    @property
    def nbytes(self) -> int:
        return sum(t.numel() * t.element_size() for t in self.buffers)

    def reserve(self, capacity: int) -> None:
        """Room for ``capacity`` tokens a sequence: larger buffers with the same rows,
        those beyond ``max_length`` among them (written at explicit places)."""
        cap = -(-int(capacity) // CAPACITY_STEP) * CAPACITY_STEP
        if cap <= self.capacity:
            return
        new = []
        with _normal_tensors():
            for t in self.buffers:
                n = t.new_empty((*t.shape[:2], cap, *t.shape[3:]))
                n[:, :, :self.capacity] = t
                new.append(n)
        self._take(new)

    def select(self, rows: torch.Tensor) -> None:
        """Keep the sequences ``rows``: an index along the batch (repeats and negative
        ones allowed), or a truth value for each."""
        with _normal_tensors():
            rows = rows.to(self.device)
            rows = rows.nonzero().flatten() if rows.dtype is torch.bool else rows.to(torch.int64)
            rows = torch.where(rows < 0, rows + self.batch, rows)
            lengths = self.lengths.index_select(0, rows)
            self._take([t.index_select(0, rows) for t in self.buffers])
        self._lengths = lengths

    def crop(self, length: int) -> None:
        """Forget the tokens from ``length`` on."""
        length = max(0, int(length))
        self.lengths.clamp_(max=length)
        self.max_length = min(self.max_length, length)

    def _take(self, buffers) -> None:
        lengths, n = self._lengths, self.max_length
        self.__init__(*buffers)
        self._lengths, self.max_length = lengths, n

    @property
    def buffers(self):
        return self.k_codes, self.k_meta, self.v_codes, self.v_meta

    def reset(self) -> None:
        """Forget every token (the buffers stay)."""
        self.lengths.zero_()
        self.max_length = 0

    def append(self, keys: torch.Tensor, values: torch.Tensor, *, index: torch.Tensor | None = None,
               counts: torch.Tensor | None = None) -> None:
        """Quantise rows (B, Hkv, T, 128) behind each sequence's tokens.  ``index``
        (B, n) picks source rows instead; ``counts`` (B,) writes only the first
        counts[b] of them.  A source row out of range is skipped and reported by
        ``ops.status``; the sequence then ends before it.  ``max_length`` grows by n
        whatever ``counts`` says (it is not read back); ``crop`` lowers it."""
        n = keys.shape[2] if index is None else index.shape[1]
        if n == 0:
            return
        if self.max_length + n > self.capacity:
            raise ValueError(f"{self.max_length} + {n} tokens exceed the cache's capacity {self.capacity}")
        ops.kv_quantize(keys, values, self, self.lengths, index=index, counts=counts)
        added = n if counts is None else counts.clamp(0, n)
        if index is not None:
            there = ((index >= 0) & (index < keys.shape[2])).cumprod(1).sum(1, dtype=torch.int32)
            added = there if counts is None else torch.minimum(there, added)
        self.lengths.add_(added)
        self.max_length += n

    def read(self, *, index: torch.Tensor | None = None, dtype: torch.dtype = torch.bfloat16):
        """(keys, values) of the picked slots, or of the first ``max_length``."""
        if index is None:
            return ops.kv_dequantize(self, count=self.max_length, dtype=dtype)
        return ops.kv_dequantize(self, index=index, dtype=dtype)

    def attend(self, q: torch.Tensor, **kwargs):
        """``ops.attention_quantized`` over this cache's tokens."""
        return ops.attention_quantized(q, self, self.lengths, max_length=self.max_length, **kwargs)
