"""A transformers cache whose layers hold their rows in 4 or 8 bits.

``quantized_cache(config)`` is a ``transformers.Cache`` for ``model(...,
past_key_values=cache)`` or ``model.generate``.  The prompt attends to its own
keys and values in full precision and is quantised on the way (as transformers'
``QuantizedCache`` does); later forwards quantise the new rows and attend to the
codes.  Under this package's attention (``attention.register()``, attention
implementation "core_b200") they are read as codes by
``ops.attention_quantized``; any other implementation is given the rows read back
in the model's dtype.  A press on the model reads a layer's rows back to score
them and stores the ones it keeps (``press.read_cache_layer`` /
``write_cache_layer``).
"""

from __future__ import annotations

import torch
from transformers.cache_utils import Cache, CacheLayerMixin

from . import attention, ops
from .kvcache import QuantizedKV


def _room(tokens: int) -> int:
    """Slots for a layer of ``tokens``: an eighth more, and 256 at least, so that the
    buffers stay close to their rows and decoding copies them rarely."""
    return tokens + max(256, tokens // 8)


class QuantizedCacheLayer(CacheLayerMixin):
    """One layer: a ``QuantizedKV`` that grows as tokens arrive."""

    is_sliding = False

    def __init__(self, *, bits: int = 4, group: int = 64, by_codes: bool = False):
        super().__init__()
        if bits not in (4, 8) or group not in (32, 64, 128):
            raise ValueError("bits must be 4 or 8 and group 32, 64 or 128")
        self.bits, self.group, self.by_codes = bits, group, by_codes
        self.kv: QuantizedKV | None = None

    def lazy_initialization(self, key_states: torch.Tensor, value_states: torch.Tensor) -> None:
        if key_states.shape[-1] != ops.HEAD_DIM or value_states.shape != key_states.shape:
            raise ValueError(f"the quantised cache takes keys and values of head_dim {ops.HEAD_DIM}")
        self.dtype, self.device = key_states.dtype, key_states.device
        self.kv = self._empty(key_states)
        self.is_initialized = True

    def _empty(self, rows: torch.Tensor) -> QuantizedKV:
        B, H, n = rows.shape[:3]
        return QuantizedKV.empty(B, H, _room(n), bits=self.bits, group=self.group, device=rows.device)

    def update(self, key_states: torch.Tensor, value_states: torch.Tensor, *args, **kwargs):
        if self.kv is None:
            self.lazy_initialization(key_states, value_states)
        kv, n = self.kv, key_states.shape[2]
        first = kv.max_length == 0
        if kv.max_length + n > kv.capacity:
            kv.reserve(_room(kv.max_length + n))
        kv.append(key_states, value_states)
        if first:
            return key_states, value_states
        if self.by_codes:
            return self._stand_in(key_states), self._stand_in(value_states)
        return self.read_rows()

    def _stand_in(self, rows: torch.Tensor) -> torch.Tensor:
        """A tensor of the cached rows' shape without their data, which tells
        ``attention.attention_forward`` where the codes are.  It reads as NaN: an
        attention that does not know it cannot give a plausible result."""
        kv = self.kv
        t = rows.new_full((1,), float("nan")).expand(kv.batch, kv.n_kv_heads, kv.max_length, ops.HEAD_DIM)
        setattr(t, attention.CODES, self)
        return t

    def read_rows(self):
        """(keys, values) read back in the model's dtype."""
        return self.kv.read(dtype=self.dtype)

    def write_rows(self, keys: torch.Tensor, values: torch.Tensor) -> None:
        """Replace every row (a press stores the ones it kept), in buffers of their size."""
        if self.kv is None:
            self.lazy_initialization(keys, values)
        kv = self._empty(keys)
        kv.append(keys, values)
        self.kv = kv

    def get_seq_length(self) -> int:
        return 0 if self.kv is None else self.kv.max_length

    def get_mask_sizes(self, query_length: int) -> tuple[int, int]:
        return self.get_seq_length() + query_length, 0

    def get_max_cache_shape(self) -> int:
        return -1

    def reset(self) -> None:
        if self.kv is not None:
            self.kv.reset()

    def crop(self, max_length: int) -> None:
        if self.kv is not None:
            self.kv.crop(max_length if max_length >= 0 else self.kv.max_length + max_length)

    def reorder_cache(self, beam_idx: torch.LongTensor) -> None:
        self.batch_select_indices(beam_idx)

    def batch_select_indices(self, indices: torch.Tensor) -> None:
        if self.kv is not None:
            self.kv.select(indices)

    def batch_repeat_interleave(self, repeats: int) -> None:
        if self.kv is not None:
            self.kv.select(torch.arange(self.kv.batch).repeat_interleave(repeats))


def quantized_cache(config, *, bits: int = 4, group: int = 64) -> Cache:
    """A cache for a model of ``config`` (a transformers config)."""
    config = config.get_text_config(decoder=True)
    by_codes = getattr(config, "_attn_implementation", None) == attention.IMPLEMENTATION
    return Cache(layers=[QuantizedCacheLayer(bits=bits, group=group, by_codes=by_codes)
                         for _ in range(config.num_hidden_layers)])
