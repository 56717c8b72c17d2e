"""Torch-facing wrappers of the C ABI (one function per entry point).

Each wrapper validates shapes/dtypes/devices, allocates outputs and the
workspace with torch on the tensors' device, and calls the CUDA library on
the current torch stream.  There is no CPU path: inputs must be CUDA tensors.
"""

from __future__ import annotations

import ctypes
import math

import torch

from . import _lib
from ._lib import CoreDims, check

HEAD_DIM = 128


def _ptr(t: torch.Tensor | None):
    return ctypes.c_void_p(0 if t is None else t.data_ptr())


def _stream(device: torch.device):
    return ctypes.c_void_p(torch.cuda.current_stream(device).cuda_stream)


def _require_cuda(*ts):
    for t in ts:
        if t is not None and not t.is_cuda:
            raise ValueError("core_b200 operates on CUDA tensors only (no CPU path)")


_DTYPES = {torch.bfloat16: _lib.CORE_DTYPE_BF16, torch.float32: _lib.CORE_DTYPE_F32}


def _dtype_code(dtype: torch.dtype) -> int:
    """bf16 caches run on the tensor cores with the reference's bf16 roundings;
    f32 caches (the reference's fp32 path) on CUDA cores in f32."""
    if dtype not in _DTYPES:
        raise TypeError(f"core_b200 takes bfloat16 or float32 caches; got {dtype}")
    return _DTYPES[dtype]


_READOUT_DTYPES = {torch.bfloat16: _lib.CORE_DTYPE_BF16, torch.float16: _lib.CORE_DTYPE_F16,
                   torch.float32: _lib.CORE_DTYPE_F32}


def gate_value(gate_override) -> float:
    """The C-ABI gate argument: NaN selects the learned gate, a finite value
    is the constant gate (negative values included, as in the reference)."""
    if gate_override is None:
        return float("nan")
    g = float(gate_override)
    if not math.isfinite(g):
        raise ValueError(f"memory_gate_override must be finite, got {gate_override!r}")
    return g


def _dims(keys: torch.Tensor, n_q_heads: int, n_queries: int) -> CoreDims:
    b, hkv, L, d = keys.shape
    return CoreDims(b, n_q_heads, hkv, d, n_queries, L, _dtype_code(keys.dtype))


def _workspace(nbytes: int, device) -> torch.Tensor:
    return torch.empty(max(int(nbytes), 256), dtype=torch.uint8, device=device)


def status(device=None) -> None:
    """Raise if a kernel recorded a device-side error (synchronises the stream)."""
    device = device or torch.device("cuda", torch.cuda.current_device())
    check(_lib.load().core_check_device_status(_stream(device)))


class sm_budget:
    """Context manager (and plain call) capping the SMs the persistent grids
    plan for, process-wide; ``sm_budget(0)`` restores all SMs."""

    def __init__(self, n_sms: int):
        self.n = int(n_sms)
        check(_lib.load().core_set_sm_budget(self.n))

    def __enter__(self):
        return self

    def __exit__(self, *exc):
        check(_lib.load().core_set_sm_budget(0))


# ---------------------------------------------------------------------------
def qk_features(q: torch.Tensor, k: torch.Tensor, *, topk_qk: int = 4,
                n_recent_queries: int = 16, lse: torch.Tensor | None = None,
                features: torch.Tensor | None = None):
    """f1..f6 of every cached key (``strict_causal_qk_features``).

    q: (B, Hq, nq, 128), k: (B, Hkv, L, 128), both bf16 (tensor-core path,
    logits rounded to bf16 like the reference's bf16 matmul) or both f32
    (CUDA-core path, unrounded f32 logits).  Returns
    (features (B, L, 6) or the given (B, L, F>=6) buffer, lse (B, Hq, nq)).
    """
    _require_cuda(q, k, lse)
    q = q.contiguous()
    k = k.contiguous()
    B, Hq, nq, d = q.shape
    dims = _dims(k, Hq, nq)
    if q.dtype != k.dtype or d != HEAD_DIM:
        raise TypeError("q must have the cache dtype and head_dim 128")
    lib = _lib.load()
    if features is None:
        features = torch.empty(B, k.shape[2], 6, dtype=torch.float32, device=k.device)
    lse_out = torch.empty(B, Hq, nq, dtype=torch.float32, device=k.device)
    ws = _workspace(lib.core_qk_features_workspace_bytes(ctypes.byref(dims)), k.device)
    lse_in = None if lse is None else lse.to(torch.float32).contiguous()
    check(lib.core_qk_features(ctypes.byref(dims), _ptr(q), _ptr(k), topk_qk, n_recent_queries,
                               _ptr(lse_in), _ptr(lse_out), _ptr(features), features.shape[-1],
                               _ptr(ws), ws.numel(), _stream(k.device)))
    return features, lse_out


_ATTN_DTYPES = {torch.bfloat16: _lib.CORE_DTYPE_BF16, torch.float16: _lib.CORE_DTYPE_F16}


def attention_prefill(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, *,
                      softmax_scale: float | None = None, out: torch.Tensor | None = None):
    """Causal attention with the row LSE (``flash_attn_func(..., causal=True,
    return_attn_probs=True)`` as ``_core_flash_attention_forward`` calls it).

    q: (B, Hq, Lq, 128), k, v: (B, Hkv, Lk, 128), bf16 or f16, any strides with
    the head dim contiguous (the layout an HF attention module passes).
    Returns (out (B, Lq, Hq, 128) in q's dtype, lse (B, Hq, Lq) f32).
    """
    _require_cuda(q, k, v)
    if q.dtype not in _ATTN_DTYPES or k.dtype != q.dtype or v.dtype != q.dtype:
        raise TypeError("attention_prefill takes q, k, v of one dtype, bfloat16 or float16")
    B, Hq, Lq, d = q.shape
    _, Hkv, Lk, _ = k.shape
    if d != HEAD_DIM or k.shape[-1] != HEAD_DIM or v.shape != k.shape or k.shape[0] != B:
        raise ValueError("attention_prefill: head_dim 128 and matching batch / K, V shapes")

    def inner(t):
        # the head dim must be contiguous and every other stride 16-byte aligned
        if t.stride(-1) != 1 or any(s % 8 for s in t.stride()[:-1]) or t.data_ptr() % 16:
            t = t.contiguous()
        return t

    q, k, v = inner(q), inner(k), inner(v)
    dims = CoreDims(B, Hq, Hkv, HEAD_DIM, Lq, Lk, _ATTN_DTYPES[q.dtype])
    if out is None:
        out = torch.empty(B, Lq, Hq, HEAD_DIM, dtype=q.dtype, device=q.device)
    elif out.shape != (B, Lq, Hq, HEAD_DIM) or not out.is_contiguous() or out.dtype != q.dtype:
        raise ValueError("out must be a contiguous (B, Lq, Hq, 128) tensor of q's dtype")
    lse = torch.empty(B, Hq, Lq, dtype=torch.float32, device=q.device)
    scale = HEAD_DIM ** -0.5 if softmax_scale is None else float(softmax_scale)
    arrs = [(ctypes.c_int64 * 3)(t.stride(0), t.stride(1), t.stride(2)) for t in (q, k, v)]
    strides = [ctypes.cast(a, ctypes.c_void_p) for a in arrs]
    check(_lib.load().core_attention_prefill(
        ctypes.byref(dims), _ptr(q), strides[0], _ptr(k), strides[1], _ptr(v), strides[2],
        _ptr(out), _ptr(lse), scale, _stream(q.device)))
    return out, lse


# ---------------------------------------------------------------------------
# Quantised KV cache (core_b200.kvcache.QuantizedKV)
# ---------------------------------------------------------------------------

_KVQ_DTYPES = _READOUT_DTYPES
_I64X3 = ctypes.c_int64 * 3
_KVQ_SCALE = HEAD_DIM ** -0.5
_KVQ_EXACT_KEYS = 0x100  # CORE_KVQ_EXACT_KEYS

# One token is written, read or attended to in a few microseconds: these wrappers
# check in as few calls as they can.


# The C entries launch on the current device: for a cache on another one a wrapper
# calls itself again with that one current.


def _raw_stream(index: int) -> int:
    return torch._C._cuda_getCurrentRawStream(index)


def _wrong_device(t: torch.Tensor, name: str):
    if not t.is_cuda:
        return ValueError("core_b200 operates on CUDA tensors only (no CPU path)")
    return ValueError(f"{name} must be on the cache's device")


def _aligned_rows(t: torch.Tensor):
    """(t, its outer strides) where t's last dim is contiguous and its base and
    other strides are 16-byte aligned, else those of a contiguous copy."""
    s0, s1, s2, s3 = t.stride()
    if s3 != 1 or t.data_ptr() % 16 or (s0 | s1 | s2) * t.element_size() % 16:
        t = t.clone(memory_format=torch.contiguous_format)
        s0, s1, s2, _ = t.stride()
    return t, _I64X3(s0, s1, s2)


def _int32(value, name: str) -> int:
    """A host number that the C entry takes in 32 bits: ctypes would cut it off."""
    n = int(value)
    if not -2 ** 31 <= n < 2 ** 31:
        raise ValueError(f"{name} does not fit 32 bits: {n}")
    return n


def _per_sequence(value, cache, name: str):
    """(pointer to (B,) int32 on the device, scalar) of an int or a tensor."""
    if not isinstance(value, torch.Tensor):
        return None, _int32(value, name)
    if value.shape != (cache.batch,) or value.dtype is not torch.int32 or not value.is_contiguous():
        raise ValueError(f"{name} must be an int or a contiguous (B,) int32 tensor")
    if value.get_device() != cache.index:
        raise _wrong_device(value, name)
    return value.data_ptr(), 0


def _row_index(index, cache, name: str):
    if index.dim() != 2 or index.shape[0] != cache.batch:
        raise ValueError(f"{name} must be (B, n)")
    if index.get_device() != cache.index:
        raise _wrong_device(index, name)
    if index.dtype is torch.int64:  # what does not fit 32 bits stays out of range
        index = index.clamp(-1, 2 ** 31 - 1).to(torch.int32)
    elif index.dtype is not torch.int32:
        raise TypeError(f"{name} must be int32 or int64; got {index.dtype}")
    return index if index.is_contiguous() else index.contiguous()


def kv_quantize(keys: torch.Tensor, values: torch.Tensor, cache, start, *,
                index: torch.Tensor | None = None, counts: torch.Tensor | None = None) -> None:
    """Quantise rows of K and V into ``cache`` (a ``kvcache.QuantizedKV``).

    keys, values: (B, Hkv, L, 128), bf16, f16 or f32, any strides.  Row t of
    sequence b goes to slot ``start`` + t; ``start`` is an int or a (B,) int32
    device tensor.  ``index`` (B, n) picks the source rows (a selection's kept
    rows are compacted and quantised in one pass); ``counts`` (B,) int32 writes
    only the first counts[b] rows.  Slots or source rows out of range are
    skipped and reported by :func:`status`.
    """
    at_device = cache.index
    if keys.get_device() != at_device or values.get_device() != at_device:
        raise _wrong_device(values if keys.get_device() == at_device else keys, "keys and values")
    if torch._C._cuda_getDevice() != at_device:
        with torch.cuda.device(at_device):
            return kv_quantize(keys, values, cache, start, index=index, counts=counts)
    code = _KVQ_DTYPES.get(keys.dtype)
    if code is None or values.dtype is not keys.dtype:
        raise TypeError("kv_quantize takes keys and values of one dtype, bf16, f16 or f32")
    shape = keys.shape
    if (len(shape) != 4 or shape != values.shape or shape[0] != cache.batch
            or shape[1] != cache.n_kv_heads or shape[3] != HEAD_DIM):
        raise ValueError(f"keys and values must be ({cache.batch}, {cache.n_kv_heads}, L, {HEAD_DIM})")
    keys, ks = _aligned_rows(keys)
    values, vs = _aligned_rows(values)
    n = L = shape[2]
    if index is not None:
        index = _row_index(index, cache, "index")
        n = index.shape[1]
    if n == 0:
        return
    at, at0 = _per_sequence(start, cache, "start")
    cnt = None
    if counts is not None:
        if not isinstance(counts, torch.Tensor):
            raise ValueError("counts must be a contiguous (B,) int32 tensor")
        cnt = _per_sequence(counts, cache, "counts")[0]
    check(_lib.load().core_kvq_quantize(
        cache.handle, code, keys.data_ptr(), ks, values.data_ptr(), vs, L, n,
        None if index is None else index.data_ptr(), at, at0, cnt, _raw_stream(cache.index)))


def kv_dequantize(cache, *, start=0, count: int | None = None, index: torch.Tensor | None = None,
                  dtype: torch.dtype = torch.bfloat16):
    """(keys, values) (B, Hkv, n, 128) read back from ``cache``: ``count`` slots
    from ``start`` (an int or a (B,) int32 device tensor), or the slots ``index``
    (B, n).  Each value is n s + z rounded once to ``dtype`` (bf16, f16, f32)."""
    if torch._C._cuda_getDevice() != cache.index:
        with torch.cuda.device(cache.index):
            return kv_dequantize(cache, start=start, count=count, index=index, dtype=dtype)
    code = _KVQ_DTYPES.get(dtype)
    if code is None:
        raise TypeError(f"kv_dequantize gives bf16, f16 or f32; got {dtype}")
    at, at0, idx = None, 0, None
    if index is not None:
        index = _row_index(index, cache, "index")
        n, idx = index.shape[1], index.data_ptr()
        if isinstance(start, torch.Tensor) or start != 0 or count not in (None, n):
            raise ValueError("kv_dequantize reads the slots of index: no start, and no other count")
    else:
        if count is None or count < 0:
            raise ValueError("kv_dequantize needs index, or a count of slots")
        n = _int32(count, "count")
        at, at0 = _per_sequence(start, cache, "start")
    k = cache.k_meta.new_empty((cache.batch, cache.n_kv_heads, n, HEAD_DIM), dtype=dtype)
    v = torch.empty_like(k)
    if n:
        check(_lib.load().core_kvq_dequantize(cache.handle, code, n, idx, at, at0, k.data_ptr(),
                                              v.data_ptr(), _raw_stream(cache.index)))
    return k, v


def attention_quantized(q: torch.Tensor, cache, lengths, *, max_length: int | None = None,
                        key_mask: torch.Tensor | None = None, softmax_scale: float | None = None,
                        causal: bool = True, exact_keys: bool = False,
                        out: torch.Tensor | None = None):
    """Attention of q over a quantised cache, read as codes.

    q: (B, Hq, Lq, 128), bf16 or f16, any strides; Hq a multiple of the cache's
    KV heads.  ``lengths``: tokens of each sequence, an int or a (B,) int32 device
    tensor; ``max_length``: a host-side bound of them (default: the capacity).
    The queries are the sequence's last ones (``causal``; query i sees the tokens
    before lengths - Lq + i + 1) or see every token (``causal=False``).
    ``key_mask`` (B, n >= max_length) bool or uint8: False hides a token.
    Returns (out (B, Lq, Hq, 128) in q's dtype, lse (B, Hq, Lq) f32); a row that
    sees no token gives 0 and -inf.

    Statistics, sums and the LSE are f32, the weights and the cached values f16.  Up to
    32 query rows a KV head (Lq times the heads that share it) scores are exact to f32;
    with more, the faster kernel for the sizes may round the keys to f16 as well, which
    moves scores and LSE by up to 2^-11 softmax_scale sum |q||k|
    (:func:`attention_quantized_plan` tells); ``exact_keys`` rules that kernel out.
    No gradient is recorded.
    """
    if q.get_device() != cache.index:
        raise _wrong_device(q, "q")
    if torch._C._cuda_getDevice() != cache.index:
        with torch.cuda.device(cache.index):
            return attention_quantized(q, cache, lengths, max_length=max_length, key_mask=key_mask,
                                       softmax_scale=softmax_scale, causal=causal, exact_keys=exact_keys,
                                       out=out)
    dtype = q.dtype
    code = _ATTN_DTYPES.get(dtype)
    if code is None:
        raise TypeError(f"attention_quantized takes bf16 or f16 queries; got {dtype}")
    shape = q.shape
    if len(shape) != 4 or shape[0] != cache.batch or shape[3] != HEAD_DIM or shape[1] % cache.n_kv_heads:
        raise ValueError(f"q must be ({cache.batch}, Hq, Lq, {HEAD_DIM}) with Hq a multiple of "
                         f"{cache.n_kv_heads}")
    q, strides = _aligned_rows(q)
    B, Hq, Lq, _ = shape
    at, n = _per_sequence(lengths, cache, "lengths")
    if at is not None:
        n = cache.capacity if max_length is None else _int32(max_length, "max_length")
    mask, mask_stride = None, 0
    if key_mask is not None:
        if (key_mask.dim() != 2 or key_mask.shape[0] != B or key_mask.shape[1] < n
                or key_mask.dtype not in (torch.bool, torch.uint8)):
            raise ValueError("key_mask must be a (B, >= max_length) bool or uint8 tensor")
        if key_mask.get_device() != cache.index:
            raise _wrong_device(key_mask, "key_mask")
        if key_mask.stride(1) != 1 or (B > 1 and key_mask.stride(0) < key_mask.shape[1]):
            key_mask = key_mask.contiguous()
        mask, mask_stride = key_mask.data_ptr(), key_mask.stride(0) if B > 1 else key_mask.shape[1]
    if out is None:
        out = q.new_empty((B, Lq, Hq, HEAD_DIM))
    else:
        if out.shape != (B, Lq, Hq, HEAD_DIM) or not out.is_contiguous() or out.dtype is not dtype:
            raise ValueError("out must be a contiguous (B, Lq, Hq, 128) tensor of q's dtype")
        if out.get_device() != cache.index:
            raise _wrong_device(out, "out")
    lse = q.new_empty((B, Hq, Lq), dtype=torch.float32)
    if Lq == 0:
        return out, lse
    lib = _lib.load()
    mode = 1 if causal else 0
    if exact_keys:
        mode |= _KVQ_EXACT_KEYS
        need = attention_quantized_plan(cache, Hq, Lq, n, exact_keys=True)["workspace_bytes"]
    else:
        need = lib.core_kvq_attention_workspace_bytes(cache.handle, Hq, Lq, n)
    ws = q.new_empty(need, dtype=torch.uint8) if need else None
    rc = lib.core_kvq_attention(
        cache.handle, code, Hq, Lq, q.data_ptr(), strides, at, n, mask, mask_stride, mode,
        _KVQ_SCALE if softmax_scale is None else softmax_scale, out.data_ptr(), lse.data_ptr(),
        None if ws is None else ws.data_ptr(), need, _raw_stream(cache.index))
    if rc:
        check(rc)
    return out, lse


def attention_quantized_plan(cache, n_q_heads: int, n_queries: int, max_length: int, *,
                             exact_keys: bool = False) -> dict:
    """How :func:`attention_quantized` carries out a call of these sizes: ``row_tile``
    (query rows of a KV head a CTA takes: 8, 16, 24, or 256 on tcgen05), ``ctas_per_sm``,
    ``parts`` (CTAs a sequence is cut over), ``join_rows`` (parts joined by a warp a
    row), ``f16_keys`` (keys rounded to f16; otherwise scores are exact to f32) and
    ``workspace_bytes``."""
    plan = _lib.CoreKvqPlan()
    check(_lib.load().core_kvq_attention_plan(
        cache.handle, _int32(n_q_heads, "n_q_heads"), _int32(n_queries, "n_queries"),
        _int32(max_length, "max_length"), _KVQ_EXACT_KEYS if exact_keys else 0, ctypes.byref(plan)))
    return {name: bool(getattr(plan, name)) if name in ("join_rows", "f16_keys") else getattr(plan, name)
            for name, _ in plan._fields_}


def split_bf16(w: torch.Tensor, terms: int) -> torch.Tensor:
    """f32 -> (terms, *w.shape) bf16 whose sum reproduces w (hi, mid, lo)."""
    _require_cuda(w)
    w = w.to(torch.float32).contiguous()
    out = torch.empty((terms, *w.shape), dtype=torch.bfloat16, device=w.device)
    check(_lib.load().core_split_bf16(_ptr(w), w.numel(), terms, _ptr(out), _stream(w.device)))
    return out


def prepare_geometry(geometry: torch.Tensor, hadamard: torch.Tensor) -> torch.Tensor:
    """(3, 128, Hkv*d) bf16 terms of [W ; R W] for ``coverage_features``."""
    _require_cuda(geometry, hadamard)
    g = geometry.to(torch.float32).contiguous()
    r = hadamard.to(torch.float32).contiguous()
    if g.shape[0] != 64 or tuple(r.shape) != (64, 64):
        raise ValueError("geometry must be (64, Hkv*d) and hadamard (64, 64)")
    out = torch.empty(3, 128, g.shape[1], dtype=torch.bfloat16, device=g.device)
    check(_lib.load().core_prepare_geometry(_ptr(g), _ptr(r), g.shape[1], _ptr(out), _stream(g.device)))
    return out


def coverage_features(k: torch.Tensor, geometry_ext: torch.Tensor, prototypes: torch.Tensor, *,
                      shrinkage_rho: float = 0.1, features: torch.Tensor | None = None,
                      col0: int = 0):
    """o, d_proto, delta_proto, g (``compute_coverage_features``)."""
    _require_cuda(k, geometry_ext, prototypes)
    k = k.contiguous()
    B, hkv, L, d = k.shape
    dims = _dims(k, hkv, 0)
    if tuple(geometry_ext.shape) != (3, 128, hkv * d):
        raise ValueError("geometry_ext must be (3, 128, Hkv*d) (see prepare_geometry)")
    lib = _lib.load()
    if features is None:
        features = torch.empty(B, L, 4, dtype=torch.float32, device=k.device)
        col0 = 0
    ws = _workspace(lib.core_coverage_workspace_bytes(ctypes.byref(dims)), k.device)
    check(lib.core_coverage_features(
        ctypes.byref(dims), _ptr(k), _ptr(geometry_ext.contiguous()),
        _ptr(prototypes.float().contiguous()), float(shrinkage_rho), _ptr(features),
        features.shape[-1], col0, _ptr(ws), ws.numel(), _stream(k.device)))
    return features


def pack_mlp(mlp_params) -> torch.Tensor:
    """The prepared indexer MLP of ``core_prepare_indexer_mlp``: [w1 (128,14) | b1 |
    w2^T (in 128, out 128) | b2 | w3 (128) | b3] as f32 (nn.Linear weights are
    (out, in); layer 2 is stored transposed), followed on the device by layer 2's
    three-term bf16 tensor-core image."""
    w1, b1, w2, b2, w3, b3 = mlp_params
    flat = torch.cat([w1.reshape(-1), b1.reshape(-1), w2.t().reshape(-1), b2.reshape(-1),
                      w3.reshape(-1), b3.reshape(-1)]).to(torch.float32)
    _require_cuda(flat)
    lib = _lib.load()
    out = torch.zeros(lib.core_indexer_mlp_bytes() // 4, dtype=torch.float32, device=flat.device)
    out[:flat.numel()] = flat
    check(lib.core_prepare_indexer_mlp(_ptr(out), _stream(out.device)))
    return out


def indexer_scores(v: torch.Tensor, positions: torch.Tensor, features: torch.Tensor,
                   mlp_packed: torch.Tensor, *, original_length: int, is_prefill: bool,
                   n_sink: int = 4, special: torch.Tensor | None = None) -> torch.Tensor:
    """Auxiliary features into columns 10..13 of ``features`` (B, L, 14) and the
    indexer MLP scores (B, L)."""
    _require_cuda(v, positions, features, mlp_packed, special)
    v = v.contiguous()
    B, hkv, L, d = v.shape
    dims = _dims(v, hkv, 0)
    if features.shape != (B, L, 14) or not features.is_contiguous():
        raise ValueError("features must be a contiguous (B, L, 14) float32 tensor")
    pos = positions.to(torch.int64).reshape(B, L).contiguous()
    sp = None if special is None else special.to(torch.uint8).reshape(B, L).contiguous()
    scores = torch.empty(B, L, dtype=torch.float32, device=v.device)
    check(_lib.load().core_indexer_scores(
        ctypes.byref(dims), _ptr(v), _ptr(pos), _ptr(sp), int(original_length), int(is_prefill),
        int(n_sink), _ptr(features), _ptr(mlp_packed), _ptr(scores), _stream(v.device)))
    return scores


def topb_select(scores: torch.Tensor, n_kept: int, n_sink: int):
    """(keep (B, n_kept), evict (B, L - n_kept)) int32, both ascending."""
    _require_cuda(scores)
    scores = scores.to(torch.float32).contiguous()
    B, L = scores.shape
    keep = torch.empty(B, n_kept, dtype=torch.int32, device=scores.device)
    evict = torch.empty(B, max(L - n_kept, 1), dtype=torch.int32, device=scores.device)
    check(_lib.load().core_topb_select(_ptr(scores), B, L, int(n_kept), int(n_sink), _ptr(keep),
                                       _ptr(evict), _ptr(None), 0, _stream(scores.device)))
    return keep, evict[:, : L - n_kept]


def memory_write(k: torch.Tensor, v: torch.Tensor, scores_cal: torch.Tensor,
                 evict: torch.Tensor, theta_split: torch.Tensor, M: torch.Tensor,
                 b_state: torch.Tensor, Z: torch.Tensor, *, gamma: float, eta: float,
                 student_temp: float) -> None:
    """Update (M, b, Z) in place with the evicted tokens (``compress`` memory write).

    ``theta_split``: for bf16 caches the (2, d_mem, Hkv*d) bf16 terms of the
    group-folded Theta (``split_bf16(fold, 2)``); for f32 caches the folded
    (d_mem, Hkv*d) f32 Theta itself.
    """
    _require_cuda(k, v, scores_cal, evict, theta_split, M, b_state, Z)
    k = k.contiguous()
    v = v.contiguous()
    B, hkv, L, d = k.shape
    dims = _dims(k, hkv, 0)
    if v.dtype != k.dtype:
        raise TypeError("keys and values must have one dtype")
    n_evict = evict.shape[1]
    if k.dtype == torch.float32:
        if theta_split.dim() != 2 or theta_split.dtype != torch.float32:
            raise ValueError("f32 caches take the folded (d_mem, Hkv*d) f32 Theta")
        d_mem = theta_split.shape[0]
    else:
        if theta_split.dim() != 3 or theta_split.dtype != torch.bfloat16:
            raise ValueError("bf16 caches take the (2, d_mem, Hkv*d) bf16 terms of Theta")
        d_mem = theta_split.shape[1]
    for name, t, shape in (("M", M, (B, d_mem, hkv * d)), ("b", b_state, (B, d_mem)), ("Z", Z, (B,))):
        if tuple(t.shape) != shape or t.dtype != torch.float32 or not t.is_contiguous():
            raise ValueError(f"{name} must be a contiguous float32 tensor of shape {shape}")
    lib = _lib.load()
    ws = _workspace(lib.core_memory_write_workspace_bytes(ctypes.byref(dims), n_evict, d_mem), k.device)
    check(lib.core_memory_write(
        ctypes.byref(dims), _ptr(k), _ptr(v), _ptr(scores_cal.float().contiguous()),
        _ptr(evict.to(torch.int32).contiguous()), n_evict, _ptr(theta_split.contiguous()), d_mem,
        float(gamma), float(eta), float(student_temp), _ptr(M), _ptr(b_state), _ptr(Z), _ptr(ws),
        ws.numel(), _stream(k.device)))


def compact_kv(k: torch.Tensor, v: torch.Tensor, keep: torch.Tensor):
    """Gather the kept rows: (B, Hkv, n_kept, d) keys and values (bf16, fp16
    or f32 caches: the rows are copied bit for bit)."""
    _require_cuda(k, v, keep)
    k = k.contiguous()
    v = v.contiguous()
    B, hkv, L, d = k.shape
    n_kept = keep.shape[1]
    if k.dtype == torch.float16:
        dims = CoreDims(B, hkv, hkv, d, 0, L, _lib.CORE_DTYPE_F16)
    else:
        dims = _dims(k, hkv, 0)
    ok = torch.empty(B, hkv, n_kept, d, dtype=k.dtype, device=k.device)
    ov = torch.empty_like(ok)
    check(_lib.load().core_compact_kv(ctypes.byref(dims), _ptr(k), _ptr(v),
                                      _ptr(keep.to(torch.int32).contiguous()), n_kept, _ptr(ok),
                                      _ptr(ov), _stream(k.device)))
    return ok, ov


def memory_readout(q: torch.Tensor, theta: torch.Tensor, gate, M: torch.Tensor,
                   b_state: torch.Tensor, o_fold: torch.Tensor, attn_out: torch.Tensor,
                   *, n_kv_heads: int, gate_override: float | None = None,
                   workspace: torch.Tensor | None = None) -> torch.Tensor:
    """attn_out (B, q_len, hidden) += o_fold(g(q) m(q)); updated in place and returned.
    attn_out's dtype (bf16, fp16 or f32) selects the arithmetic; q is cast to it.
    ``gate_override``: None for the learned gate, else any finite constant gate.

    gate = (w1 (gh, Hq*d), b1 (gh), w2 (gh), b2 (1)) f32 tensors.  ``workspace``:
    an optional uint8 device buffer of at least ``core_memory_readout_workspace_bytes``
    (allocated here when absent or too small).
    """
    _require_cuda(q, theta, M, b_state, o_fold, attn_out)
    code = _READOUT_DTYPES.get(attn_out.dtype)
    if code is None:
        raise TypeError(f"memory_readout takes bf16, fp16 or f32 outputs; got {attn_out.dtype}")
    q = q.to(attn_out.dtype).contiguous()
    B, Hq, q_len, d = q.shape
    dims = CoreDims(B, Hq, n_kv_heads, d, q_len, max(q_len, 1), code)
    d_mem = theta.shape[0]
    hidden = o_fold.shape[0]
    w1, b1, w2, b2 = gate
    gh = w1.shape[0]
    if not attn_out.is_contiguous():
        raise ValueError("attn_out must be contiguous")
    lib = _lib.load()
    need = lib.core_memory_readout_workspace_bytes(ctypes.byref(dims), q_len, d_mem, gh)
    ws = workspace if workspace is not None and workspace.numel() >= need else _workspace(need, q.device)
    go = gate_value(gate_override)
    check(lib.core_memory_readout(
        ctypes.byref(dims), q_len, _ptr(q), _ptr(theta), _ptr(w1), _ptr(b1), _ptr(w2), _ptr(b2),
        d_mem, gh, go, _ptr(M), _ptr(b_state), _ptr(o_fold), hidden, _ptr(attn_out), _ptr(ws),
        ws.numel(), _stream(q.device)))
    return attn_out


_ROPE_DTYPES = _READOUT_DTYPES


def rope_queries(q_proj: torch.Tensor, n_q_heads: int, *, positions: torch.Tensor | None = None,
                 inv_freq: torch.Tensor | None = None, attention_scaling: float = 1.0,
                 cos: torch.Tensor | None = None, sin: torch.Tensor | None = None,
                 out: torch.Tensor | None = None) -> torch.Tensor:
    """Post-RoPE queries (B, Hq, T, d) from q_proj rows (B, T, Hq*d).

    Either ``positions`` (B or 1, T) int64 with the rotary ``inv_freq`` (d/2)
    and ``attention_scaling`` of a LlamaRotaryEmbedding, or the (cos, sin)
    position embeddings (B or 1, T, d) a model computed.  Roundings are those
    of transformers' apply_rotary_pos_emb in q_proj's dtype.
    """
    _require_cuda(q_proj, positions, inv_freq, cos, sin)
    if q_proj.dim() != 3 or q_proj.stride(-1) != 1:
        raise ValueError("q_proj must be (B, T, Hq*d) with unit inner stride")
    code = _ROPE_DTYPES.get(q_proj.dtype)
    if code is None:
        raise TypeError(f"rope_queries takes bf16, fp16 or f32; got {q_proj.dtype}")
    B, T, width = q_proj.shape
    if width % n_q_heads:
        raise ValueError("q_proj width must be a multiple of n_q_heads")
    d = width // n_q_heads
    if q_proj.stride(0) != T * q_proj.stride(1):
        q_proj = q_proj.contiguous()
    row_stride = q_proj.stride(1)
    if out is None:
        out = torch.empty(B, n_q_heads, T, d, dtype=q_proj.dtype, device=q_proj.device)
    pos = inv = c = s = None
    cb = 1
    if cos is not None:
        c = cos.to(q_proj.dtype).reshape(-1, T, d).contiguous()
        s = sin.to(q_proj.dtype).reshape(-1, T, d).contiguous()
        cb = c.shape[0]
        if cb not in (1, B) or s.shape != c.shape:
            raise ValueError("cos/sin must be (1 or B, T, d)")
    else:
        if positions is None or inv_freq is None:
            raise ValueError("rope_queries needs positions and inv_freq, or cos and sin")
        pos = positions.to(torch.int64).reshape(-1, T).expand(B, T).contiguous()
        inv = inv_freq.to(torch.float32).contiguous()
        if inv.numel() != d // 2:
            raise ValueError("inv_freq must hold head_dim/2 frequencies")
    check(_lib.load().core_rope_queries(B, T, n_q_heads, d, code, _ptr(q_proj), row_stride,
                                        _ptr(pos), _ptr(inv), float(attention_scaling), _ptr(c),
                                        _ptr(s), cb, _ptr(out), _stream(q_proj.device)))
    return out


# ---------------------------------------------------------------------------
# Head-sharded caches (one sequence, KV heads split across ranks).  Each call
# is one rank's part of a layer step; the cross-head sums between them are
# the caller's (core_b200.sharded runs them with NCCL).
# ---------------------------------------------------------------------------

def qk_summary_words(n_queries: int) -> int:
    return int(_lib.load().core_qk_summary_words(int(n_queries)))


def qk_head_summary(q: torch.Tensor, k: torch.Tensor, summary: torch.Tensor, *,
                    topk_qk: int = 4, n_recent_queries: int = 16) -> torch.Tensor:
    """Per-key summaries of this rank's heads into ``summary`` (rows >= L,
    core_qk_summary_words(nq)) int32; returns the rank's LSE (Hq_rank, nq)."""
    _require_cuda(q, k, summary)
    q = q.contiguous()
    k = k.contiguous()
    B, Hq, nq, d = q.shape
    if B != 1 or k.dtype != torch.bfloat16 or q.dtype != torch.bfloat16:
        raise ValueError("head-sharded summaries take one bf16 sequence")
    words = qk_summary_words(nq)
    if (summary.dim() != 2 or summary.shape[0] < k.shape[2] or summary.shape[1] != words
            or summary.dtype != torch.int32 or not summary.is_contiguous()):
        raise ValueError(f"summary must be a contiguous (>= L, {words}) int32 tensor")
    dims = _dims(k, Hq, nq)
    lib = _lib.load()
    lse = torch.empty(Hq, nq, dtype=torch.float32, device=k.device)
    ws = _workspace(lib.core_qk_features_workspace_bytes(ctypes.byref(dims)), k.device)
    check(lib.core_qk_head_summary(ctypes.byref(dims), _ptr(q), _ptr(k), int(topk_qk),
                                   int(n_recent_queries), _ptr(lse), _ptr(summary), _ptr(ws),
                                   ws.numel(), _stream(k.device)))
    return lse


def qk_merge_summaries(parts: torch.Tensor, features: torch.Tensor, *, key0: int, n_keys: int,
                       seq_len: int, n_queries: int, n_kv_heads: int, topk_qk: int = 4,
                       n_recent_queries: int = 16) -> None:
    """f1..f6 of keys key0 .. key0 + n_keys - 1 into features[:n_keys, :6] from
    the ranks' summaries ``parts`` (n_parts, rows, words)."""
    _require_cuda(parts, features)
    if parts.dim() != 3 or not parts.is_contiguous() or parts.dtype != torch.int32:
        raise ValueError("parts must be a contiguous (n_parts, rows, words) int32 tensor")
    if features.dim() != 2 or not features.is_contiguous() or features.shape[0] < n_keys:
        raise ValueError("features must be a contiguous (>= n_keys, F) float32 tensor")
    check(_lib.load().core_qk_merge_summaries(
        _ptr(parts), parts.shape[0], parts.shape[1], int(key0), int(n_keys), int(seq_len),
        int(n_queries), int(n_kv_heads), int(topk_qk), int(n_recent_queries), _ptr(features),
        features.shape[1], _stream(parts.device)))


def coverage_partial_projection(k: torch.Tensor, geometry_ext: torch.Tensor, y: torch.Tensor) -> None:
    """y[:L] = sum over this rank's heads of W_h k_h / |k_h| (raw, (L, 64) f32)."""
    _require_cuda(k, geometry_ext, y)
    k = k.contiguous()
    B, hkv, L, d = k.shape
    if B != 1:
        raise ValueError("head-sharded coverage takes one sequence")
    if tuple(geometry_ext.shape) != (3, 128, hkv * d):
        raise ValueError("geometry_ext must hold this rank's columns, (3, 128, Hkv_rank*d)")
    if y.dim() != 2 or y.shape[0] < L or y.shape[1] != 64 or not y.is_contiguous():
        raise ValueError("y must be a contiguous (>= L, 64) float32 tensor")
    dims = _dims(k, hkv, 0)
    lib = _lib.load()
    ws = _workspace(lib.core_coverage_workspace_bytes(ctypes.byref(dims)), k.device)
    check(lib.core_coverage_partial_projection(ctypes.byref(dims), _ptr(k),
                                               _ptr(geometry_ext.contiguous()), _ptr(y), _ptr(ws),
                                               ws.numel(), _stream(k.device)))


def coverage_range_totals(y: torch.Tensor, hadamard: torch.Tensor):
    """(z, zt, totals (192,) f64) for the summed projections y (n, 64) of a key range."""
    _require_cuda(y, hadamard)
    n = y.shape[0]
    y = y.contiguous()
    z = torch.empty(n, 64, dtype=torch.float32, device=y.device)
    zt = torch.empty_like(z)
    totals = torch.empty(192, dtype=torch.float64, device=y.device)
    lib = _lib.load()
    ws = _workspace(lib.core_coverage_range_workspace_bytes(n), y.device)
    check(lib.core_coverage_range_totals(_ptr(y), n, _ptr(hadamard.float().contiguous()), _ptr(z),
                                         _ptr(zt), _ptr(totals), _ptr(ws), ws.numel(),
                                         _stream(y.device)))
    return z, zt, totals


def coverage_range_assign(totals: torch.Tensor, seq_len: int, z: torch.Tensor, zt: torch.Tensor,
                          prototypes: torch.Tensor, features: torch.Tensor, *, col0: int = 6,
                          shrinkage_rho: float = 0.1):
    """Statistics of the summed totals, then d, delta and g of the range's keys
    into features[:, col0 + 1 .. col0 + 3]; returns (assign, hist (64,) int32)."""
    _require_cuda(totals, z, zt, prototypes, features)
    n = z.shape[0]
    assign = torch.empty(max(n, 1), dtype=torch.int32, device=z.device)
    hist = torch.empty(64, dtype=torch.int32, device=z.device)
    lib = _lib.load()
    ws = _workspace(lib.core_coverage_range_workspace_bytes(n), z.device)
    check(lib.core_coverage_range_assign(
        _ptr(totals.contiguous()), int(seq_len), float(shrinkage_rho), _ptr(z), _ptr(zt), n,
        _ptr(prototypes.float().contiguous()), _ptr(assign), _ptr(hist), _ptr(features),
        features.shape[-1], int(col0), _ptr(ws), ws.numel(), _stream(z.device)))
    return assign, hist


def coverage_range_occupancy(assign: torch.Tensor, hist: torch.Tensor, features: torch.Tensor,
                             n_keys: int, *, col0: int = 6) -> None:
    _require_cuda(assign, hist, features)
    check(_lib.load().core_coverage_range_occupancy(_ptr(assign), _ptr(hist.contiguous()),
                                                    int(n_keys), _ptr(features),
                                                    features.shape[-1], int(col0),
                                                    _stream(features.device)))


def value_head_sums(v: torch.Tensor, out: torch.Tensor) -> None:
    """out[h, :L] = the bf16 sum of bf16 squares of each value row of this rank's heads."""
    _require_cuda(v, out)
    v = v.contiguous()
    B, hkv, L, d = v.shape
    if out.dim() != 2 or out.shape[0] != hkv or out.shape[1] < L or not out.is_contiguous():
        raise ValueError("out must be a contiguous (Hkv_rank, >= L) float32 tensor")
    dims = _dims(v, hkv, 0)
    check(_lib.load().core_value_head_sums(ctypes.byref(dims), _ptr(v), _ptr(out), out.shape[1],
                                           _stream(v.device)))


def indexer_scores_from_sums(head_sums: torch.Tensor, key0: int, n_keys: int,
                             positions: torch.Tensor, features: torch.Tensor,
                             mlp_packed: torch.Tensor, *, original_length: int, is_prefill: bool,
                             n_sink: int = 4, special: torch.Tensor | None = None) -> torch.Tensor:
    """Scores of keys key0 .. key0 + n_keys - 1 from all heads' value sums
    head_sums (Hkv, stride); positions/special are the whole sequence's,
    features (n_keys, 14) the range's."""
    _require_cuda(head_sums, positions, features, mlp_packed, special)
    if not head_sums.is_contiguous() or head_sums.dim() != 2:
        raise ValueError("head_sums must be a contiguous (Hkv, stride) float32 tensor")
    if features.shape[0] < n_keys or features.shape[1] != 14 or not features.is_contiguous():
        raise ValueError("features must be a contiguous (>= n_keys, 14) float32 tensor")
    pos = positions.to(torch.int64).reshape(-1).contiguous()
    sp = None if special is None else special.to(torch.uint8).reshape(-1).contiguous()
    scores = torch.empty(max(n_keys, 1), dtype=torch.float32, device=features.device)
    hs_ptr = head_sums.data_ptr() + 4 * int(key0)
    pos_ptr = pos.data_ptr() + 8 * int(key0)
    sp_ptr = None if sp is None else sp.data_ptr() + int(key0)
    check(_lib.load().core_indexer_scores_from_sums(
        head_sums.shape[0], int(n_keys), ctypes.c_void_p(hs_ptr), head_sums.shape[1],
        ctypes.c_void_p(pos_ptr), ctypes.c_void_p(sp_ptr), int(original_length), int(is_prefill),
        int(n_sink), _ptr(features), _ptr(mlp_packed), _ptr(scores), _stream(features.device)))
    return scores[:n_keys]


def memory_write_gathered(k_ev: torch.Tensor, v_ev: torch.Tensor, scores_cal: torch.Tensor,
                          evict: torch.Tensor, theta_split: torch.Tensor, M: torch.Tensor,
                          b_state: torch.Tensor, Z: torch.Tensor, *, gamma: float, eta: float,
                          student_temp: float) -> None:
    """``memory_write`` with the evicted rows already gathered: k_ev, v_ev =
    (B, Hkv, n_evict, d) in evict order; scores_cal (B, L)."""
    _require_cuda(k_ev, v_ev, scores_cal, evict, theta_split, M, b_state, Z)
    k_ev = k_ev.contiguous()
    v_ev = v_ev.contiguous()
    B, hkv, n_evict, d = k_ev.shape
    L = scores_cal.shape[-1]
    if evict.shape != (B, n_evict):
        raise ValueError("evict must be (B, n_evict)")
    if k_ev.dtype != torch.bfloat16 or theta_split.dim() != 3:
        raise ValueError("gathered memory write takes bf16 rows and the (2, d_mem, Hkv*d) terms")
    d_mem = theta_split.shape[1]
    dims = CoreDims(B, hkv, hkv, d, 0, L, _lib.CORE_DTYPE_BF16)
    lib = _lib.load()
    ws = _workspace(lib.core_memory_write_workspace_bytes(ctypes.byref(dims), n_evict, d_mem),
                    k_ev.device)
    check(lib.core_memory_write_gathered(
        ctypes.byref(dims), _ptr(k_ev), _ptr(v_ev), _ptr(scores_cal.float().contiguous()),
        _ptr(evict.to(torch.int32).contiguous()), n_evict, _ptr(theta_split.contiguous()), d_mem,
        float(gamma), float(eta), float(student_temp), _ptr(M), _ptr(b_state), _ptr(Z), _ptr(ws),
        ws.numel(), _stream(k_ev.device)))
