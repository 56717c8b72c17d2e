"""Host-side checks of the quantised KV cache: what its entry points refuse
without touching a GPU."""

import ctypes

from core_b200 import _lib

def test_quantised_cache_arguments_rejected_on_host():
    """The quantised-cache entry points refuse bad shapes before any CUDA call."""
    lib = _lib.load()
    s = ctypes.cast((ctypes.c_int64 * 3)(1 << 20, 1 << 14, 128), ctypes.c_void_p)
    p, bad = ctypes.c_void_p(256), ctypes.c_void_p(264)

    def cache(k=256, bits=4, group=64, cap=128, heads=2):
        return ctypes.byref(_lib.CoreKvq(k, 256, 256, 256, 1, heads, cap, bits, group))

    def write(c, k=p, n=4, start=0, dtype=_lib.CORE_DTYPE_BF16):
        return lib.core_kvq_quantize(c, dtype, k, s, p, s, 4, n, None, None, start, None, None)

    assert write(cache(k=None)) == -1 and write(cache(bits=3)) == -2 and write(cache(group=16)) == -2
    assert write(cache(cap=100)) == -1 and write(cache(k=264)) == -1 and write(cache(), k=bad) == -1
    assert write(cache(), n=5) == -1 and write(cache(), n=0) == -1 and write(cache(), start=125) == -1
    assert lib.core_kvq_dequantize(cache(), 1, 4, None, None, 126, p, p, None) == -1
    assert lib.core_kvq_dequantize(cache(), 1, 4, None, None, 0, p, bad, None) == -1

    def attend(c, hq=4, lq=1, n=64, dtype=_lib.CORE_DTYPE_BF16, q=p, scale=0.1, mask=None, ms=0):
        return lib.core_kvq_attention(c, dtype, hq, lq, q, s, None, n, mask, ms, 1, scale, p, p, None, 0, None)

    assert attend(cache(), hq=3) == -1 and attend(cache(), lq=0) == -1 and attend(cache(), n=129) == -1
    assert attend(cache(), dtype=_lib.CORE_DTYPE_F32) == -2 and attend(cache(), q=bad) == -1
    assert attend(cache(), scale=-1.0) == -1 and attend(cache(), mask=p, ms=63) == -1
    assert "key_mask" in _lib.last_error()
    # one KV head's long sequence is cut into parts: the workspace is missing
    assert attend(cache(cap=4096, heads=1), hq=1, n=4096) == -6


def test_row_counts_whose_last_block_passes_31_bits_rejected_on_host():
    lib = _lib.load()
    s = ctypes.cast((ctypes.c_int64 * 3)(1 << 20, 1 << 14, 128), ctypes.c_void_p)
    p, n = ctypes.c_void_p(256), 2 ** 31 - 10
    cache = ctypes.byref(_lib.CoreKvq(256, 256, 256, 256, 1, 1, 128, 4, 64))
    assert lib.core_kvq_quantize(cache, _lib.CORE_DTYPE_BF16, p, s, p, s, 4, n, p, p, 0, None, None) == -1
    assert lib.core_kvq_dequantize(cache, _lib.CORE_DTYPE_BF16, n, p, None, 0, p, p, None) == -1


def test_operators_run_with_the_cache_device_current(monkeypatch):
    """A cache on another device than the current one: the call runs with its
    device current (torch's switch is a stand-in; each call ends in a refusal
    that comes after it)."""
    import contextlib
    import types

    import pytest
    import torch

    from core_b200 import ops
    now, seen = [0], []

    @contextlib.contextmanager
    def switch(index):
        before, now[0] = now[0], index
        seen.append(index)
        try:
            yield
        finally:
            now[0] = before

    monkeypatch.setattr(torch._C, "_cuda_getDevice", lambda: now[0], raising=False)
    monkeypatch.setattr(torch.cuda, "device", switch)
    for index in (0, 1):
        cache = types.SimpleNamespace(index=index)
        rows = types.SimpleNamespace(get_device=lambda: index, dtype=torch.float64)
        with pytest.raises(TypeError, match="kv_quantize takes"):
            ops.kv_quantize(rows, rows, cache, 0)
        with pytest.raises(TypeError, match="kv_dequantize gives"):
            ops.kv_dequantize(cache, count=1, dtype=torch.float64)
        with pytest.raises(TypeError, match="attention_quantized takes"):
            ops.attention_quantized(rows, cache, 4)
    assert now == [0] and seen == [1, 1, 1]


def test_attention_plan_on_host():
    """The plan can be asked for without a GPU: few rows keep the keys exact, many long rows go to tcgen05,
    bad sizes are refused."""
    import types

    import pytest

    from core_b200 import ops

    def plan(hq, nq, n, heads=8, cap=1 << 20, bits=4, **kw):
        kvq = _lib.CoreKvq(256, 256, 256, 256, 1, heads, cap, bits, 64)
        return ops.attention_quantized_plan(types.SimpleNamespace(handle=ctypes.byref(kvq)), hq, nq, n, **kw)

    for nq in (1, 2, 3, 4, 8):
        p = plan(32, nq, 131072)
        assert not p["f16_keys"] and p["row_tile"] == min(8 * -(-4 * nq // 8), 24 if p["row_tile"] == 24 else 16)
    assert plan(8, 1, 131072, heads=1)["parts"] > 1  # the host counts one SM
    assert plan(8, 1, 0)["parts"] == 1
    p = plan(32, 2048, 16384)
    assert p["f16_keys"] and p["row_tile"] == 256
    p = plan(32, 2048, 16384, exact_keys=True)
    assert not p["f16_keys"] and p["row_tile"] < 256
    one = plan(8, 1, 131072, heads=1)
    assert one["workspace_bytes"] >= 8 * one["parts"] * 129 * 4
    for bad in (lambda: plan(12, 1, 5), lambda: plan(8, 0, 5), lambda: plan(8, 1, -1), lambda: plan(8, 1, 129, cap=128),
                lambda: plan(8, 1, 5, bits=3)):
        with pytest.raises(RuntimeError):
            bad()
    assert _lib.load().core_kvq_attention_plan(ctypes.byref(_lib.CoreKvq(256, 256, 256, 256, 1, 8, 128, 4, 64)),
                                               8, 1, 5, 0, None) == -1
