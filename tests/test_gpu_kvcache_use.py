"""The quantised cache's objects in use: modes of autograd, growth, selection, what a
press keeps, and calls that used to mislead."""

import pytest
import torch

from test_gpu_kvcache import _dev, _rows

pytestmark = pytest.mark.gpu


def _cache(dev, B=2, H=2, cap=256, n=60, bits=4, group=32, seed=300):
    """(cache with n tokens, its keys, its values)."""
    from core_b200.kvcache import QuantizedKV
    c = QuantizedKV.empty(B, H, cap, bits=bits, group=group, device=dev)
    k = _rows(seed, (B, H, n, 128), torch.bfloat16, 6.0).to(dev)
    v = _rows(seed + 1, (B, H, n, 128), torch.bfloat16).to(dev)
    c.append(k, v)
    return c, k, v


def test_filled_under_inference_mode_used_under_no_grad():
    """A prompt under inference_mode, then decoding, selecting, growing, cropping and
    resetting outside of it, as transformers' own layers accept."""
    dev = _dev()
    with torch.inference_mode():
        c, k, v = _cache(dev)
        c.select(torch.tensor([1, 0], device=dev))
        c.reserve(300)
    want = c.read()
    with torch.no_grad():
        c.append(k[:, :, :1].clone(), v[:, :, :1].clone())
        assert c.lengths.tolist() == [61, 61]
        c.select(torch.tensor([1, 0]))
        c.reserve(500)
        assert torch.equal(c.read()[0][:, :, :60], want[0][[1, 0]])
        c.k_codes[:, :, -1].zero_()
        c.crop(30)
        assert c.lengths.tolist() == [30, 30]
    c.append(k[:, :, :1].clone(), v[:, :, :1].clone())
    assert c.lengths.tolist() == [31, 31]
    with torch.inference_mode():
        c.append(k[:, :, :1], v[:, :, :1])
    c.reset()
    assert c.lengths.tolist() == [0, 0]


def test_reserve_keeps_rows_written_at_explicit_places():
    """A cache around filled buffers, or one written with ops.kv_quantize, has rows that
    its lengths do not count."""
    from core_b200 import ops
    from core_b200.kvcache import QuantizedKV
    dev = _dev()
    c, k, v = _cache(dev, n=200)
    want = ops.kv_dequantize(c, count=200)
    w = QuantizedKV(*c.buffers)
    w.reserve(900)
    assert w.capacity == 1024
    got = ops.kv_dequantize(w, count=200)
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])


def test_append_counts_only_rows_that_were_written():
    """A source row out of range is skipped and reported: the sequence ends before it, so
    that no slot that was never written is attended to."""
    from core_b200 import ops
    from core_b200._lib import CoreError
    dev = _dev()
    c, k, v = _cache(dev, B=4, n=10)
    index = torch.tensor([[3, 4, 5, 6], [3, 60, 5, 6], [-1, 4, 5, 6], [0, 1, 2, 99]], device=dev)
    counts = torch.tensor([4, 4, 4, 2], dtype=torch.int32, device=dev)
    for idx in (index, index.int()):
        c.append(k, v, index=idx, counts=counts)
        with pytest.raises(CoreError, match="where=1402"):
            ops.status(dev)
        assert c.lengths.tolist() == [14, 11, 10, 12]
        c.crop(10)
    c.append(k, v, index=index[:1].expand(4, -1))
    assert c.lengths.tolist() == [14] * 4
    ops.status(dev)


def test_reading_picked_rows_takes_no_start_and_no_other_count():
    from core_b200 import ops
    dev = _dev()
    c, _, _ = _cache(dev)
    index = torch.tensor([[3, 4, 5], [6, 7, 8]], device=dev)
    want = ops.kv_dequantize(c, index=index)
    assert torch.equal(ops.kv_dequantize(c, index=index, count=3)[1], want[1])
    for bad in (dict(start=1), dict(start=torch.zeros(2, dtype=torch.int32, device=dev)), dict(count=2)):
        with pytest.raises(ValueError):
            ops.kv_dequantize(c, index=index, **bad)


def test_numbers_beyond_32_bits_are_refused():
    """They would wrap to other rows at the C boundary."""
    from core_b200 import ops
    dev = _dev()
    c, k, v = _cache(dev)
    before = [t.view(torch.uint8).clone() for t in c.buffers]
    q = _rows(310, (2, 4, 1, 128), torch.bfloat16).to(dev)
    at = torch.full((2,), 60, dtype=torch.int32, device=dev)
    for far in (2 ** 32, 2 ** 32 + 3, -2 ** 32, 2 ** 31):
        for call in (lambda: ops.kv_quantize(k, v, c, far), lambda: ops.kv_dequantize(c, start=far, count=3),
                     lambda: ops.attention_quantized(q, c, far),
                     lambda: ops.attention_quantized(q, c, at, max_length=far),
                     lambda: ops.attention_quantized_plan(c, 4, 1, far)):
            with pytest.raises((ValueError, RuntimeError)):
                call()
    assert all(torch.equal(a, b.view(torch.uint8)) for a, b in zip(before, c.buffers))


def test_select_takes_what_indexing_takes():
    """Truth values and indexes from the end, as transformers' layers do."""
    dev = _dev()
    c, k, v = _cache(dev, B=4)
    want = c.read()[0]
    c.select(torch.tensor([True, False, True, True]))
    assert c.batch == 3 and torch.equal(c.read()[0], want[[0, 2, 3]])
    c.select(torch.tensor([-1, 0], device=dev))
    assert c.lengths.tolist() == [60, 60] and torch.equal(c.read()[0], want[[3, 0]])


def test_attention_after_the_sm_budget_changed():
    """The workspace that was asked for serves the call of the same sizes, although
    another thread changed the process-wide SM budget in between."""
    import ctypes
    from core_b200 import _lib, ops
    dev = _dev()
    c, _, _ = _cache(dev, B=1, n=3000, cap=3072)
    q = _rows(311, (1, 8, 1, 128), torch.bfloat16).to(dev)
    want, _ = ops.attention_quantized(q, c, 3000)
    lib = _lib.load()
    with ops.sm_budget(8):
        need = lib.core_kvq_attention_workspace_bytes(c.handle, 8, 1, 3000)
    ws = torch.empty(need, dtype=torch.uint8, device=dev)
    out, lse = torch.empty(1, 1, 8, 128, dtype=torch.bfloat16, device=dev), torch.empty(1, 8, 1, device=dev)
    strides = (ctypes.c_int64 * 3)(*q.stride()[:3])
    rc = lib.core_kvq_attention(c.handle, _lib.CORE_DTYPE_BF16, 8, 1, q.data_ptr(), strides, None, 3000, None, 0, 1,
                                128 ** -0.5, out.data_ptr(), lse.data_ptr(), ws.data_ptr() if need else None, need,
                                torch.cuda.current_stream(dev).cuda_stream)
    assert rc == 0, _lib.last_error()
    assert (out.float() - want.float()).abs().max() <= 2.0 ** -7 * want.float().abs().max()
