"""Attention over the quantised cache, every value and LSE against a plain f64
computation, at sizes that reach each kernel, tile and join; the plan of each call is
asked for, so that a change of the plan cannot leave one untested.

Tolerances, of the kernel that the plan names.  The few-row kernels' scores are off by
2^-20 scale sum|q||k| (f32 sums of exact products).  On tcgen05 K, V and P are rounded to f16 (relative 2^-11 at most, 0.41 of it in the
mean square).  A score is then off by 2^-11 scale sum|q||k| at most, which moves the
output by twice that times max|v| beside P's and V's 2^-10 max|v|, and the LSE by as much.
Each weight and value is off by an independent relative error, so the error's norm stands
to the output's as one term's to 1: with sqrt(sum q^2 k^2) scale below 2.5 for these
inputs it is sqrt(2.5^2 + 2) 0.41 2^-11 < 2^-10, and 2^-9 leaves a factor of two; the output's
rounding adds 2^-9 (bf16) or 2^-12 (f16).  The mean of the LSE's error stays below the
scores' mean square, 2.5 0.41 2^-11 < 2^-10."""

import itertools

import pytest
import torch

from test_gpu_kvcache import DT, _decode, _dev, _filled, _rows

pytestmark = pytest.mark.gpu


def _reference(q, cache, lengths, mask, causal, scale):
    """f64 (out (B, Lq, Hq, 128), lse (B, Hq, Lq), largest scale sum|q||k|, largest |v|) on q's device."""
    K, V = (x.to(q.device) for x in _decode(cache))
    B, Hq, Lq, _ = q.shape
    H = cache.n_kv_heads
    out = torch.zeros(B, Lq, Hq, 128, dtype=torch.float64, device=q.device)
    lse = torch.full((B, Hq, Lq), -float("inf"), dtype=torch.float64, device=q.device)
    bound = vmax = 0.0
    for b in range(B):
        n = int(lengths[b])
        see = torch.arange(n, device=q.device).expand(Lq, n)
        see = see <= torch.arange(n - Lq, n, device=q.device)[:, None] if causal else see >= 0
        if mask is not None:
            see = see & mask[b, :n].bool()
        some = see.any(1)
        if not some.any():
            continue
        # what no query sees may hold anything
        k, v = (torch.where(see.any(0)[:, None], x[b, :, :n], 0.0) for x in (K, V))
        k, v = (x.repeat_interleave(Hq // H, 0) for x in (k, v))
        qq = q[b].double()
        s = (qq @ k.transpose(1, 2) * scale).masked_fill(~see, -float("inf"))[:, some]
        lse[b][:, some] = torch.logsumexp(s, 2)
        out[b, some] = (torch.softmax(s, 2) @ v).transpose(0, 1)
        bound = max(bound, float((qq.abs() @ k.abs().transpose(1, 2)).max()) * scale)
        vmax = max(vmax, float(v.abs().max()))
    return out, lse, bound, vmax


def _check_plan(q, cache, lengths, plan, *, mask=None, causal=True, scale=128 ** -0.5, exact_keys=False):
    """``plan``: what ops.attention_quantized_plan has to say of the call."""
    from core_b200 import ops
    got = ops.attention_quantized_plan(cache, q.shape[1], q.shape[2], max(lengths), exact_keys=exact_keys)
    assert {k: got[k] > 1 if k == "parts" else got[k] for k in plan} == plan, got
    at = torch.tensor(lengths, dtype=torch.int32, device=q.device)
    out, lse = ops.attention_quantized(q, cache, at, max_length=max(lengths), key_mask=mask, causal=causal,
                                       softmax_scale=scale, exact_keys=exact_keys)
    ops.status(q.device)
    want, wl, bound, vmax = _reference(q, cache, lengths, mask, causal, scale)
    ds = bound * (2.0 ** -20 + (2.0 ** -11 if got["f16_keys"] else 0.0))
    got, gl = out.double(), lse.double()
    bf16 = q.dtype == torch.bfloat16
    empty = torch.isinf(wl)
    assert torch.equal(torch.isinf(gl), empty) and (got.transpose(1, 2)[empty] == 0).all()
    tol = (2.0 ** -10 + max(lengths) * 2.0 ** -25 + 2 * ds) * vmax + (2.0 ** -8 if bf16 else 2.0 ** -11) * want.abs()
    assert ((got - want).abs() <= tol).all(), float(((got - want).abs() - tol).max())
    assert (got - want).norm() <= (2.0 ** -9 + (2.0 ** -9 if bf16 else 2.0 ** -12)) * want.norm()
    err = (gl - wl)[~empty].abs()
    assert (err <= ds + 2e-5 + 1e-6 * wl[~empty].abs()).all() and err.mean() <= 2.0 ** -10
    return out, lse


MANY = dict(row_tile=256, f16_keys=True)
ONE, CTA, WARP = dict(parts=False), dict(parts=True, join_rows=False), dict(parts=True, join_rows=True)
FORMATS = list(itertools.product((4, 8), (32, 64, 128)))


@pytest.mark.parametrize("bits,group", FORMATS)
@pytest.mark.parametrize("batch,heads,groups,queries,length,plan", [
    (4, 8, 1, 381, 100, ONE),  # two row tiles, the last row in the middle of a warp
    (2, 8, 1, 439, 767, WARP),  # a partial second tile of rows
    (1, 4, 5, 133, 2900, CTA),  # 665 rows: a third pair of tiles with 25 of 32 lanes of a warp
])
def test_rows_that_end_inside_a_warp(bits, group, batch, heads, groups, queries, length, plan):
    dev = _dev()
    lengths = [max(length - 61 * b, 0) for b in range(batch)]
    c = _filled(200, batch, heads, -(-length // 128) * 128, bits, group, dev, lengths)
    q = _rows(202, (batch, heads * groups, queries, 128), DT["bf16"], 2.0).to(dev)
    _check_plan(q, c, lengths, dict(MANY, **plan))


@pytest.mark.parametrize("bits,group", FORMATS)
@pytest.mark.parametrize("batch,heads,groups,queries,length,plan", [
    (16, 8, 3, 17, 100, ONE), (1, 8, 11, 11, 3308, CTA), (8, 8, 1, 79, 767, WARP),  # one row tile
    (8, 8, 11, 17, 100, ONE), (1, 8, 6, 27, 3970, CTA), (4, 8, 3, 83, 767, WARP),  # two
])
def test_row_tiles_masks_and_lengths(bits, group, batch, heads, groups, queries, length, plan):
    """One and two row tiles, alone and cut into parts that either join takes: ragged and
    empty sequences, causal and not, and masks with NaN and infinities behind them."""
    from core_b200 import ops
    dev = _dev()
    lengths = [length if b % 3 == 0 else 0 if b % 5 == 4 else length * (b + 1) // (batch + 1) for b in range(batch)]
    cap = -(-length // 128) * 128
    c = _filled(210, batch, heads, cap, bits, group, dev, lengths)
    q = _rows(212, (batch, heads * groups, queries, 128), DT["f16"], 2.0).to(dev)
    plan = dict(MANY, **plan)
    _check_plan(q, c, lengths, plan)
    _check_plan(q.to(torch.bfloat16), c, lengths, plan, causal=False, scale=0.06)
    mask = torch.rand(batch, cap, generator=torch.Generator().manual_seed(213)) < 0.5
    mask[0, :length // 2] = False
    mask[batch // 2, :length // 3] = True
    if batch > 2:
        mask[2] = False
    k, v = _rows(214, (batch, heads, length, 128), DT["bf16"], 6.0), _rows(215, (batch, heads, length, 128), DT["bf16"])
    hidden = ~mask[:, None, :length, None].expand_as(k)
    k[hidden], v[hidden] = float("nan"), float("inf")
    v[:, 1:][hidden[:, 1:]] = float("nan")
    ops.kv_quantize(k.to(dev), v.to(dev), c, 0)
    _check_plan(q, c, [length] * batch, plan, mask=mask.to(dev))
    _check_plan(q, c, lengths, plan, mask=mask.to(dev), causal=False)


@pytest.mark.parametrize("bits,group", FORMATS)
@pytest.mark.parametrize("heads,groups,queries,length,plan", [
    (50, 4, 5, 2400, dict(row_tile=24, **CTA)), (50, 6, 4, 2400, dict(row_tile=24, **CTA)),
    (113, 4, 6, 2000, dict(row_tile=24, **WARP)), (1, 1, 1, 492, dict(row_tile=8, ctas_per_sm=3, **CTA)),
    (64, 1, 1, 3096, dict(row_tile=8, **CTA)), (64, 8, 1, 3096, dict(row_tile=8, **CTA)),
    (1, 4, 4, 3000, dict(row_tile=16, **CTA)),
])
def test_few_rows_tiles_and_joins(bits, group, heads, groups, queries, length, plan):
    """8, 16 and 24 rows a CTA whose parts are joined, in every format."""
    dev = _dev()
    c = _filled(220, 1, heads, -(-length // 128) * 128, bits, group, dev, [length])
    q = _rows(222, (1, heads * groups, queries, 128), DT["bf16"], 2.0).to(dev)
    plan = dict(plan, f16_keys=False)
    if (heads, bits) == (64, 4):
        plan["ctas_per_sm"] = 4
    _check_plan(q, c, [length], plan)
    mask = torch.rand(1, length, generator=torch.Generator().manual_seed(223)).to(dev) > 0.3
    _check_plan(q.half(), c, [length], plan, mask=mask)


@pytest.mark.parametrize("bits,group", [(4, 64), (8, 32)])
def test_exact_keys_rules_the_rounding_out(bits, group):
    """Sizes that go to tcgen05 by themselves: with exact_keys the scores, and so the LSE,
    are as exact as a few rows', parts and workspace included."""
    dev = _dev()
    for batch, heads, groups, queries, length in ((1, 4, 5, 133, 2900), (4, 8, 1, 381, 100)):
        lengths = [length - 13 * b for b in range(batch)]
        c = _filled(230, batch, heads, -(-length // 128) * 128, bits, group, dev, lengths)
        q = _rows(232, (batch, heads * groups, queries, 128), DT["f16"], 2.0).to(dev)
        _check_plan(q, c, lengths, MANY)
        for causal in (True, False):
            _check_plan(q, c, lengths, dict(f16_keys=False), causal=causal, exact_keys=True)


@pytest.mark.parametrize("bits", (4, 8))
@pytest.mark.parametrize("heads,queries,length", [(160, 48, 16384), (600, 1, 8192)], ids=["many", "few"])
def test_long_flat_tail_behind_a_large_score(bits, heads, queries, length):
    """One token whose weight is 2^25.6 times each of the others', with value 0 where
    theirs is 1: the output is the others' share.  Each weight is rounded at 2^-25 of f16's
    range, at 2^7 for the largest: off by 2^-32 of 2^-25.6, so by less than 2^-6 of itself."""
    from core_b200 import ops
    from core_b200.kvcache import QuantizedKV
    dev = _dev()
    c = QuantizedKV.empty(1, heads, length, bits=bits, group=128, device=dev)
    c.k_codes.zero_(), c.v_codes.zero_(), c.k_meta.zero_(), c.v_meta.zero_()
    c.k_meta[:, :, 0, :, 1] = 25.6 / 128
    c.v_meta[:, :, 1:, :, 1] = 1.0
    q = torch.ones(1, heads, queries, 128, dtype=torch.bfloat16, device=dev)
    scale = 0.6931471805599453
    out, lse = ops.attention_quantized(q, c, length, causal=False, softmax_scale=scale)
    s0 = torch.tensor(25.6 / 128).half().double() * 128 * scale
    share = (length - 1) * torch.exp(-s0) / (1 + (length - 1) * torch.exp(-s0))
    assert ((out.double() / share - 1).abs() <= 2.0 ** -6 + 2.0 ** -8).all(), float(out.max()) / float(share)
    assert ((lse.double().cpu() - s0 - torch.log1p((length - 1) * torch.exp(-s0))).abs() < 1e-4).all()


@pytest.mark.parametrize("heads,queries", [(160, 48), (2, 1)], ids=["many", "few"])
@pytest.mark.parametrize("power", (20, 23, 24, 25, 26))
def test_scores_whose_last_place_is_whole_numbers(power, heads, queries):
    """Scores of 2^power and a few units that rise along the sequence: P stays within f16
    although the maxima are rounded.  All values are 1, so the output is 1."""
    from core_b200 import ops
    from core_b200.kvcache import QuantizedKV
    dev = _dev()
    n = 4096
    c = QuantizedKV.empty(1, heads, n, bits=8, group=32, device=dev)
    c.k_codes.zero_(), c.v_codes.zero_(), c.k_meta.zero_(), c.v_meta.zero_()
    c.k_meta[:, :, :, 0, 1] = 256.0
    c.k_meta[:, :, :, 1, 1] = torch.linspace(0, 64, n, device=dev)
    c.v_meta[..., 1] = 1.0
    q = torch.zeros(1, heads, queries, 128, dtype=torch.float16, device=dev)
    q[..., 0], q[..., 32] = 2.0 ** (power - 8 - 8), 2.0 ** -8
    scale = 0.6931471805599453 * 2.0 ** 8
    out, lse = ops.attention_quantized(q, c, n, causal=False, softmax_scale=scale)
    assert (out == 1).all()
    assert ((lse / 0.6931471805599453 / 2.0 ** power - 1).abs() < 1e-4).all()
