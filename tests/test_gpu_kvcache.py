"""The quantised KV cache: kv_quantize, kv_dequantize and attention_quantized
against plain implementations on the CPU in f64 (and, for the codes, in the f32
steps that define them).

Tolerances.  Codes, scales, zeros and read-back values are defined by single
correctly rounded steps: they are compared bit for bit.  Attention: P and the
values n s + z are rounded to f16 (unit roundoff 2^-11; P below 2^-14 to 2^-25
absolute, against a sum of at least 2^-8 since the running maximum may lag by
2^8), which moves an output by at most (2^-10 + n 2^-17) max|v|; scores are f32 sums
of exact products, off by at most 2^-20 sum|q||k| scale (128 terms of 2^-24 and
the matrix units' truncation), which moves the output by twice that times
max|v|; the output rounding adds 2^-8 (bf16) or 2^-11 (f16) of it.  The LSE is
off by the scores' error plus 2e-5."""

import itertools

import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu

LIMIT = 61440.0
DT = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}


def _dev():
    if not torch.cuda.is_available():
        pytest.skip("no CUDA device")
    return torch.device("cuda", 0)


# ---- plain forms -----------------------------------------------------------
def _quantise(x, bits, group):
    """(codes (.., 128) int64, scale, zero (.., 128 / group) f16) on the CPU."""
    top = 2 ** bits - 1
    g = x.float().clamp(-LIMIT, LIMIT).unflatten(-1, (128 // group, group))
    lo, hi = g.amin(-1), g.amax(-1)  # NaN propagates
    z = lo.half()
    s = ((hi - lo) * np.float32(1.0 / top).item()).half()
    sf = s.float()
    inv = torch.where(sf > 0, 1.0 / sf, torch.zeros_like(sf))
    n = ((g - z.float()[..., None]) * inv[..., None]).round().clamp(0, top)
    return torch.nan_to_num(n).long().flatten(-2), s, z


def _word_and_bit(bits, keys, token):
    """For each of 128 channels: its word in the row and its first bit in the word."""
    word, bit = [], []
    for c in range(128):
        if bits == 4:
            e = c % 8
            bit.append([0, 16, 4, 20, 8, 24, 12, 28][e])
            w = 4 * (c % 32 // 8) + c // 32 if keys else (c // 8) ^ (8 if token & 2 else 0)
        else:
            e = c % 4
            bit.append([0, 16, 8, 24][e])
            if keys:
                b, t, h = c // 32, c % 32 // 8, c % 8 // 4
                w = (16 * (b // 2) + 4 * t + 2 * (b % 2) + h) ^ (16 if token & 1 else 0)
            else:
                w = (c // 4) ^ (8 * (token % 4))
        word.append(w)
    return np.array(word), np.array(bit)


def _unpack(codes, bits, keys):
    """Buffer (B, H, cap, bytes) -> codes (B, H, cap, 128)."""
    w = codes.cpu().numpy().view(np.uint32)
    out = np.empty(w.shape[:3] + (128,), np.int64)
    for par in range(4):
        word, bit = _word_and_bit(bits, keys, par)
        out[:, :, par::4] = (w[:, :, par::4][..., word] >> bit.astype(np.uint32)) & (2 ** bits - 1)
    return torch.from_numpy(out)


def _decode(cache):
    """f64 (keys, values) of every slot."""
    got = []
    for codes, meta, keys in ((cache.k_codes, cache.k_meta, True), (cache.v_codes, cache.v_meta, False)):
        n = _unpack(codes, cache.bits, keys).double()
        m = meta.cpu().double()
        g = m.shape[3]
        got.append((n.unflatten(-1, (g, 128 // g)) * m[..., 0:1] + m[..., 1:2]).flatten(-2))
    return got


def _rows(seed, shape, dtype, spread=1.0):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(shape, generator=g)
    x[..., 5] *= spread
    x[..., 77] *= spread
    return x.to(dtype)


def _poisoned(B, H, cap, bits, group, dev):
    """A cache whose untouched slots read as NaN."""
    from core_b200.kvcache import QuantizedKV
    c = QuantizedKV.empty(B, H, cap, bits=bits, group=group, device=dev)
    for t in (c.k_codes, c.k_meta, c.v_codes, c.v_meta):
        t.view(torch.uint8).fill_(0x7F)
    return c


# ---- writing and reading ----------------------------------------------------
@pytest.mark.parametrize("bits,group,dtype", list(itertools.product((4, 8), (32, 64, 128), ("bf16", "f16", "f32"))))
def test_quantize_and_read_back_bit_exact(bits, group, dtype):
    from core_b200 import ops
    dev = _dev()
    B, H, L, cap = 2, 3, 37, 128
    k, v = _rows(1, (B, H, L, 128), DT[dtype], 6.0), _rows(2, (B, H, L, 128), DT[dtype])
    start = torch.tensor([5, 88], dtype=torch.int32)
    c = _poisoned(B, H, cap, bits, group, dev)
    ops.kv_quantize(k.to(dev), v.to(dev), c, start.to(dev))
    for x, codes, meta, keys in ((k, c.k_codes, c.k_meta, True), (v, c.v_codes, c.v_meta, False)):
        n, s, z = _quantise(x, bits, group)
        got, m = _unpack(codes, bits, keys), meta.cpu()
        for b in range(B):
            a = int(start[b])
            assert torch.equal(got[b, :, a:a + L], n[b])
            assert torch.equal(m[b, :, a:a + L, :, 0], s[b]) and torch.equal(m[b, :, a:a + L, :, 1], z[b])
            # nothing else was touched
            rest = torch.ones(cap, dtype=torch.bool)
            rest[a:a + L] = False
            assert (codes[b].cpu()[:, rest] == 0x7F).all() and m[b][:, rest].isnan().all()
    for out in DT:
        rk, rv = ops.kv_dequantize(c, start=start.to(dev), count=L, dtype=DT[out])
        for x, r in ((k, rk), (v, rv)):
            n, s, z = _quantise(x, bits, group)
            want = (n.double().unflatten(-1, (128 // group, group)) * s.double()[..., None]
                    + z.double()[..., None]).flatten(-2).float().to(DT[out])
            assert torch.equal(r.cpu(), want)
    # error of the format: half a step, plus the f16 rounding of scale and zero
    err = (rk.cpu().double() - k.double()).abs().unflatten(-1, (128 // group, group)).amax(-1)
    n, s, z = _quantise(k, bits, group)
    assert (err <= s.double() * (0.5 + 2.0 ** bits * 2 ** -11) + z.double().abs() * 2 ** -10).all()
    ops.status(dev)


@pytest.mark.parametrize("bits", (4, 8))
def test_quantize_picked_rows_counts_and_strides(bits):
    """index picks source rows, counts stops a sequence early, and transposed,
    sliced and misaligned sources are taken as they are."""
    from core_b200 import ops
    dev = _dev()
    B, H, L, n = 3, 2, 300, 101
    base_k, base_v = _rows(3, (B, L, H, 128), torch.bfloat16, 6.0), _rows(4, (B, L, H, 128), torch.bfloat16)
    k, v = base_k.transpose(1, 2), base_v.transpose(1, 2)
    g = torch.Generator().manual_seed(5)
    idx = torch.stack([torch.randperm(L, generator=g)[:n].sort().values for _ in range(B)]).int()
    counts = torch.tensor([n, 0, 17], dtype=torch.int32)
    c = _poisoned(B, H, 128, bits, 64, dev)
    odd = torch.empty(B * L * H * 128 + 1, dtype=torch.bfloat16, device=dev)[1:].view(B, L, H, 128)
    odd.copy_(base_v)
    ops.kv_quantize(base_k.to(dev).transpose(1, 2), odd.transpose(1, 2), c, 3, index=idx.to(dev),
                    counts=counts.to(dev))
    ops.status(dev)
    for x, codes, meta, keys in ((k, c.k_codes, c.k_meta, True), (v, c.v_codes, c.v_meta, False)):
        got = _unpack(codes, bits, keys)
        for b in range(B):
            m = int(counts[b])
            want = _quantise(x[b][:, idx[b].long()], bits, 64)[0]
            assert torch.equal(got[b, :, 3:3 + m], want[:, :m])
            assert (codes[b].cpu()[:, 3 + m:] == 0x7F).all()


@pytest.mark.parametrize("bits,group", list(itertools.product((4, 8), (32, 64, 128))))
def test_quantize_extremes(bits, group):
    """Constant groups, zeros, subnormal ranges, values beyond the limit,
    infinities and NaN."""
    from core_b200 import ops
    dev = _dev()
    x = torch.randn(1, 1, 9, 128, generator=torch.Generator().manual_seed(6))
    x[0, 0, 0] = 3.25
    x[0, 0, 1] = 0.0
    x[0, 0, 2] *= 1e-7
    x[0, 0, 3, ::2] = 1e30
    x[0, 0, 4, 3] = float("inf")
    x[0, 0, 5, 100] = float("-inf")
    x[0, 0, 6, 64] = float("nan")
    x[0, 0, 7] = float("inf")
    x[0, 0, 8] = x[0, 0, 8] * 1e-3 - 60000.0
    c = _poisoned(1, 1, 128, bits, group, dev)
    ops.kv_quantize(x.to(dev), x.to(dev), c, 0)
    n, s, z = _quantise(x, bits, group)
    for codes, meta, keys in ((c.k_codes, c.k_meta, True), (c.v_codes, c.v_meta, False)):
        good = ~z[0, 0].isnan()
        got = _unpack(codes, bits, keys)[0, 0, :9].unflatten(-1, (128 // group, group))
        assert torch.equal(got[good], n[0, 0].unflatten(-1, (128 // group, group))[good])
        m = meta.cpu()[0, 0, :9]
        assert torch.equal(m[..., 0][good], s[0, 0][good]) and torch.equal(m[..., 1][good], z[0, 0][good])
        assert m[..., 1][~good].isnan().all()
    k, v = ops.kv_dequantize(c, count=9, dtype=torch.float16)
    bad = torch.zeros(128, dtype=torch.bool)
    bad[64 // group * group:64 // group * group + group] = True
    for r in (k.cpu()[0, 0], v.cpu()[0, 0]):
        assert r[6, bad].isnan().all() and torch.isfinite(r[6, ~bad]).all()
        assert torch.isfinite(r[[0, 1, 2, 3, 4, 5, 7, 8]]).all()
        assert (r[0] == 3.25).all() and (r[1] == 0).all() and (r[7] == LIMIT).all()


def test_read_picked_rows_in_any_order():
    from core_b200 import ops
    dev = _dev()
    c = _poisoned(2, 2, 256, 4, 32, dev)
    k, v = _rows(7, (2, 2, 256, 128), torch.float16), _rows(8, (2, 2, 256, 128), torch.float16)
    ops.kv_quantize(k.to(dev), v.to(dev), c, 0)
    idx = torch.tensor([[255, 0, 17, 17], [1, 200, 3, 2]])
    rk, rv = ops.kv_dequantize(c, index=idx.to(dev), dtype=torch.float32)
    dk, dv = _decode(c)
    for b in range(2):
        assert torch.equal(rk[b].cpu(), dk[b][:, idx[b]].float())
        assert torch.equal(rv[b].cpu(), dv[b][:, idx[b]].float())


def test_long_cache_offsets_pass_32_bits():
    """A cache whose buffers pass 2^32 bytes: the last head's last rows."""
    from core_b200 import ops
    from core_b200.kvcache import QuantizedKV
    dev = _dev()
    H, cap = 33, 1 << 20
    c = QuantizedKV.empty(1, H, cap, bits=8, group=128, device=dev)
    assert c.k_codes.numel() > 2 ** 32
    k, v = _rows(9, (1, H, 40, 128), torch.bfloat16, 4.0), _rows(10, (1, H, 40, 128), torch.bfloat16)
    c.k_codes[:, -1].zero_(), c.v_codes[:, -1].zero_(), c.k_meta[:, -1].zero_(), c.v_meta[:, -1].zero_()
    ops.kv_quantize(k.to(dev), v.to(dev), c, cap - 40)
    rk, _ = ops.kv_dequantize(c, start=cap - 40, count=40, dtype=torch.float32)
    n, s, z = _quantise(k, 8, 128)
    assert torch.equal(rk.cpu(), (n.double() * s.double() + z.double()).float())
    q = _rows(11, (1, H, 1, 128), torch.bfloat16)
    mask = torch.zeros(1, cap, dtype=torch.bool, device=dev)
    mask[:, cap - 40:] = True
    out, lse = ops.attention_quantized(q.to(dev), c, cap, key_mask=mask)
    nv, sv, zv = _quantise(v, 8, 128)
    kk, vv = (n.double() * s.double() + z.double())[0, -1], (nv.double() * sv.double() + zv.double())[0, -1]
    sc = (kk @ q[0, -1, 0].double()) * 128 ** -0.5
    want = torch.softmax(sc, 0) @ vv
    assert abs(float(lse[0, -1, 0]) - float(torch.logsumexp(sc, 0))) < 1e-4
    assert (out[0, 0, -1].cpu().double() - want).abs().max() <= 2 ** -8 * want.abs().max() + 2 ** -9 * vv.abs().max()


# ---- attention ---------------------------------------------------------------
def _attention(q, cache, lengths, mask, causal, scale):
    """f64 (out (B, Lq, Hq, 128), lse (B, Hq, Lq)) and the score error bound."""
    K, V = _decode(cache)
    B, Hq, Lq, _ = q.shape
    G = Hq // cache.n_kv_heads
    out = torch.zeros(B, Lq, Hq, 128, dtype=torch.float64)
    lse = torch.full((B, Hq, Lq), -float("inf"), dtype=torch.float64)
    bound, vmax = 0.0, 0.0
    for b in range(B):
        n = int(lengths[b])
        for h in range(Hq):
            for i in range(Lq):
                end = max(0, n - Lq + i + 1) if causal else n
                see = torch.arange(end)
                if mask is not None:
                    see = see[mask[b, :end].bool()]
                if len(see) == 0:
                    continue
                kk, vv, qq = K[b, h // G, see], V[b, h // G, see], q[b, h, i].double()
                s = kk @ qq * scale
                lse[b, h, i] = torch.logsumexp(s, 0)
                out[b, i, h] = torch.softmax(s, 0) @ vv
                bound = max(bound, float((kk.abs() @ qq.abs()).max()) * scale)
                vmax = max(vmax, float(vv.abs().max()))
    return out, lse, bound * (2.0 ** -20 if G * Lq <= 32 else 2.0 ** -11 + 2.0 ** -20), vmax


def _check(q, cache, lengths, dev, *, mask=None, causal=True, scale=None, max_length=None):
    from core_b200 import ops
    as_int = isinstance(lengths, int)
    ln = [lengths] * q.shape[0] if as_int else lengths
    dl = lengths if as_int else torch.tensor(lengths, dtype=torch.int32, device=dev)
    out, lse = ops.attention_quantized(q.to(dev), cache, dl, max_length=max_length, causal=causal,
                                       key_mask=None if mask is None else mask.to(dev), softmax_scale=scale)
    ops.status(dev)
    want, wl, ds, vmax = _attention(q, cache, ln, mask, causal, scale or 128 ** -0.5)
    got, gl = out.cpu().double(), lse.cpu().double()
    u = 2.0 ** -8 if q.dtype == torch.bfloat16 else 2.0 ** -11
    n = max(ln) if ln else 0
    tol = (2.0 ** -10 + n * 2.0 ** -17 + 2 * ds) * vmax + u * want.abs()
    assert torch.equal(torch.isinf(gl), torch.isinf(wl))
    empty = torch.isinf(wl)
    assert ((gl - wl)[~empty].abs() <= ds + 2e-5 + 1e-6 * wl[~empty].abs()).all(), (gl - wl)[~empty].abs().max()
    assert (got.transpose(1, 2)[empty] == 0).all()
    assert ((got - want).abs() <= tol).all(), float(((got - want).abs() - tol).max())
    assert (got - want).norm() <= 2.0 ** -8 * want.norm()
    return out, lse


def _filled(seed, B, H, cap, bits, group, dev, lengths, dtype=torch.bfloat16):
    from core_b200 import ops
    c = _poisoned(B, H, cap, bits, group, dev)
    n = max(max(lengths), 1)
    k, v = _rows(seed, (B, H, n, 128), dtype, 6.0), _rows(seed + 1, (B, H, n, 128), dtype)
    ops.kv_quantize(k.to(dev), v.to(dev), c, 0, counts=torch.tensor(lengths, dtype=torch.int32, device=dev))
    return c


@pytest.mark.parametrize("bits,group,dtype", list(itertools.product((4, 8), (32, 64, 128), ("bf16", "f16"))))
def test_attention_formats(bits, group, dtype):
    dev = _dev()
    lengths = [333, 64]
    c = _filled(20, 2, 2, 384, bits, group, dev, lengths)
    _check(_rows(22, (2, 8, 1, 128), DT[dtype], 2.0), c, lengths, dev, max_length=333)
    _check(_rows(23, (2, 8, 3, 128), DT[dtype], 2.0), c, lengths, dev, max_length=333)
    _check(_rows(24, (2, 8, 70, 128), DT[dtype], 2.0), c, lengths, dev, max_length=333)


@pytest.mark.parametrize("groups,queries", [(1, 1), (3, 1), (4, 1), (7, 1), (8, 1), (16, 1), (5, 2), (7, 5), (4, 8),
                                            (1, 33), (4, 40), (3, 67)])
def test_attention_rows(groups, queries):
    """Every number of query rows a KV head: one tile, odd ones, several."""
    dev = _dev()
    lengths = [130, 97]
    c = _filled(30, 2, 2, 256, 4, 64, dev, lengths)
    q = _rows(32, (2, 2 * groups, queries, 128), torch.bfloat16, 2.0)
    _check(q, c, lengths, dev, max_length=130)
    _check(q, c, lengths, dev, causal=False)


@pytest.mark.parametrize("length", [0, 1, 2, 15, 31, 32, 33, 63, 64, 65, 127, 128, 129, 255, 256, 1000, 2047])
def test_attention_lengths(length):
    """Tiles that end anywhere; sequences of length 0 and 1; splits."""
    dev = _dev()
    lengths = [length, 1, 0]
    c = _filled(40 + length, 3, 1, 2048, 4, 32, dev, lengths)
    for queries in (1, 4, 36):
        q = _rows(43, (3, 4, queries, 128), torch.float16, 2.0)
        _check(q, c, lengths, dev, max_length=max(lengths))
        _check(q, c, lengths, dev)  # bound left at the capacity


@pytest.mark.parametrize("bits,group", list(itertools.product((4, 8), (32, 64, 128))))
@pytest.mark.parametrize("heads,length", [(288, 300), (8, 16001)], ids=["many_heads", "long"])
def test_attention_three_tiles_of_rows(bits, group, heads, length):
    """17 to 24 rows a KV head, which one CTA takes together where there are many
    heads, or long sequences whose parts are joined."""
    dev = _dev()
    lengths = [length]
    c = _filled(140, 1, heads, -(-length // 128) * 128, bits, group, dev, lengths)
    mask = torch.rand(1, length, generator=torch.Generator().manual_seed(3)) > 0.2
    for queries in (5, 6):
        q = _rows(141, (1, 4 * heads, queries, 128), torch.bfloat16, 2.0)
        _check(q, c, lengths, dev, max_length=length)
    _check(q, c, lengths, dev, mask=mask, max_length=length)


@pytest.mark.parametrize("bits,group", list(itertools.product((4, 8), (32, 64, 128))))
def test_attention_full_device(bits, group):
    """Few rows and enough heads to fill every SM: single tokens of a large batch."""
    dev = _dev()
    lengths = [200, 0, 131, 64]
    c = _filled(160, 4, 140, 256, bits, group, dev, lengths)
    _check(_rows(162, (4, 280, 1, 128), torch.bfloat16, 2.0), c, lengths, dev, max_length=200)
    _check(_rows(163, (4, 280, 3, 128), torch.float16, 2.0), c, lengths, dev, max_length=200)


@pytest.mark.parametrize("lengths", [[5000, 0, 17, 3000, 128, 1], [700] * 5, [0, 0, 0], [1, 2, 4096],
                                     [(37 * i) % 1500 if i % 7 else 0 for i in range(45)]],
                         ids=["uneven", "even", "empty", "one_long", "many"])
def test_attention_ragged_batches(lengths):
    """Parts dealt out over sequences of unequal lengths, empty ones and more than
    a warp's worth of them; few and many query rows; a bound far above the lengths."""
    dev = _dev()
    B = len(lengths)
    cap = -(-max(max(lengths), 1) // 128) * 128 + 2048
    c = _filled(120, B, 1, cap, 4, 64, dev, lengths)
    for queries in (1, 3, 20):
        q = _rows(122, (B, 2, queries, 128), torch.float16, 2.0)
        _check(q, c, lengths, dev, max_length=max(lengths))
        _check(q, c, lengths, dev)


def test_attention_masks():
    """Hidden tokens anywhere, rows that see nothing, NaN and infinities in
    hidden places; bool and uint8 masks, broadcast and strided."""
    dev = _dev()
    B, H, n = 4, 2, 700
    from core_b200 import ops
    g = torch.Generator().manual_seed(50)
    k, v = _rows(51, (B, H, n, 128), torch.bfloat16, 6.0), _rows(52, (B, H, n, 128), torch.bfloat16)
    mask = torch.rand(B, 1024, generator=g) < 0.5
    mask[1] = False
    mask[2, :650] = False
    mask[3] = True
    hidden = ~mask[:, None, :n, None].expand(B, H, n, 128)
    k[hidden] = float("nan")
    v[hidden] = float("inf")
    v[0, :, 3] = torch.where(mask[0, 3], v[0, :, 3], torch.full_like(v[0, :, 3], float("nan")))
    c = _poisoned(B, H, 1024, 4, 64, dev)
    ops.kv_quantize(k.to(dev), v.to(dev), c, 0)
    for queries in (1, 6, 40):
        q = _rows(53, (B, 4 * H, queries, 128), torch.bfloat16, 2.0)
        a = _check(q, c, n, dev, mask=mask)
        b = _check(q, c, n, dev, mask=mask.to(torch.uint8) * 255)
        assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])
        wide = torch.zeros(B, 2048, dtype=torch.bool)
        wide[:, ::2] = mask
        d = ops.attention_quantized(q.to(dev), c, n, key_mask=wide.to(dev)[:, ::2])
        assert torch.equal(a[0], d[0])
    one = mask[3:].expand(B, -1).to(dev)
    e = ops.attention_quantized(q.to(dev)[3:].expand(B, -1, -1, -1), c, n, key_mask=one)
    assert torch.equal(e[0][3], a[0][3])


def test_attention_extreme_scores_and_queries():
    """Scores of thousands, a lone large key late in the sequence (the running
    maximum is raised again and again), zero and tiny queries."""
    dev = _dev()
    from core_b200 import ops
    n = 600
    k, v = _rows(60, (1, 1, n, 128), torch.float32), _rows(61, (1, 1, n, 128), torch.float32)
    k *= torch.linspace(0.1, 40.0, n)[None, None, :, None]
    c = _poisoned(1, 1, 640, 8, 32, dev)
    ops.kv_quantize(k.to(dev), v.to(dev), c, 0)
    q = _rows(62, (1, 6, 1, 128), torch.bfloat16)
    q[0, 1] = 0
    q[0, 2] *= 1e-30
    q[0, 3] *= 30
    q[0, 4] = k[0, 0, -1].to(torch.bfloat16)
    _check(q, c, n, dev)


def test_attention_nan_query_and_key_stay_in_their_rows():
    dev = _dev()
    from core_b200 import ops
    c = _filled(70, 2, 1, 256, 4, 64, dev, [200, 200])
    q = _rows(72, (2, 4, 1, 128), torch.bfloat16)
    clean, _ = ops.attention_quantized(q.to(dev), c, 200)
    q[0, 2, 0, 9] = float("nan")
    out, lse = ops.attention_quantized(q.to(dev), c, 200)
    bad = torch.zeros(2, 1, 4, dtype=torch.bool)
    bad[0, 0, 2] = True
    assert out.cpu()[bad].isnan().all() and lse.cpu()[0, 2].isnan().all()
    assert torch.equal(out.cpu()[~bad], clean.cpu()[~bad])


def test_attention_strided_queries_scale_and_streams():
    """Queries as an attention module passes them, another scale, another stream."""
    dev = _dev()
    from core_b200 import ops
    lengths = [300, 77]
    c = _filled(80, 2, 2, 384, 4, 128, dev, lengths)
    q = _rows(82, (2, 5, 8, 128), torch.float16).transpose(1, 2)
    _check(q, c, lengths, dev, scale=0.3)
    a, la = ops.attention_quantized(q.to(dev), c, 77)
    s = torch.cuda.Stream(dev)
    qd = q.to(dev)
    s.wait_stream(torch.cuda.current_stream(dev))
    with torch.cuda.stream(s):
        b, lb = ops.attention_quantized(qd, c, 77)
    torch.cuda.current_stream(dev).wait_stream(s)
    assert torch.equal(a, b) and torch.equal(la, lb)


def test_attention_is_the_same_twice():
    dev = _dev()
    from core_b200 import ops
    c = _filled(90, 1, 8, 20096, 4, 64, dev, [20011])
    for queries in (1, 3, 64):
        q = _rows(92, (1, 32, queries, 128), torch.bfloat16, 2.0).to(dev)
        a, la = ops.attention_quantized(q, c, 20011)
        b, lb = ops.attention_quantized(q, c, 20011)
        assert torch.equal(a, b) and torch.equal(la, lb)


def test_attention_in_a_cuda_graph():
    dev = _dev()
    from core_b200 import ops
    c = _filled(95, 1, 2, 4096, 4, 64, dev, [4000])
    q = _rows(96, (1, 8, 1, 128), torch.bfloat16).to(dev)
    n = torch.tensor([4000], dtype=torch.int32, device=dev)
    want, _ = ops.attention_quantized(q, c, n, max_length=4096)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        out, _ = ops.attention_quantized(q, c, n, max_length=4096)
    g.replay()
    torch.cuda.synchronize()
    assert torch.equal(out, want)
    n.fill_(1234)
    want, _ = ops.attention_quantized(q, c, n, max_length=4096)
    g.replay()
    assert torch.equal(out, want)


# ---- the cache object -----------------------------------------------------------
def test_append_and_attend_token_by_token():
    """Decoding: appended tokens are seen by the next step."""
    from core_b200.kvcache import QuantizedKV
    dev = _dev()
    c = QuantizedKV.empty(2, 2, 100, bits=4, group=32, device=dev)
    assert c.capacity == 128
    k, v = _rows(100, (2, 2, 60, 128), torch.bfloat16, 6.0), _rows(101, (2, 2, 60, 128), torch.bfloat16)
    c.append(k[:, :, :50].to(dev), v[:, :, :50].to(dev),
             counts=torch.tensor([50, 20], dtype=torch.int32, device=dev))
    for t in range(50, 60):
        c.append(k[:, :, t:t + 1].to(dev), v[:, :, t:t + 1].to(dev))
        q = _rows(102 + t, (2, 4, 1, 128), torch.bfloat16)
        out, lse = c.attend(q.to(dev))
        lengths = c.lengths.tolist()
        assert lengths == [t + 1, t - 29] and c.max_length == t + 1
        want, wl, ds, vmax = _attention(q, c, lengths, None, True, 128 ** -0.5)
        assert (lse.cpu().double() - wl).abs().max() <= ds + 3e-5
        assert ((out.cpu().double() - want).abs() <= (2 ** -9 + 2 * ds) * vmax + 2 ** -8 * want.abs()).all()
    rk, rv = c.read(dtype=torch.float32)
    n, s, z = _quantise(k, 4, 32)
    assert torch.equal(rk[0].cpu(), (n.unflatten(-1, (4, 32)) * s.double()[..., None]
                                     + z.double()[..., None]).flatten(-2)[0].float())
    with pytest.raises(ValueError, match="capacity"):
        c.append(torch.zeros(2, 2, 69, 128, dtype=torch.bfloat16, device=dev),
                 torch.zeros(2, 2, 69, 128, dtype=torch.bfloat16, device=dev))
    c.reset()
    assert c.max_length == 0 and c.lengths.tolist() == [0, 0]


def test_device_side_range_errors_are_reported():
    """Slots, source rows and lengths out of range are skipped or clamped and recorded."""
    from core_b200 import ops
    from core_b200._lib import CoreError
    dev = _dev()
    c = _poisoned(2, 1, 128, 4, 64, dev)
    k = _rows(110, (2, 1, 8, 128), torch.bfloat16).to(dev)
    ops.kv_quantize(k, k, c, torch.tensor([0, 124], dtype=torch.int32, device=dev))
    with pytest.raises(CoreError, match="where=1401"):
        ops.status(dev)
    assert not c.k_meta[1, 0, 124:].isnan().any() and not c.k_meta[0, 0, :8].isnan().any()
    ops.kv_quantize(k, k, c, 0, index=torch.tensor([[0, 8], [-1, 1]], device=dev))
    with pytest.raises(CoreError, match="where=1402"):
        ops.status(dev)
    got, _ = ops.kv_dequantize(c, index=torch.tensor([[0, 128], [1, -1]], device=dev))
    with pytest.raises(CoreError, match="where=1411"):
        ops.status(dev)
    assert (got[0, :, 1] == 0).all() and (got[1, :, 1] == 0).all()
    q = _rows(111, (2, 1, 1, 128), torch.bfloat16).to(dev)
    ops.attention_quantized(q, c, torch.tensor([9, -3], dtype=torch.int32, device=dev), max_length=8)
    with pytest.raises(CoreError, match="where=1421"):
        ops.status(dev)
    ops.status(dev)


def test_refusals():
    from core_b200 import ops
    from core_b200.kvcache import QuantizedKV
    dev = _dev()
    c = QuantizedKV.empty(2, 2, 128, device=dev)
    k = torch.zeros(2, 2, 4, 128, dtype=torch.bfloat16, device=dev)
    q = torch.zeros(2, 4, 1, 128, dtype=torch.bfloat16, device=dev)
    i32 = torch.zeros(2, dtype=torch.int32, device=dev)
    bad = [
        (ValueError, lambda: QuantizedKV.empty(1, 1, 128, bits=2, device=dev)),
        (ValueError, lambda: QuantizedKV.empty(1, 1, 128, group=16, device=dev)),
        (ValueError, lambda: QuantizedKV.empty(0, 1, 128, device=dev)),
        (ValueError, lambda: QuantizedKV(c.k_codes[:, :, :100].contiguous(), c.k_meta, c.v_codes, c.v_meta)),
        (ValueError, lambda: QuantizedKV(c.k_codes, c.k_meta.float(), c.v_codes, c.v_meta)),
        (ValueError, lambda: QuantizedKV(c.k_codes, c.k_meta, c.v_codes.cpu(), c.v_meta)),
        (ValueError, lambda: ops.kv_quantize(k.cpu(), k.cpu(), c, 0)),
        (TypeError, lambda: ops.kv_quantize(k.double(), k.double(), c, 0)),
        (TypeError, lambda: ops.kv_quantize(k, k.half(), c, 0)),
        (ValueError, lambda: ops.kv_quantize(k[..., :64], k[..., :64], c, 0)),
        (ValueError, lambda: ops.kv_quantize(k[:1], k[:1], c, 0)),
        (ValueError, lambda: ops.kv_quantize(k, k, c, i32.long())),
        (ValueError, lambda: ops.kv_quantize(k, k, c, i32.cpu())),
        (ValueError, lambda: ops.kv_quantize(k, k, c, 0, index=i32)),
        (RuntimeError, lambda: ops.kv_quantize(k, k, c, 125)),
        (RuntimeError, lambda: ops.kv_quantize(k, k, c, -1)),
        (TypeError, lambda: ops.kv_dequantize(c, count=3, dtype=torch.float64)),
        (ValueError, lambda: ops.kv_dequantize(c)),
        (ValueError, lambda: ops.kv_dequantize(c, count=-1)),
        (RuntimeError, lambda: ops.kv_dequantize(c, start=120, count=9)),
        (TypeError, lambda: ops.attention_quantized(q.float(), c, 4)),
        (ValueError, lambda: ops.attention_quantized(q[:, :3], c, 4)),
        (ValueError, lambda: ops.attention_quantized(q[..., :64], c, 4)),
        (ValueError, lambda: ops.attention_quantized(q[:1], c, 4)),
        (RuntimeError, lambda: ops.attention_quantized(q, c, 129)),
        (RuntimeError, lambda: ops.attention_quantized(q, c, -1)),
        (RuntimeError, lambda: ops.attention_quantized(q, c, 4, softmax_scale=0.0)),
        (ValueError, lambda: ops.attention_quantized(q, c, i32[:1])),
        (ValueError, lambda: ops.attention_quantized(q, c, 4, key_mask=torch.ones(2, 3, dtype=torch.bool, device=dev))),
        (ValueError, lambda: ops.attention_quantized(q, c, 4, key_mask=torch.ones(2, 4, device=dev))),
        (ValueError, lambda: ops.attention_quantized(q, c, 4, out=q)),
    ]
    for kind, call in bad:
        with pytest.raises(kind):
            call()
    e, _ = ops.kv_dequantize(c, count=0)
    assert e.shape == (2, 2, 0, 128)
    ops.status(dev)


def test_index_types_and_values_beyond_32_bits():
    """Indexes are int32 or int64; a value that does not fit 32 bits is out of
    range, not some other row."""
    from core_b200 import ops
    from core_b200._lib import CoreError
    from core_b200.kvcache import QuantizedKV
    dev = _dev()
    c = QuantizedKV.empty(1, 1, 128, device=dev)
    k = _rows(150, (1, 1, 4, 128), torch.bfloat16).to(dev)
    c.append(k, k)
    want = ops.kv_dequantize(c, index=torch.tensor([[2, 0]], dtype=torch.int32, device=dev))[0]
    assert torch.equal(ops.kv_dequantize(c, index=torch.tensor([[2, 0]], device=dev))[0], want)
    for far in (2 ** 32 + 1, -2 ** 32 + 1, 2 ** 31):
        got = ops.kv_dequantize(c, index=torch.tensor([[2, far]], device=dev))[0]
        assert torch.equal(got[0, 0, 0], want[0, 0, 0]) and (got[0, 0, 1] == 0).all()
        with pytest.raises(CoreError, match="where=1411"):
            ops.status(dev)
        before = c.k_codes.clone()
        ops.kv_quantize(k, k, c, 4, index=torch.tensor([[far]], device=dev))
        with pytest.raises(CoreError, match="where=1402"):
            ops.status(dev)
        assert torch.equal(c.k_codes, before)
    for bad in (torch.float32, torch.bool, torch.int16):
        with pytest.raises(TypeError):
            ops.kv_dequantize(c, index=torch.zeros(1, 2, device=dev, dtype=bad))
        with pytest.raises(TypeError):
            ops.kv_quantize(k, k, c, 0, index=torch.zeros(1, 2, device=dev, dtype=bad))
    ops.status(dev)
