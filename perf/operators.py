"""Cases that measure the quantised KV cache: writing rows into it, reading them back, and attention over it.

The cache holds keys and values in 4 or 8 bits.  A row is one token of one KV head, 128 channels.  Each group of
`group` neighbouring channels (32, 64 or 128) has an f16 scale s and an f16 zero z, and a code n stands for n s + z.

    lo, hi = the group's least and greatest value, both kept within +-61440
    z = f16(lo)     s = f16((hi - lo) / N)     n = round((x - z) / s), kept in 0..N     N = 15 or 255

Layout (all tensors contiguous; capacity a multiple of 128):
    codes (B, Hkv, capacity, 16 bits) uint8     meta (B, Hkv, capacity, 128 / group, 2) f16: (s, z)
    A 32-bit word holds 8 (4) channels e0.. of one row: 4 bits: e0 e2 e4 e6 e1 e3 e5 e7 from the lowest nibble up;
    8 bits: bytes e0 e2 e1 e3.
    Keys, 4 bits: the word of channels 32 b + 8 t .. + 7 is word 4 t + b of the row (b, t in 0..3).
    Keys, 8 bits: the word of channels 32 b + 8 t + 4 h .. + 3 is word 16 (b / 2) + 4 t + 2 (b % 2) + h, and odd tokens
    have the row's two halves exchanged (word ^ 16).
    Values: words in channel order; tokens with bit 1 set have word ^ 8 (4 bits), token t has word ^ 8 (t % 4) (8 bits).
"""
import math

import torch

own = False

D = 128          # head dimension
LIMIT = 61440.0  # values beyond +-LIMIT saturate
DTYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}


# ---------------------------------------------------------------- cases

def _write(name, **c):
    return dict(name=name, op="write", **c)


def _read(name, **c):
    return dict(name=name, op="read", **c)


def _attend(name, **c):
    return dict(name=name, op="attention", **c)


def listed():
    return [
        # the token that every sequence of a decoding batch adds to its cache, at its own place
        _write("write_token", batch=8, heads=8, rows=1, source=0, capacity=4224, bits=4, group=64, dtype="bf16"),
        # a 16384-token prompt of one sequence into the cache
        _write("write_prompt", batch=1, heads=8, rows=16384, source=0, capacity=16384, bits=4, group=64, dtype="bf16"),
        # the rows that a compression step kept, picked from the full cache; 8 bits, an odd number of f16 rows
        _write("write_kept", batch=2, heads=8, rows=4099, source=16387, capacity=4224, bits=8, group=32, dtype="f16"),
        # the prompts of a served batch
        _write("write_batch", batch=8, heads=8, rows=32768, source=0, capacity=32768, bits=4, group=32, dtype="bf16"),
        # a whole cache back as bf16 keys and values, as a scoring pass takes them
        _read("read_all", batch=1, heads=8, rows=16384, picked=False, capacity=16384, bits=4, group=64, dtype="bf16"),
        # picked rows of a batch in f32, 8 bits
        _read("read_picked", batch=3, heads=2, rows=1001, picked=True, capacity=2944, bits=8, group=128, dtype="f32"),
        # one new token over a short answer's cache: latency counts
        _attend("decode_short", batch=1, heads=8, groups=4, queries=1, length=333, ragged=False, padded=False, capacity=384, bits=4, group=64, dtype="bf16"),
        # one new token over the longest sequence
        _attend("decode_long", batch=1, heads=8, groups=4, queries=1, length=131072, ragged=False, padded=False, capacity=131072, bits=4, group=64, dtype="bf16"),
        # one new token for each of a served batch of unequal lengths, one of them empty
        _attend("decode_batch", batch=8, heads=8, groups=4, queries=1, length=32768, ragged=True, padded=False, capacity=32768, bits=4, group=32, dtype="bf16"),
        # a few proposed tokens checked at once, left-padded batch, 8 bits, seven query heads to a KV head
        _attend("verify_padded", batch=4, heads=4, groups=7, queries=5, length=8191, ragged=False, padded=True, capacity=8192, bits=8, group=32, dtype="f16"),
        # a piece of a prompt over what the cache holds of it
        _attend("chunk", batch=1, heads=8, groups=4, queries=512, length=16384, ragged=False, padded=False, capacity=16384, bits=4, group=128, dtype="bf16"),
        # the same for a ragged batch of odd sizes, 8 bits
        _attend("chunk_ragged", batch=3, heads=2, groups=4, queries=129, length=5000, ragged=True, padded=False, capacity=5120, bits=8, group=64, dtype="f16"),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    bits, group = rng.choice((4, 4, 8)), rng.choice((32, 64, 128))
    heads = rng.choice((1, 2, 4, 8))
    op = rng.choice(("write", "read", "attention", "attention", "attention"))
    if op == "write":
        batch = _log(rng, 1, 16)
        rows = _log(rng, 1, max(2, 131072 // batch))
        source = rows + _log(rng, 1, 4 * rows) if rows < 16384 and rng.random() < 0.4 else 0
        capacity = -(-(rows + rng.randrange(1, 700)) // 128) * 128
        return dict(op=op, batch=batch, heads=heads, rows=rows, source=source, capacity=capacity, bits=bits, group=group,
                    dtype=rng.choice(("bf16", "bf16", "f16", "f32")))
    if op == "read":
        batch = _log(rng, 1, 16)
        rows = _log(rng, 1, max(2, 131072 // batch))
        capacity = -(-(rows + rng.randrange(1, 700)) // 128) * 128
        return dict(op=op, batch=batch, heads=heads, rows=rows, picked=rng.random() < 0.5, capacity=capacity, bits=bits,
                    group=group, dtype=rng.choice(("bf16", "bf16", "f16", "f32")))
    groups = rng.choice((1, 2, 4, 4, 5, 7, 8))
    if rng.random() < 0.6:  # decoding
        batch, queries = _log(rng, 1, 16), rng.choice((1, 1, 1, 2, 3, 7))
        length = _log(rng, 1, max(2, 131072 // batch))
    else:  # pieces of prompts
        batch, queries = rng.choice((1, 1, 2, 3)), _log(rng, 8, 700)
        length = queries + _log(rng, 1, 16384 // batch)
        heads, groups = min(heads, 4), min(groups, 4)
    capacity = -(-(length + rng.randrange(1, 300)) // 128) * 128
    return dict(op=op, batch=batch, heads=heads, groups=groups, queries=queries, length=length, ragged=batch > 1 and rng.random() < 0.5,
                padded=rng.random() < 0.3, capacity=capacity, bits=bits, group=group, dtype=rng.choice(("bf16", "f16")))


def _lengths(case):
    """Tokens of each sequence: all alike, or falling to three eighths with the last one (of four or more) empty."""
    n, batch = case["length"], case["batch"]
    if not case["ragged"]:
        return [n] * batch
    got = [n - (5 * n * b) // (8 * batch) for b in range(batch)]
    if batch >= 4:
        got[-1] = 0
    return got


def _pads(case):
    """Masked tokens at the front of each sequence of a left-padded batch."""
    return [(case["length"] * b) // (2 * case["batch"]) if case["padded"] else 0 for b in range(case["batch"])]


def _with_lse(case):
    """Decoding returns the f32 row log-sum-exp too (what joins it with attention over other keys).  A prompt's attention
    is used for its 16-bit output, and many-row kernels may take keys in 16 bits."""
    return case["queries"] * case["groups"] <= 32


def work(case):
    size = {"bf16": 2, "f16": 2, "f32": 4}[case["dtype"]]
    packed = 16 * case["bits"] + 4 * (D // case["group"])  # bytes of one row
    if case["op"] == "attention":
        q, per, read, pairs = case["queries"], case["heads"] * case["groups"], 0, 0
        for n, pad in zip(_lengths(case), _pads(case)):
            read += 2 * case["heads"] * max(0, n - pad) * packed
            pairs += sum(max(0, n - q + i + 1 - pad) for i in range(q)) * per
        out = case["batch"] * per * q * (2 * D * size + 4)
        return {"bytes": read + out, "flops": 4 * D * pairs}
    rows = 2 * case["batch"] * case["heads"] * case["rows"]
    if case["op"] == "write":
        return {"bytes": rows * (2 * D * size + packed), "flops": 8 * D * rows}
    return {"bytes": rows * (D * size + packed), "flops": 2 * D * rows}


# ---------------------------------------------------------------- inputs

def _rows(batch, heads, n, gen, spread, dtype):
    """Rows as models have them: normal, with four channels of each head `spread` times as large."""
    x = torch.randn(batch, heads, n, D, generator=gen, device="cuda")
    if spread != 1.0:
        at = torch.rand(heads, D, generator=gen, device="cuda").argsort(1)[:, :4]
        x *= torch.ones(heads, D, device="cuda").scatter_(1, at, spread)[None, :, None, :]
    return x.to(dtype)


def _quantise(x, bits, group):
    """Codes (.., 128) and scale and zero (.., 128 / group) of rows, in 32 bits."""
    top = float(2 ** bits - 1)
    g = x.float().clamp(-LIMIT, LIMIT).unflatten(-1, (D // group, group))
    lo, hi = g.amin(-1), g.amax(-1)
    z = lo.half()
    s = ((hi - lo) * torch.tensor(1.0 / top, dtype=torch.float32, device=x.device)).half()
    inv = torch.where(s > 0, 1.0 / s.float(), torch.zeros_like(lo))
    n = ((g - z.float()[..., None]) * inv[..., None]).round().clamp(0.0, top)
    return torch.nan_to_num(n).flatten(-2), s, z


def _pack(n, bits, keys):
    """Codes (.., rows, 128) in the cache's layout, as bytes."""
    tokens = torch.arange(n.shape[-2], device=n.device)
    n = n.to(torch.uint8).int()
    if bits == 4:
        w = n.unflatten(-1, (16, 4, 2))
        w = (w << (torch.arange(4, device=n.device)[:, None] * 4 + torch.arange(2, device=n.device) * 16)).sum((-1, -2), dtype=torch.int64)
        order = torch.arange(16, device=n.device)
        if keys:
            at = (4 * (order % 4) + order // 4).expand(len(tokens), 16)
        else:
            at = order ^ (((tokens[:, None] >> 1) & 1) * 8)
    else:
        w = n.unflatten(-1, (32, 2, 2))
        w = (w << (torch.arange(2, device=n.device)[:, None] * 8 + torch.arange(2, device=n.device) * 16)).sum((-1, -2), dtype=torch.int64)
        order = torch.arange(32, device=n.device)
        if keys:
            b, t, h = order // 8, order // 2 % 4, order % 2
            at = (16 * (b // 2) + 4 * t + 2 * (b % 2) + h) ^ ((tokens[:, None] & 1) * 16)
        else:
            at = order ^ ((tokens[:, None] & 3) * 8)
    w = torch.where(w >= 2 ** 31, w - 2 ** 32, w).int()
    out = torch.empty_like(w)
    out.scatter_(-1, at.expand(w.shape), w)
    return out.view(torch.uint8)


def _filled(case, gen, lengths):
    """Buffers of a cache with `lengths` tokens; what follows them was never written (here: bytes that read as NaN)."""
    batch, heads, cap, bits, group = (case[k] for k in ("batch", "heads", "capacity", "bits", "group"))
    got = []
    for keys in (True, False):
        codes = torch.full((batch, heads, cap, 16 * bits), 0x7F, dtype=torch.uint8, device="cuda")
        meta = torch.full((batch, heads, cap, D // group, 4), 0x7F, dtype=torch.uint8, device="cuda").view(torch.float16)
        for b, n in enumerate(lengths):
            if n:
                x = _rows(1, heads, n, gen, 6.0 if keys else 1.0, torch.float32)
                c, s, z = _quantise(x, bits, group)
                codes[b, :, :n] = _pack(c, bits, keys)[0]
                meta[b, :, :n] = torch.stack((s, z), -1)[0]
        got += [codes, meta]
    return got


def prepare(case, seed):
    gen = torch.Generator(device="cuda")
    gen.manual_seed(int(seed))
    batch, heads, cap, bits, group = (case[k] for k in ("batch", "heads", "capacity", "bits", "group"))
    dtype = DTYPES[case["dtype"]]
    state = {"case": case, "dtype": dtype, "bits": bits, "group": group}
    if case["op"] == "write":
        n, source = case["rows"], case["source"] or case["rows"]
        state["k"] = _rows(batch, heads, source, gen, 6.0, dtype)
        state["v"] = _rows(batch, heads, source, gen, 1.0, dtype)
        room = cap - n
        state["start"] = torch.randint(0, room + 1, (batch,), generator=gen, device="cuda").int()
        state["index"] = None
        if case["source"]:
            at = torch.rand(batch, source, generator=gen, device="cuda").argsort(1)[:, :n]
            state["index"] = at.sort(1).values.int().contiguous()
        state["buffers"] = [torch.empty(batch, heads, cap, 16 * bits, dtype=torch.uint8, device="cuda"),
                            torch.empty(batch, heads, cap, D // group, 2, dtype=torch.float16, device="cuda")]
        state["buffers"] += [torch.empty_like(t) for t in state["buffers"]]
    elif case["op"] == "read":
        state["buffers"] = _filled(case, gen, [cap] * batch)
        state["rows"] = case["rows"]
        if case["picked"]:
            at = torch.rand(batch, cap, generator=gen, device="cuda").argsort(1)[:, :case["rows"]]
            state["index"] = at.sort(1).values.int().contiguous()
        else:
            state["index"] = None
    else:
        lengths = _lengths(case)
        state["buffers"] = _filled(case, gen, lengths)
        state["lengths"] = torch.tensor(lengths, dtype=torch.int32, device="cuda")
        state["longest"] = case["length"]
        state["q"] = _rows(batch, heads * case["groups"], case["queries"], gen, 2.0, dtype)
        state["mask"] = None
        if case["padded"]:
            pads = torch.tensor(_pads(case), device="cuda")
            state["mask"] = torch.arange(cap, device="cuda")[None, :] >= pads[:, None]
    return state


# ---------------------------------------------------------------- the operators

def _unpack(codes, bits, keys):
    """Bytes in the cache's layout, (B, H, capacity, bytes), as codes (B, H, capacity, 128) in 32 bits."""
    w = codes.view(torch.int32)
    tokens = torch.arange(w.shape[2], device=w.device)[:, None]
    words = 4 * bits
    order = torch.arange(words, device=w.device)
    if keys and bits == 4:
        at = (4 * (order % 4) + order // 4).expand(len(tokens), words)
    elif keys:
        at = (16 * (order // 16) + 4 * (order // 2 % 4) + 2 * (order // 8 % 2) + order % 2) ^ ((tokens & 1) * 16)
    else:
        at = order ^ (((tokens >> 1) & 1) * 8 if bits == 4 else (tokens & 3) * 8)
    w = w.gather(-1, at.expand(w.shape))
    low = (torch.arange(16 // bits, device=w.device) * bits)[:, None] + torch.arange(2, device=w.device) * 16
    return ((w[..., None, None] >> low) & (2 ** bits - 1)).flatten(-3).float()


def _values(codes, meta, bits, keys):
    n = _unpack(codes, bits, keys)
    s, z = meta[..., 0].float(), meta[..., 1].float()
    g = s.shape[-1]
    return (n.unflatten(-1, (g, D // g)) * s[..., None] + z[..., None]).flatten(-2)


def _plain(state):
    case, bits, dtype = state["case"], state["bits"], state["dtype"]
    if case["op"] == "write":
        out = []
        for x in (state["k"], state["v"]):
            if state["index"] is not None:
                x = x.gather(2, state["index"].long()[:, None, :, None].expand(-1, x.shape[1], -1, D))
            n, s, z = _quantise(x, bits, state["group"])
            v = n.unflatten(-1, (D // state["group"], state["group"])) * s.float()[..., None] + z.float()[..., None]
            out.append(v.flatten(-2).to(dtype))
        return out
    picked = case["op"] == "read" and state["index"] is not None
    n = case["capacity"] if picked else state["rows"] if case["op"] == "read" else state["longest"]
    kc, km, vc, vm = (t[:, :, :n] for t in state["buffers"])
    k, v = _values(kc, km, bits, True), _values(vc, vm, bits, False)
    if case["op"] == "read":
        if picked:
            at = state["index"].long()[:, None, :, None].expand(-1, k.shape[1], -1, D)
            k, v = k.gather(2, at), v.gather(2, at)
        return [k.to(dtype), v.to(dtype)]
    nq, g = case["queries"], case["groups"]
    at = torch.arange(n, device="cuda")
    seen = at[None, :] < state["lengths"][:, None]
    if state["mask"] is not None:
        seen = seen & state["mask"][:, :n]
    k = torch.where(seen[:, None, :, None], k, 0.0)
    v = torch.where(seen[:, None, :, None], v, 0.0)
    q = state["q"].float().unflatten(1, (-1, g)).flatten(2, 3)  # (B, Hkv, g nq, 128)
    s = (q @ k.transpose(-1, -2)) * D ** -0.5
    last = state["lengths"][:, None] - nq + torch.arange(nq, device="cuda")  # the last token that a query sees
    ok = (seen[:, None, :] & (at <= last[:, :, None])).repeat(1, g, 1)[:, None]
    s = torch.where(ok, s, -math.inf)
    m = s.amax(-1, keepdim=True).clamp(min=-1e30)
    p = torch.exp(s - m)
    total = p.sum(-1, keepdim=True)
    o = (p @ v) / total.clamp(min=1e-37)
    lse = (m + torch.log(total)).squeeze(-1).unflatten(-1, (g, nq)).flatten(1, 2)
    out = o.unflatten(2, (g, nq)).flatten(1, 2).transpose(1, 2).to(dtype).contiguous()
    return [out, lse] if _with_lse(case) else [out]


def run(state):
    if not own:
        return _plain(state)
    from core_b200 import kvcache, ops

    cache = kvcache.QuantizedKV(*state["buffers"])
    case = state["case"]
    if case["op"] == "write":
        ops.kv_quantize(state["k"], state["v"], cache, state["start"], index=state["index"])
        return ops.kv_dequantize(cache, start=state["start"], count=case["rows"], dtype=state["dtype"])
    if case["op"] == "read":
        return ops.kv_dequantize(cache, count=state["rows"], index=state["index"], dtype=state["dtype"])
    out, lse = ops.attention_quantized(state["q"], cache, state["lengths"], max_length=state["longest"], key_mask=state["mask"])
    return [out, lse] if _with_lse(case) else [out]


# ---------------------------------------------------------------- the same in 64 bits

def _decoded(codes, meta, bits, keys):
    """(rows, 128) in f64 from one head's bytes: where each channel's bits lie, channel by channel."""
    rows = codes.shape[0]
    c = torch.arange(D, device=codes.device)
    t = torch.arange(rows, device=codes.device)[:, None]
    if bits == 4:
        e = c % 8
        bit = 16 * (e % 2) + 4 * (e // 2)
        word = 4 * (c % 32 // 8) + c // 32 if keys else c // 8
        word = word + 0 * t if keys else word ^ (8 * (t // 2 % 2))
    else:
        e = c % 4
        bit = 16 * (e % 2) + 8 * (e // 2)
        if keys:
            word = (16 * (c // 64) + 4 * (c % 32 // 8) + 2 * (c // 32 % 2) + c % 8 // 4) ^ (16 * (t % 2))
        else:
            word = (c // 4) ^ (8 * (t % 4))
    byte = codes.gather(1, 4 * word + bit // 8).to(torch.int64)
    n = torch.remainder(byte // 2 ** (bit % 8), 2 ** bits).double()
    of = c // (D // meta.shape[1])
    return n * meta[:, of, 0].double() + meta[:, of, 1].double()


def exact(case, seed):
    state = prepare(case, seed)
    batch, heads, bits = case["batch"], case["heads"], case["bits"]
    if case["op"] == "write":
        out, size = [], case["group"]
        for x in (state["k"], state["v"]):
            y = torch.empty(batch, heads, case["rows"], D, dtype=torch.float64, device="cuda")
            for b in range(batch):
                r = x[b] if state["index"] is None else x[b][:, state["index"][b].long()]
                r = r.double().clamp(-LIMIT, LIMIT)
                for c in range(0, D, size):
                    part = r[:, :, c:c + size]
                    z = part.amin(2, keepdim=True)
                    s = ((part.amax(2, keepdim=True) - z) / (2 ** bits - 1)).half().double()
                    z = z.half().double()
                    n = torch.where(s > 0, torch.round((part - z) / s), 0.0).clamp(0, 2 ** bits - 1)
                    y[b, :, :, c:c + size] = n * s + z
            out.append(y)
        return out
    kc, km, vc, vm = state["buffers"]
    if case["op"] == "read":
        out = [torch.empty(batch, heads, case["rows"], D, dtype=torch.float64, device="cuda") for _ in range(2)]
        for b in range(batch):
            at = torch.arange(case["rows"], device="cuda") if state["index"] is None else state["index"][b].long()
            for h in range(heads):
                out[0][b, h] = _decoded(kc[b, h], km[b, h], bits, True)[at]
                out[1][b, h] = _decoded(vc[b, h], vm[b, h], bits, False)[at]
        return out
    nq, g = case["queries"], case["groups"]
    out = torch.zeros(batch, nq, heads * g, D, dtype=torch.float64, device="cuda")
    lse = torch.full((batch, heads * g, nq), -math.inf, dtype=torch.float64, device="cuda")
    for b, n in enumerate(_lengths(case)):
        pad = _pads(case)[b]
        if n <= pad:
            continue
        for h in range(heads):
            k = _decoded(kc[b, h, :n], km[b, h, :n], bits, True)[pad:]
            v = _decoded(vc[b, h, :n], vm[b, h, :n], bits, False)[pad:]
            for j in range(h * g, h * g + g):
                s = state["q"][b, j].double() @ k.T / math.sqrt(D)
                hidden = torch.arange(pad, n, device="cuda")[None] > torch.arange(n - nq, n, device="cuda")[:, None]
                s[hidden] = -math.inf
                some = ~hidden.all(1)
                if some.any():
                    l = torch.logsumexp(s[some], 1)
                    lse[b, j, some] = l
                    out[b, some, j] = torch.exp(s[some] - l[:, None]) @ v
    return [out, lse] if _with_lse(case) else [out]
