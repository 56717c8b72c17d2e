"""The quantised transformers cache under a small random Llama: its layers against
the rows they stand for, the attention hook on codes against the same cache read
back, padding, beams, growth, and the press hooks' read and write.

Tolerance of the logits: both sides attend to the same cached values; the hook
rounds P and the values to f16 where the other rounds them to bf16, and each
layer's bf16 outputs may differ in the last place (2^-8): over two layers the
logits agree to 2^-5 of their largest."""

import pytest
import torch

pytestmark = pytest.mark.gpu


def _dev():
    if not torch.cuda.is_available():
        pytest.skip("no CUDA device")
    return torch.device("cuda", 0)


def _model(dev, impl):
    from core_b200 import attention
    from transformers import LlamaConfig, LlamaForCausalLM
    attention.register()
    torch.manual_seed(0)
    cfg = LlamaConfig(vocab_size=97, hidden_size=512, intermediate_size=256, num_hidden_layers=2,
                      num_attention_heads=4, num_key_value_heads=2, head_dim=128,
                      max_position_embeddings=4096, attn_implementation=impl)
    return LlamaForCausalLM(cfg).to(dev, torch.bfloat16).eval()


def _steps(model, cache, ids, mask=None, pieces=(1,) * 6):
    """Logits of the tokens behind the prompt, fed in pieces."""
    out, at = [], ids.shape[1] - sum(pieces)
    with torch.no_grad():
        model(ids[:, :at], past_key_values=cache, attention_mask=None if mask is None else mask[:, :at])
        for n in pieces:
            r = model(ids[:, at:at + n], past_key_values=cache,
                      attention_mask=None if mask is None else mask[:, :at + n])
            out.append(r.logits)
            at += n
    return torch.cat(out, 1).float()


@pytest.mark.parametrize("bits,group", [(4, 64), (8, 32)])
@pytest.mark.parametrize("pieces", [(1,) * 6, (5, 1, 40, 1)])
def test_codes_against_rows_read_back(bits, group, pieces):
    from core_b200.hf_cache import QuantizedCacheLayer, quantized_cache
    dev = _dev()
    ids = torch.randint(0, 97, (2, 300), generator=torch.Generator().manual_seed(1)).to(dev)
    model = _model(dev, "core_b200")
    cache = quantized_cache(model.config, bits=bits, group=group)
    assert isinstance(cache.layers[0], QuantizedCacheLayer) and cache.layers[0].by_codes
    a = _steps(model, cache, ids, pieces=pieces)
    assert cache.get_seq_length() == 300
    ref = _model(dev, "sdpa")
    back = quantized_cache(ref.config, bits=bits, group=group)
    assert not back.layers[0].by_codes
    b = _steps(ref, back, ids, pieces=pieces)
    assert (a - b).abs().max() <= 2 ** -5 * b.abs().max()


def test_left_padding():
    from core_b200.hf_cache import quantized_cache
    dev = _dev()
    ids = torch.randint(0, 97, (3, 130), generator=torch.Generator().manual_seed(2)).to(dev)
    mask = torch.ones(3, 130, dtype=torch.long, device=dev)
    mask[1, :50] = 0
    mask[2, :7] = 0
    a = _steps(_model(dev, "core_b200"), quantized_cache(_model(dev, "core_b200").config), ids, mask)
    ref = _model(dev, "sdpa")
    b = _steps(ref, quantized_cache(ref.config), ids, mask)
    assert (a - b).abs().max() <= 2 ** -5 * b.abs().max()


def test_generate_and_layer_rows():
    """generate() with beams runs through reorder_cache; a layer's rows stay within
    half a step of what was written."""
    from core_b200.hf_cache import quantized_cache
    dev = _dev()
    model = _model(dev, "core_b200")
    ids = torch.randint(0, 97, (2, 40), generator=torch.Generator().manual_seed(3)).to(dev)
    cache = quantized_cache(model.config, bits=8, group=32)
    out = model.generate(ids, past_key_values=cache, max_new_tokens=12, num_beams=2, do_sample=False,
                         pad_token_id=0, eos_token_id=None)
    assert out.shape == (2, 52)
    layer = cache.layers[0]
    assert layer.kv.batch == 4 and layer.get_seq_length() == 51
    k, v = layer.read_rows()
    assert k.shape == (4, 2, 51, 128) and k.dtype == torch.bfloat16 and torch.isfinite(k.float()).all()
    layer.crop(20)
    assert layer.get_seq_length() == 20
    assert torch.equal(layer.read_rows()[0], k[:, :, :20])
    layer.batch_select_indices(torch.tensor([2, 0]))
    assert torch.equal(layer.read_rows()[1], v[[2, 0], :, :20])
    layer.batch_repeat_interleave(2)
    assert torch.equal(layer.read_rows()[1], v[[2, 2, 0, 0], :, :20])


def test_growth_keeps_the_rows():
    from core_b200.kvcache import QuantizedKV
    dev = _dev()
    c = QuantizedKV.empty(2, 2, 128, bits=4, group=32, device=dev)
    k = torch.randn(2, 2, 300, 128, device=dev, dtype=torch.bfloat16)
    c.append(k[:, :, :100], -k[:, :, :100])
    before = c.read()
    c.reserve(1000)
    assert c.capacity == 1024 and c.max_length == 100 and c.lengths.tolist() == [100, 100]
    assert all(torch.equal(x, y) for x, y in zip(before, c.read()))
    c.append(k[:, :, 100:], -k[:, :, 100:])
    whole = QuantizedKV.empty(2, 2, 300, bits=4, group=32, device=dev)
    whole.append(k, -k)
    assert all(torch.equal(x, y) for x, y in zip(whole.read(), c.read()))


def test_press_hooks_read_and_write_rows():
    from core_b200 import press
    from core_b200.hf_cache import quantized_cache
    dev = _dev()
    model = _model(dev, "core_b200")
    cache = quantized_cache(model.config)
    ids = torch.randint(0, 97, (1, 200), generator=torch.Generator().manual_seed(4)).to(dev)
    with torch.no_grad():
        model(ids, past_key_values=cache)
    k, v = press.read_cache_layer(cache, 1)
    assert k.shape == (1, 2, 200, 128)
    keep = torch.arange(0, 200, 3, device=dev)
    press.write_cache_layer(cache, 1, k[:, :, keep], v[:, :, keep])
    assert cache.layers[1].get_seq_length() == len(keep)
    k2, v2 = press.read_cache_layer(cache, 1)
    # re-quantising rows that were read back as bf16 moves them by at most that
    # rounding and the rounding of their own grid: a step is 1/15 of a group's range
    step = (k[:, :, keep].float().unflatten(-1, (2, 64)).amax(-1) - k[:, :, keep].float().unflatten(-1, (2, 64)).amin(-1)) / 15
    err = (k2 - k[:, :, keep]).float().abs().unflatten(-1, (2, 64)).amax(-1)
    assert (err <= 0.51 * step + 2 ** -7 * k.float().abs().max()).all()


def test_another_attention_on_codes_is_loud():
    """A cache made for the hook, handed to an attention that does not know it."""
    from core_b200.hf_cache import quantized_cache
    dev = _dev()
    cache = quantized_cache(_model(dev, "core_b200").config)
    ids = torch.randint(0, 97, (1, 30), generator=torch.Generator().manual_seed(5)).to(dev)
    assert _steps(_model(dev, "sdpa"), cache, ids, pieces=(1,)).isnan().all()


def test_refuses_other_head_dims():
    from core_b200.hf_cache import QuantizedCacheLayer
    dev = _dev()
    with pytest.raises(ValueError, match="head_dim"):
        QuantizedCacheLayer().update(torch.zeros(1, 1, 2, 64, device=dev), torch.zeros(1, 1, 2, 64, device=dev))
    with pytest.raises(ValueError, match="bits"):
        QuantizedCacheLayer(bits=3)


def test_prompt_under_inference_mode_decoding_under_no_grad():
    from core_b200.hf_cache import quantized_cache
    dev = _dev()
    ids = torch.randint(0, 97, (1, 60), generator=torch.Generator().manual_seed(6)).to(dev)
    model = _model(dev, "core_b200")
    want = _steps(model, quantized_cache(model.config), ids, pieces=(1, 1, 3))
    cache = quantized_cache(model.config)
    with torch.inference_mode():
        model(ids[:, :55], past_key_values=cache)
    with torch.no_grad():
        got = [model(ids[:, a:b], past_key_values=cache).logits for a, b in ((55, 56), (56, 57), (57, 60))]
        cache.crop(40)
        cache.reset()
    assert torch.equal(torch.cat(got, 1).float(), want)


def test_room_follows_the_rows():
    """A layer holds little more than its rows: after the prompt, as tokens come, and
    after a press kept a quarter; 4 bits take less than a third of bf16 throughout."""
    from core_b200.hf_cache import QuantizedCacheLayer
    dev = _dev()
    layer = QuantizedCacheLayer(bits=4, group=64)
    k = torch.randn(1, 2, 16384, 128, device=dev, dtype=torch.bfloat16)

    def check(n):
        assert layer.get_seq_length() == n
        row = 2 * 2 * (64 + 8)  # K and V of two heads: codes, scales and zeros
        assert layer.kv.nbytes <= row * (n + max(256, n // 8) + 127)

    layer.update(k, -k)
    check(16384)
    for t in range(2100):
        layer.update(k[:, :, t:t + 1], -k[:, :, t:t + 1])
    check(18484)
    rows = layer.read_rows()
    assert torch.equal(rows[0][:, :, 16384:], rows[0][:, :, :2100])
    kept = [r[:, :, ::4].contiguous() for r in rows]
    layer.write_rows(*kept)
    check(4621)
    before = layer.read_rows()
    with pytest.raises((ValueError, TypeError)):  # a refusal leaves the rows as they were
        layer.write_rows(kept[0], kept[1].double())
    assert layer.get_seq_length() == 4621 and torch.equal(layer.read_rows()[0], before[0])
    layer.update(k[:, :, :300], -k[:, :, :300])
    check(4921)


@pytest.mark.parametrize("bits,group", [(4, 64), (8, 128)])
def test_a_press_keeps_codes_as_they_are(monkeypatch, bits, group):
    """The CORE press over a model with this cache: prefill compression and the
    recompressions while decoding.  Rows read back as bf16 quantise to the codes, scales
    and zeros that they came from, so the kept rows stay bit for bit."""
    from core_b200 import attention, ops, press as P
    from core_b200.hf_cache import quantized_cache
    from helpers import HOOK_CASE, load_case
    from test_gpu_kvcache import _decode
    from transformers import LlamaConfig, LlamaForCausalLM
    dev = _dev()
    _, meta = load_case(HOOK_CASE)
    attention.register()
    torch.manual_seed(0)
    model = LlamaForCausalLM(LlamaConfig(
        vocab_size=97, hidden_size=meta["hidden"], intermediate_size=256, num_hidden_layers=2,
        num_attention_heads=meta["hq"], num_key_value_heads=meta["hkv"], head_dim=128, max_position_embeddings=4096,
        attn_implementation="core_b200")).to(dev, torch.bfloat16).eval()
    press = P.load_core_prefill_decoding_press("tests/golden/core_indexer_hook.pt", device=str(dev),
                                               compression_ratio=0.5, decoding_compression_interval=4)
    ids = torch.randint(0, 97, (1, 300), generator=torch.Generator().manual_seed(7)).to(dev)
    cache = quantized_cache(model.config, bits=bits, group=group)
    before, events = {}, []  # a layer's rows when the press reads them; what it keeps
    scorer = press.prefilling_press.base_press
    read, retain = P.read_cache_layer, scorer.retain_metadata

    def reading(c, layer):
        before[layer] = _decode(c.layers[layer].kv)
        return read(c, layer)

    def retaining(layer, keep):
        events.append((int(layer), keep[0].long().cpu()))
        return retain(layer, keep)

    monkeypatch.setattr(P, "read_cache_layer", reading)
    monkeypatch.setattr(scorer, "retain_metadata", retaining)
    press.reset_cache()
    press.begin_sequence(290)
    press.set_token_ids(ids[:, :290])
    with torch.no_grad(), press(model):
        model(ids[:, :290], past_key_values=cache, cache_position=torch.arange(290, device=dev))
        for t in range(290, 300):
            n = cache.get_seq_length()
            if events:
                assert [e[0] for e in events] == [0, 1] and n == 145
            for layer, keep in events:
                kv = cache.layers[layer].kv
                assert kv.max_length == len(keep) and kv.lengths.tolist() == [len(keep)]
                for got, want in zip(_decode(kv), before[layer]):
                    assert torch.equal(got[0, :, :len(keep)], want[0][:, keep])
            events.clear()
            pid = torch.tensor([[t]], device=dev)
            press.record_input_tokens(ids[:, t:t + 1], pid)
            model(ids[:, t:t + 1], past_key_values=cache, position_ids=pid,
                  cache_position=torch.tensor([n], device=dev))
    ops.status(dev)
    assert cache.get_seq_length() == 145 + 2  # two recompressions in ten steps, two tokens since


def test_a_press_that_drops_nothing_or_writes_in_place(monkeypatch):
    """Rows that a press returns as they were keep their codes; what it wrote into them is stored."""
    from core_b200 import press as P
    from core_b200.hf_cache import quantized_cache
    dev = _dev()
    model = _model(dev, "core_b200")
    ids = torch.randint(0, 97, (1, 50), generator=torch.Generator().manual_seed(8)).to(dev)
    before, read = {}, P.read_cache_layer

    def reading(c, layer):
        before[layer] = [t.clone() for t in c.layers[layer].kv.buffers]
        return read(c, layer)

    monkeypatch.setattr(P, "read_cache_layer", reading)

    class Nothing(P.BasePress):
        def compress(self, module, hidden_states, keys, values, attentions, kwargs):
            return keys, values

    class Halves(P.BasePress):
        def compress(self, module, hidden_states, keys, values, attentions, kwargs):
            before["rows"] = keys.clone()
            keys.mul_(0.5)
            return keys, values

    for kind in (Nothing, Halves):
        for mode in (torch.no_grad, torch.inference_mode):
            cache = quantized_cache(model.config, bits=8, group=128)
            at = torch.arange(50, device=dev)
            with mode(), kind()(model):
                model(ids, past_key_values=cache, cache_position=at)
            kv = cache.layers[1].kv
            assert kv.max_length == 50
            if kind is Halves:
                rows = before["rows"].float()
                assert (kv.read()[0].float() - 0.5 * rows).norm() < 0.1 * rows.norm()
            else:
                assert all(torch.equal(a[:, :, :50], b[:, :, :50]) for a, b in zip(kv.buffers, before[1]))
