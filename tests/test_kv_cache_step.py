"""A QuantizedCache's step through a model on the CPU, its layers' operators in plain PyTorch (float32 rows and
no pages): who is answered from the cache, and what the step demands of the layers."""

import pytest
import torch
from transformers import LlamaConfig, LlamaForCausalLM, Qwen2Config, Qwen2ForCausalLM

from talm_amd import kv_cache, patches, unpad


class PlainLayer(kv_cache.CacheLayer):
    """CacheLayer's write and attention: each sequence's rows in a list."""

    def write(self, key, value, bounds, past, max_new, query=None, rope=None):
        assert query is None and rope is None
        if not hasattr(self, "kept"):
            self.kept = {}
        for b, ((lo, hi), n) in enumerate(zip(bounds.tolist(), past.tolist())):
            rows = torch.stack((key[0, :, lo:hi], value[0, :, lo:hi])).float()
            self.kept[b] = torch.cat((self.kept[b][:, :, :n], rows), 2) if n else rows

    def attention(self, query, bounds, past, max_new, max_len, scale, window=None, sinks=0):
        heads, n, d = query.shape[1:]
        out = torch.zeros(n, heads, d, dtype=query.dtype)
        for b, ((lo, hi), p) in enumerate(zip(bounds.tolist(), past.tolist())):
            k, v = (t.repeat_interleave(heads // t.shape[0], 0) for t in self.kept[b])
            place, at = p + torch.arange(hi - lo)[:, None], torch.arange(k.shape[1])[None]
            s = (query[0, :, lo:hi].float() @ k.transpose(1, 2) * scale).masked_fill(at > place, -torch.inf)
            out[lo:hi] = (s.softmax(-1) @ v).transpose(0, 1).to(query.dtype)
        return out[None]


@pytest.fixture
def patched(monkeypatch):
    monkeypatch.setattr(kv_cache, "CacheLayer", PlainLayer)
    monkeypatch.setattr(torch.Tensor, "pin_memory", lambda self: self)
    unpad.patch_sdpa_rows()
    kv_cache.patch_qwen2_cache()
    yield
    patches.unapply()


SIZES = dict(vocab_size=50, hidden_size=128, intermediate_size=64, num_hidden_layers=2, num_attention_heads=2,
             num_key_value_heads=1, attn_implementation="sdpa")


def _qwen2(seed=0, **more):
    torch.manual_seed(seed)
    return Qwen2ForCausalLM(Qwen2Config(**{**SIZES, **more})).eval()


def _cache(model, batch=2, capacity=64, **more):
    return kv_cache.QuantizedCache(model.config, batch, capacity, device="cpu", **{"dtype": torch.float16, **more})


def _ids(batch, n, seed=1):
    return torch.randint(0, 50, (batch, n), generator=torch.Generator().manual_seed(seed))


@torch.no_grad()
def _answers(model, cache, pieces=(5, 1, 3)):
    ids, at, out = _ids(cache.batch, sum(pieces)), 0, []
    for n in pieces:
        out.append(model(input_ids=ids[:, at:at + n], past_key_values=cache, use_cache=True).logits)
        at += n
    return torch.cat(out, 1)


def test_a_step_answers_as_the_whole_text(patched):
    """What the tests below rely on: fp16 keys, values and queries against fp32 ones (u = 2^-11 a number)."""
    model = _qwen2()
    with torch.no_grad():
        want = model(input_ids=_ids(2, 9)).logits
    got = _answers(model, _cache(model))
    assert (got - want).norm() <= 2e-3 * want.norm()


def _other_models():
    torch.manual_seed(7)
    yield "another class", LlamaForCausalLM(LlamaConfig(**SIZES)).eval()
    yield "the same class", _qwen2(8, num_hidden_layers=3)


@pytest.mark.parametrize("which", [0, 1])
def test_other_models_calls_are_their_own(patched, which):
    """A second model that runs inside of a layer's call, as a probe or a guard does, with fewer rows."""
    name, probe = list(_other_models())[which]
    model = _qwen2()
    ids = _ids(1, 4, seed=5)
    with torch.no_grad():
        want = probe(input_ids=ids).logits
    alone = _answers(model, _cache(model))
    seen = []

    def hook(module, args, output):
        seen.append(probe(input_ids=ids).logits)

    handles = [layer.mlp.register_forward_hook(hook) for layer in model.model.layers]
    got = _answers(model, _cache(model))
    for h in handles:
        h.remove()
    assert len(seen) == 6 and all(torch.equal(x, want) for x in seen), name
    assert torch.equal(got, alone)


def test_other_models_with_a_cache_of_their_own(patched):
    """And one that answers from a cache of its own, step by step beside the outer one."""
    model, probe = _qwen2(), _qwen2(8, num_hidden_layers=3)
    alone, want = _answers(model, _cache(model)), _answers(probe, _cache(probe), (5, 1))
    inner, ids, seen = _cache(probe), _ids(2, 6), []

    def hook(module, args, output):
        if len(seen) < 2:
            n = inner.columns
            seen.append(probe(input_ids=ids[:, n:n + (5 if n == 0 else 1)], past_key_values=inner, use_cache=True).logits)

    model.model.layers[0].mlp.register_forward_hook(hook)
    assert torch.equal(_answers(model, _cache(model)), alone)
    assert torch.equal(torch.cat(seen, 1), want)


def test_attention_of_other_keys_than_the_caches_is_refused(patched, monkeypatch):
    """A layer whose attention is not of the keys that the cache returned to it would answer from the new tokens
    alone: the call fails, and reset() empties the cache."""
    model = _qwen2()
    cache, update = _cache(model), kv_cache.QuantizedCache.update
    want = _answers(model, _cache(model))
    with monkeypatch.context() as m:
        m.setattr(kv_cache.QuantizedCache, "update", lambda *args: tuple(x.float() for x in update(*args)))
        with pytest.raises(RuntimeError, match="attention"):
            _answers(model, cache)
    with pytest.raises(RuntimeError, match="reset"):
        _answers(model, cache)
    cache.reset()
    assert torch.equal(_answers(model, cache), want)


@pytest.mark.parametrize("layers", [(0, 1), (1,)])
def test_layers_that_leave_the_cache_out_are_refused(patched, layers):
    """transformers takes the cache from a layer that is checkpointed: its tokens would be missing from then on."""
    model = _qwen2()
    cache, want = _cache(model), _answers(model, _cache(model))
    for i in layers:
        layer = model.model.layers[i]
        layer.training, layer.gradient_checkpointing = True, True
        layer._gradient_checkpointing_func = lambda f, *args: f(*args)
    with pytest.raises(RuntimeError, match="layers"):
        _answers(model, cache)
    for layer in model.model.layers:
        layer.training = False
    with pytest.raises(RuntimeError, match="reset"):
        _answers(model, cache)
    cache.reset()
    assert torch.equal(_answers(model, cache), want)


def test_layers_that_write_twice_are_refused(patched):
    """The same tokens again would meet an open block that holds them already."""
    model = _qwen2()
    layer = model.model.layers[0]
    forward = layer.forward

    def twice(*args, **kwargs):
        forward(*args, **kwargs)
        return forward(*args, **kwargs)

    layer.forward = twice
    with pytest.raises(RuntimeError, match="layer 0"):
        _answers(model, _cache(model))


@pytest.mark.parametrize("model_type,held", [
    (torch.float16, torch.float16), (torch.bfloat16, torch.bfloat16), (torch.float32, torch.bfloat16)])
def test_a_cache_is_of_the_models_type(patched, model_type, held):
    """Unless it is named: of the first call's keys, and bfloat16 for float32 ones, whose range it has."""
    model = _qwen2().to(model_type)
    cache = _cache(model, dtype=None)
    assert cache.dtype is None
    got = _answers(model, cache)
    assert cache.dtype is held and all(layer.tail.dtype is held for layer in cache.cache_layers)
    assert torch.equal(got, _answers(model, _cache(model, dtype=held)))
    other = torch.bfloat16 if held is torch.float16 else torch.float16
    model.to(other)
    with pytest.raises(ValueError, match="dtype"), torch.no_grad():
        model(input_ids=_ids(2, 1), past_key_values=cache, use_cache=True)
    cache.reset()
    _answers(model, cache)
    assert cache.dtype is other


def test_autocast_names_the_type_of_float32_keys(patched):
    model, cache = _qwen2(), None
    for held in (torch.float16, torch.bfloat16):
        cache = _cache(model, dtype=None)
        with torch.autocast("cpu", dtype=held):
            _answers(model, cache)
        assert cache.dtype is held


@pytest.mark.parametrize("model_type", [torch.bfloat16, torch.float32])
def test_keys_past_fp16s_range_are_held(patched, model_type):
    model = _qwen2().to(model_type)
    with torch.no_grad():
        for layer in model.model.layers:
            layer.self_attn.k_proj.bias[3] = 1e5
            layer.self_attn.v_proj.bias[5] = -2e5
        want = model(input_ids=_ids(2, 9)).logits
    got = _answers(model, _cache(model, dtype=None))
    # loud biases make the softmax one of few keys: only that nothing is infinite, and the values' size
    assert got.isfinite().all() and 0.5 < got.norm() / want.norm() < 2


def test_types_that_are_not_held(patched):
    for bad in (torch.float32, torch.float64, torch.int8):
        with pytest.raises(ValueError, match="float16"):
            _cache(_qwen2(), dtype=bad)
