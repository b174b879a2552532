"""A patched Qwen2 that answers from the 8-bit cache: what runs inside of its calls, which of the cache's kernels
serve them, in which types, and sliding layers over pages."""

import pytest
import torch
from transformers import LlamaConfig, LlamaForCausalLM, Qwen2ForCausalLM

from talm_amd import engaged, patches, qgroup, qlora_model, state, unpad
from talm_amd.kv_cache import QuantizedCache
from test_gpu_kv_cache_model import Plain, _answer, _ids, _mask, _model, _near

pytestmark = pytest.mark.gpu


@pytest.fixture
def patched():
    engaged.reset()
    yield
    patches.unapply()
    qgroup.release()


def test_other_models_calls_are_their_own(patched):
    """A second model, of fewer rows, that runs inside of a layer's call."""
    model = _model()
    patches.apply()
    torch.manual_seed(7)
    probe = LlamaForCausalLM(LlamaConfig(
        vocab_size=1000, hidden_size=256, intermediate_size=128, num_hidden_layers=2, num_attention_heads=2,
        num_key_value_heads=1, head_dim=128, attn_implementation="sdpa")).to("cuda", torch.float16).eval()
    few = _ids(1, 9, seed=5)
    with torch.no_grad():
        want = probe(input_ids=few).logits
    ids, mask, pieces = _ids(2, 80), _mask(2, 70, (0, 5)), [70, 1, 9]
    alone = _answer(model, QuantizedCache(model.config, 2, 80), ids, mask, pieces)
    seen = []

    def hook(module, args, output):
        with torch.autocast("cuda", enabled=False):
            seen.append(probe(input_ids=few).logits)

    handles = [layer.register_forward_hook(hook) for layer in model.model.layers]
    got = _answer(model, QuantizedCache(model.config, 2, 80), ids, mask, pieces)
    for h in handles:
        h.remove()
    assert len(seen) == 9 and all(torch.equal(x, want) for x in seen)
    assert torch.equal(got, alone)


SLIDING = dict(use_sliding_window=True, sliding_window=50, max_window_layers=1, attention_sinks=3)


@pytest.mark.parametrize("batch,pads", [(1, (0,)), (4, (0, 69, 13, 64))])
@pytest.mark.parametrize("overrides", [{}, {"num_attention_heads": 8, "num_key_value_heads": 2, "head_dim": 64}, SLIDING])
def test_few_tokens_turn_as_they_are_written(monkeypatch, patched, batch, pads, overrides):
    """Calls of few tokens behind the first go through the write that turns queries and keys: no rotary launch
    of their own, and the bits that turning them apart gives (rope_ in fp16 rounds as the write does)."""
    model = _model(**overrides)
    patches.apply()
    answer, counts = QuantizedCache.answer, []

    def counted(self, *args):
        counts.append(args[3])
        return answer(self, *args)

    monkeypatch.setattr(QuantizedCache, "answer", counted)
    ids, mask, pieces = _ids(batch, 140), _mask(batch, 120, pads), [120, 1, 1, 5, 3, 1]
    got = _answer(model, QuantizedCache(model.config, batch, 140), ids, mask, pieces)
    assert counts == [0, 1, 2] * 5
    rotary = engaged.RAN["rope"]
    monkeypatch.setattr(QuantizedCache, "takes", lambda *args: False)
    want = _answer(model, QuantizedCache(model.config, batch, 140), ids, mask, pieces)
    assert torch.equal(got, want) and len(counts) == 15
    assert engaged.RAN["rope"] - rotary == rotary + 15  # the first call's stays


def test_few_tokens_refuse_dropout_of_attention_weights(patched):
    model = _model(attention_dropout=0.1)
    patches.apply()
    cache, ids, mask = QuantizedCache(model.config, 2, 30), _ids(2, 21), _mask(2, 20, (0, 0))
    _answer(model, cache, ids, mask, [20])
    for layer in model.model.layers:
        layer.self_attn.training = True
    with torch.no_grad(), torch.autocast("cuda", dtype=torch.float16), pytest.raises(ValueError, match="dropout"):
        model(input_ids=ids[:, 20:], past_key_values=cache, use_cache=True)


def test_a_bfloat16_model_is_held_in_bfloat16(monkeypatch, patched):
    """Keys and values past fp16's largest number, in a first call, single tokens, a completed page and a piece."""
    for fp16_only in ("swiglu", "rmsnorm", "addnorm"):
        monkeypatch.setitem(state.DISABLED, fp16_only, "a bfloat16 model")
    config = qlora_model.qwen2_config(vocab_size=1000, hidden_size=512, intermediate_size=1024, num_hidden_layers=2,
                                      num_attention_heads=4, num_key_value_heads=2, head_dim=128)
    torch.manual_seed(5)
    model = Qwen2ForCausalLM(config).to("cuda", torch.bfloat16).eval()
    with torch.no_grad():
        for layer in model.model.layers:
            layer.self_attn.k_proj.bias[3] = 1e5
            layer.self_attn.v_proj.bias[5] = -2e5
    patches.apply()
    ids, cache = _ids(2, 80), QuantizedCache(config, 2, 80)
    at = 0
    with torch.no_grad():
        for n in (60, 1, 9, 10):
            out = model(input_ids=ids[:, at:at + n], past_key_values=cache, use_cache=True).logits
            assert out.isfinite().all() and out.dtype == torch.bfloat16
            at += n
    assert cache.dtype is torch.bfloat16
    assert all(layer.tail.dtype is torch.bfloat16 for layer in cache.cache_layers)


PIECES = [70, 1, 1, 12]


def test_first_calls_are_counted(patched):
    model = _model()
    patches.apply()
    _answer(model, QuantizedCache(model.config, 2, 90), _ids(2, 90), _mask(2, 70, (0, 5)), PIECES)
    assert engaged.RAN["varlen_attn"] == 3 and engaged.RAN["cache_attn"] == 9


@pytest.mark.parametrize("overrides", [{}, SLIDING])
def test_first_calls_without_the_packed_rows_kernels(monkeypatch, patched, overrides):
    """Switched off, or failing: the first call reads the cache as the later ones do, and the cache stays whole."""
    model = _model(**overrides)
    patches.apply()
    ids, mask = _ids(2, 90), _mask(2, 70, (0, 5))
    with monkeypatch.context() as m:
        m.setattr(unpad, "window_takes", lambda *args: False)
        want = _answer(model, QuantizedCache(model.config, 2, 90), ids, mask, PIECES)
    engaged.reset()
    with monkeypatch.context() as m:
        m.setitem(state.DISABLED, "varlen_attention", "off")
        got = _answer(model, QuantizedCache(model.config, 2, 90), ids, mask, PIECES)
        assert torch.equal(got, want) and engaged.RAN["cache_attn"] == 12
        assert engaged.RAN["varlen_attn"] == engaged.RAN["window_attn"] == 0

    def broken(*args):
        raise KeyError("a kernel fails")

    monkeypatch.setattr(state, "STRICT", False)
    monkeypatch.setattr(unpad, "window_attention", broken)
    monkeypatch.setattr(unpad.VarlenAttention, "apply", broken)
    monkeypatch.delitem(state.DISABLED, "varlen_attention", raising=False)
    try:
        got = _answer(model, QuantizedCache(model.config, 2, 90), ids, mask, PIECES)
        assert "KeyError" in state.DISABLED["varlen_attention"]
    finally:
        state.DISABLED.pop("varlen_attention", None)
    assert torch.equal(got, want)
    monkeypatch.setattr(state, "STRICT", True)
    with pytest.raises(KeyError):
        _answer(model, QuantizedCache(model.config, 2, 90), ids, mask, PIECES)


@pytest.mark.parametrize("batch,pads", [(1, (0,)), (3, (0, 70, 131))])
@pytest.mark.parametrize("heads", [{}, {"num_attention_heads": 8, "num_key_value_heads": 2, "head_dim": 64}])
def test_sliding_layers_over_pages(patched, batch, pads, heads):
    """Windows and sinks over 8-bit pages: a prompt of four blocks, single tokens that complete a block, a piece and
    a short one, left-padded, against a plain cache that holds what the 8-bit one does under masks that
    say the window and the sinks."""
    model = _model(**{**SLIDING, **heads, "sliding_window": 90, "attention_sinks": 5})
    patches.apply()
    pieces = [250, 1, 1, 1, 1, 1, 1, 45, 5, 1]
    ids, mask = _ids(batch, sum(pieces)), _mask(batch, 250, pads)
    got = _answer(model, QuantizedCache(model.config, batch, 320), ids, mask, pieces)
    model.config.attention_sinks = 0  # the masks hold them
    cache, outs, at = Plain(rounded_at_first=bool(heads)), [], 0
    for n in pieces:
        seen = torch.cat((mask, mask.new_ones(batch, max(0, at + n - 250))), 1)[:, :at + n]
        place = (seen.cumsum(1) - 1).clamp_min(0)
        key, row = place[:, None], place[:, at:at + n, None]
        column = torch.arange(at + n, device="cuda")
        full = (column <= column[at:at + n, None]) & (seen[:, None] > 0)
        slide = full & ((row - key < 90) | (key < 5))
        # rows of padding look at themselves: no row is empty
        own = (column == column[at:at + n, None])[None]
        masks = {"full_attention": (full | own)[:, None], "sliding_attention": (slide | own)[:, None]}
        cache.mask = seen
        with torch.no_grad(), torch.autocast("cuda", dtype=torch.float16):
            hidden = model.model(input_ids=ids[:, at:at + n], attention_mask=masks, position_ids=place[:, at:at + n],
                                 past_key_values=cache, use_cache=True).last_hidden_state
            outs.append(model.lm_head(hidden[:, -1]).float())
        at += n
    _near(got, torch.stack(outs))
    # and the masks matter: without the sinks the answers are others
    other = _answer(model, QuantizedCache(model.config, batch, 320), ids, mask, pieces)
    assert (other - got).norm() > 5e-3 * got.norm()
