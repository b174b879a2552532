"""A patched Qwen2 that answers from the 8-bit cache (kv_cache.QuantizedCache), against the same patched
model on a plain cache that holds what the 8-bit one should: every sequence's complete blocks of 64 tokens
rounded, the others in 16 bits. Both sides round activations to fp16 at every layer boundary but sum
in other orders: logits within the bar of the generation tests, 0.5%."""

import pytest
import torch
from transformers import DynamicCache, Qwen2ForCausalLM

from talm_amd import engaged, few_tokens, patches, qgroup, qlora_model, state
from talm_amd.kv_cache import QuantizedCache

pytestmark = pytest.mark.gpu


def _model(seed=3, **overrides):
    config = qlora_model.qwen2_config(**{**dict(
        vocab_size=1000, hidden_size=512, intermediate_size=1024, num_hidden_layers=3,
        num_attention_heads=4, num_key_value_heads=2, head_dim=128), **overrides})
    model = qlora_model.build_model(config, seed=seed)
    with torch.no_grad():
        for p in qlora_model.lora_parameters(model):
            if p.abs().sum() == 0:
                p.normal_(0, 0.02)
    return model.eval()


@pytest.fixture
def patched():
    engaged.reset()
    yield
    patches.unapply()
    qgroup.release()


def _held(x):
    """[H, T, D] tokens of one sequence as the 8-bit cache holds them."""
    x = x.clone()
    for lo in range(0, x.shape[1] // 64 * 64, 64):
        block = x[:, lo:lo + 64].float()
        share, power = torch.frexp(block.abs().amax((1, 2)))
        scale = torch.ldexp(torch.ones(()), torch.where(share <= 0.875, power - 9, power - 8).cpu()).to(x.device)
        scale = scale[:, None, None]
        x[:, lo:lo + 64] = ((block / scale).to(torch.float8_e4m3fn).float() * scale).to(x.dtype)
    return x


class Plain(DynamicCache):
    """transformers' cache, whose layers answer with every sequence's tokens as they are held. A first
    call's own keys and values are not rounded."""

    def __init__(self, rounded_at_first=False):
        super().__init__()
        self.mask, self.rounded_at_first = None, rounded_at_first

    def update(self, key, value, layer_idx, *args, **kwargs):
        first = self.get_seq_length(layer_idx) == 0
        out = super().update(key.half(), value.half(), layer_idx, *args, **kwargs)
        if first and not self.rounded_at_first:
            return out
        held = []
        for x in out:
            x = x.clone()
            for b in range(x.shape[0]):
                at = self.mask[b, :x.shape[2]].nonzero().flatten()
                x[b][:, at] = _held(x[b][:, at])
            held.append(x)
        return tuple(held)


def _answer(model, cache, ids, mask, pieces, plain=False):
    """The prompt, then further pieces of given lengths; the logits of every piece's last tokens."""
    outs, at = [], 0
    batch, device = ids.shape[0], ids.device
    with torch.no_grad(), torch.autocast("cuda", dtype=torch.float16):
        for n in pieces:
            seen = torch.cat((mask, torch.ones(batch, at + n - mask.shape[1], dtype=mask.dtype, device=device)), 1) \
                if at + n > mask.shape[1] else mask[:, :at + n]
            places = (seen.cumsum(1) - 1).clamp_min(0)[:, at:at + n]
            if plain:
                cache.mask = seen
            out = model(input_ids=ids[:, at:at + n], attention_mask=seen, position_ids=places, past_key_values=cache,
                        use_cache=True)
            outs.append(out.logits[:, -1].float())
            at += n
    return torch.stack(outs)


def _ids(batch, total, seed=1):
    return torch.randint(0, 1000, (batch, total), device="cuda", generator=torch.Generator("cuda").manual_seed(seed))


def _mask(batch, prompt, pads):
    mask = torch.ones(batch, prompt, dtype=torch.int64, device="cuda")
    for b, n in enumerate(pads):
        mask[b, :n] = 0
    return mask


def _near(got, want):
    worst = ((got - want).norm(dim=-1) / want.norm(dim=-1)).max().item()
    print(f"  logits off by {worst:.2e}", flush=True)
    assert worst <= 5e-3


@pytest.mark.parametrize("batch,pads", [(1, (0,)), (3, (0, 0, 0)), (4, (0, 69, 13, 64))])
@pytest.mark.parametrize("overrides", [{}, {"num_attention_heads": 8, "num_key_value_heads": 2, "head_dim": 64}])
def test_answers_are_the_plain_caches(patched, batch, pads, overrides):
    """A prompt, single tokens on the NF4 codes that complete blocks of 64, a piece through whole layers,
    a short piece; left-padded prompts among them."""
    print(f"[case] 8-bit cache batch={batch} pads={pads} {overrides}", flush=True)
    model = _model(**overrides)
    patches.apply()
    ids, mask = _ids(batch, 260), _mask(batch, 120, pads)
    pieces = [120] + [1] * 12 + [70, 5, 1, 1]
    plain = Plain(rounded_at_first=bool(overrides))  # heads of 64: the first call reads the cache too
    want = _answer(model, plain, ids, mask, pieces, plain=True)
    engaged.reset()
    cache = QuantizedCache(model.config, batch, 260)
    got = _answer(model, cache, ids, mask, pieces)
    _near(got, want)
    assert cache.lengths == [sum(pieces) - n for n in pads] and cache.get_seq_length() == sum(pieces)
    assert engaged.RAN["cache_write"] == 3 * len(pieces)
    assert engaged.RAN["cache_attn"] == 3 * (len(pieces) - (0 if overrides else 1))
    assert engaged.RAN["gemv"] > 0


def test_sequences_of_a_padded_batch_answer_as_alone(patched):
    model = _model()
    patches.apply()
    pads, pieces = (0, 40, 99), [100, 1, 1, 30, 1]
    ids, mask = _ids(3, 140), _mask(3, 100, pads)
    got = _answer(model, QuantizedCache(model.config, 3, 200), ids, mask, pieces)
    for b, n in enumerate(pads):
        alone = _answer(model, QuantizedCache(model.config, 1, 200), ids[b:b + 1, n:], _mask(1, 100 - n, (0,)),
                        [100 - n] + pieces[1:])
        _near(got[:, b], alone[:, 0])


def test_sliding_layers_with_sinks_answer(monkeypatch, patched):
    """One full and two sliding layers, sinks visible: single tokens against the whole text as one first
    call (packed rows in the window kernels), on a cache that keeps 16 bits by never completing a
    block."""
    model = _model(use_sliding_window=True, sliding_window=20, max_window_layers=1, attention_sinks=3)
    patches.apply()
    ids = _ids(1, 60)
    whole = _answer(model, QuantizedCache(model.config, 1, 63), ids, _mask(1, 60, (0,)), [60])
    steps = _answer(model, QuantizedCache(model.config, 1, 63), ids, _mask(1, 40, (0,)), [40] + [1] * 20)
    _near(steps[-1:], whole)
    model.config.attention_sinks = 0
    other = _answer(model, QuantizedCache(model.config, 1, 63), ids, _mask(1, 60, (0,)), [60])
    assert (other - whole).norm() > 5e-3 * whole.norm()


def test_generate_takes_it(patched):
    """transformers' generate, greedy, left-padded: the tokens of its own loop's logits."""
    model = _model()
    patches.apply()
    ids, mask = _ids(2, 70), _mask(2, 70, (0, 31))
    with torch.autocast("cuda", dtype=torch.float16):
        out = model.generate(input_ids=ids, attention_mask=mask, do_sample=False, max_new_tokens=9,
                             past_key_values=QuantizedCache(model.config, 2, 80), output_logits=True,
                             return_dict_in_generate=True)
    text = out.sequences
    assert text.shape == (2, 79) and torch.equal(text[:, :70], ids)
    logits = _answer(model, QuantizedCache(model.config, 2, 80), text, mask, [70] + [1] * 8)
    _near(torch.stack(out.logits).float(), logits)


def test_few_token_products_may_be_off(monkeypatch, patched):
    monkeypatch.setattr(few_tokens, "ENABLED", False)
    model = _model()
    patches.apply()
    ids, mask, pieces = _ids(2, 90), _mask(2, 70, (0, 5)), [70, 1, 1, 8]
    want = _answer(model, Plain(), ids, mask, pieces, plain=True)
    got = _answer(model, QuantizedCache(model.config, 2, 90), ids, mask, pieces)
    _near(got, want)


def test_bfloat16_caches(patched):
    """The cache's own type: keys and values arrive in fp16 and are held, and attended to, in bfloat16
    (u = 2^-8 per value and layer: a bar of 2%)."""
    model = _model()
    patches.apply()
    ids, mask, pieces = _ids(1, 100), _mask(1, 80, (0,)), [80, 1, 1, 12]
    want = _answer(model, QuantizedCache(model.config, 1, 100), ids, mask, pieces)
    got = _answer(model, QuantizedCache(model.config, 1, 100, dtype=torch.bfloat16), ids, mask, pieces)
    assert (got - want).norm() <= 0.02 * want.norm()


@pytest.mark.parametrize("held", [torch.float16, torch.bfloat16])
def test_models_of_another_type_than_the_cache(monkeypatch, patched, held):
    """Plain bfloat16 weights, no autocast: what the attention returns is of the model's type. One call, which
    attends to its own keys and values: they, the queries and the output are rounded to the cache's type
    where transformers rounds to bfloat16 (u = 2^-8 per value and layer: a bar of 2%)."""
    for fp16_only in ("swiglu", "rmsnorm", "addnorm"):
        monkeypatch.setitem(state.DISABLED, fp16_only, "a bfloat16 model")
    config = qlora_model.qwen2_config(vocab_size=1000, hidden_size=512, intermediate_size=1024, num_hidden_layers=2,
                                      num_attention_heads=4, num_key_value_heads=2, head_dim=128)
    torch.manual_seed(5)
    model = Qwen2ForCausalLM(config).to("cuda", torch.bfloat16).eval()
    patches.apply()
    ids, mask = _ids(2, 50), _mask(2, 50, (0, 7))
    with torch.no_grad():
        want = model(input_ids=ids, attention_mask=mask, past_key_values=DynamicCache(), use_cache=True).logits[:, -1]
        cache = QuantizedCache(config, 2, 60, dtype=held)
        out = model(input_ids=ids, attention_mask=mask, past_key_values=cache, use_cache=True).logits
        again = model(input_ids=ids[:, :1], past_key_values=cache, use_cache=True).logits
    assert out.dtype == again.dtype == torch.bfloat16 and again.isfinite().all()
    assert (out[:, -1] - want).float().norm() <= 0.02 * want.float().norm()


@pytest.mark.parametrize("overrides", [{}, {"num_attention_heads": 8, "num_key_value_heads": 2, "head_dim": 64}])
def test_rows_of_padding_are_finite(patched, overrides):
    """First calls and later ones, in memory that held NaN."""
    model = _model(**overrides)
    patches.apply()
    cache, ids, mask = QuantizedCache(model.config, 2, 60), _ids(2, 60), _mask(2, 40, (0, 33))
    more = torch.cat((mask, _mask(2, 10, (4, 0))), 1)
    with torch.no_grad(), torch.autocast("cuda", dtype=torch.float16):
        for n, seen in ((40, mask), (10, more)):
            junk = [torch.full((size,), float("nan"), device="cuda") for size in (1 << 12, 1 << 16, 1 << 20, 1 << 24)]
            del junk
            out = model(input_ids=ids[:, :n], attention_mask=seen, past_key_values=cache, use_cache=True).logits
            assert out.isfinite().all()
    assert cache.lengths == [46, 17]


def test_calls_that_are_refused(patched):
    model = _model()
    ids, ones = _ids(2, 40), _mask(2, 20, (0, 0))
    cache = QuantizedCache(model.config, 2, 30)

    def call(n=20, mask=ones, rows=ids, c=cache):
        with torch.no_grad(), torch.autocast("cuda", dtype=torch.float16):
            return model(input_ids=rows[:, :n], attention_mask=mask, past_key_values=c, use_cache=True)

    with pytest.raises(RuntimeError, match="outside of a patched"):
        call()
    patches.apply()
    with pytest.raises(ValueError, match="gradient"), torch.autocast("cuda", dtype=torch.float16):
        model(input_ids=ids[:, :20], past_key_values=cache, use_cache=True)
    with pytest.raises(ValueError, match="made for 2"):
        call(rows=ids[:1], mask=ones[:1])
    with pytest.raises(ValueError, match="one run"):
        call(mask=torch.tensor([[1, 0] * 10, [1] * 20], device="cuda"))
    with pytest.raises(ValueError, match="attention mask"):
        call(mask=ones[:, :19])
    with pytest.raises(ValueError, match="31 tokens"):
        call(n=31, mask=None)
    model.config._attn_implementation = "eager"
    with pytest.raises(ValueError, match="sdpa"):
        call()
    model.config._attn_implementation = "sdpa"
    assert cache.lengths == [0, 0]  # nothing of them was kept
    call()
    call(n=10, mask=None)
    with pytest.raises(ValueError, match="31 tokens"):
        call(n=1, mask=None)
    assert cache.lengths == [30, 30]
    for name in ("reorder_cache", "crop", "batch_repeat_interleave", "batch_select_indices"):
        with pytest.raises(NotImplementedError):
            getattr(cache, name)(torch.zeros(2, dtype=torch.int64))
    cache.reset()
    inner = model.model.layers[1].mlp.forward

    def broken(x):
        raise KeyError("a layer fails")

    model.model.layers[1].mlp.forward = broken
    with pytest.raises(KeyError):
        call()
    model.model.layers[1].mlp.forward = inner
    with pytest.raises(RuntimeError, match="reset"):
        call()
    cache.reset()
    want = call(c=QuantizedCache(model.config, 2, 30)).logits
    assert torch.equal(call().logits, want)
