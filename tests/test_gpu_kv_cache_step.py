"""A patched Qwen2 that answers from the 8-bit cache: what runs inside of its calls, which of the cache's kernels
serve them, in which types, and sliding layers over pages."""

import pytest
import torch
from transformers import LlamaConfig, LlamaForCausalLM

from talm_amd import engaged, patches, qgroup
from talm_amd.kv_cache import QuantizedCache
from test_gpu_kv_cache_model import _answer, _ids, _mask, _model

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
