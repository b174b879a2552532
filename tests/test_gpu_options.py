"""The patched model under the options whose kernels are windows, counter-based dropout and few-token
products: sliding layers on packed rows, adapters with dropout on MFMA (eager and replayed from HIP
graphs), and generation token by token. On the small tied Qwen2 of test_gpu_step.py."""

import pytest
import torch

from talm_amd import dropout, engaged, few_tokens, fused_mlp, fused_proj, lora, patches, qgroup, qlora_model, unpad

pytestmark = pytest.mark.gpu


def _model(seed=3, lora_dropout=0.0, **overrides):
    config = qlora_model.qwen2_config(**{**dict(
        vocab_size=1000, hidden_size=512, intermediate_size=1024, num_hidden_layers=3,
        num_attention_heads=4, num_key_value_heads=2, head_dim=128), **overrides})
    model = qlora_model.build_model(config, seed=seed, lora_dropout=lora_dropout)
    with torch.no_grad():  # adapters in mid-training: B is not zero
        for p in qlora_model.lora_parameters(model):
            if p.abs().sum() == 0:
                p.normal_(0, 0.02)
    return model


@pytest.fixture
def patched():
    engaged.reset()
    yield
    patches.unapply()
    qgroup.release()


def _grads(model, batch):
    with torch.autocast("cuda", dtype=torch.float16):
        loss = model(**batch).loss
    params = qlora_model.lora_parameters(model)
    grads = torch.autograd.grad(loss * 1024, params)
    return float(loss), [g / 1024 for g in grads]


def _near(got, want, rel):
    for a, b in zip(got, want):
        assert (a - b).norm() <= rel * b.norm(), ((a - b).norm() / b.norm()).item()


WINDOWED = dict(use_sliding_window=True, sliding_window=40, max_window_layers=1)


@pytest.mark.parametrize("path", ["block", "per_node", "masked"])
def test_sliding_layers_run_on_packed_rows(monkeypatch, patched, path):
    """A model of one full and two sliding layers against the unpatched padded step (transformers' own
    sliding mask): loss and LoRA gradients. Both sides round activations to fp16 at every layer
    boundary but sum in other orders, as in the parity run of test_gpu_step.py, whose bars (1e-3 of
    the loss) this takes; gradients within 2% (a window off by one key of 40 changes every row's
    attention by a weight of about 1/40, 2.5%, and its value)."""
    print(f"[case] sliding layers path={path}", flush=True)
    model = _model(**WINDOWED)
    batch = qlora_model.make_batch(seed=5, step=0, vocab=1000, seq=256, lo=64, hi=256)
    want_loss, want = _grads(model, batch)
    if path != "block":
        monkeypatch.setattr(fused_proj, "ATTN_BLOCK", False)
    if path == "masked":
        monkeypatch.setattr(unpad, "window_takes", lambda *a: False)
    patches.apply()
    loss, got = _grads(model, batch)
    assert engaged.RAN["unpad"] == 1 and engaged.FELL_BACK["unpad"] == 0
    assert engaged.RAN["window_attn"] == (0 if path == "masked" else 2)
    assert engaged.RAN["rows_attn"] == (2 if path == "masked" else 0)
    assert engaged.RAN["attn_block"] == (3 if path == "block" else 0)
    assert abs(loss - want_loss) <= 1e-3 * abs(want_loss)
    _near(got, want, 0.02)


def test_sinks_come_from_the_config_and_are_refused_elsewhere(monkeypatch, patched):
    """The attention block and the masked rows agree with sinks (and differ from none); a call off the
    packed rows, whose mask does not hold them, is refused."""
    model = _model(**WINDOWED, attention_sinks=4)
    batch = qlora_model.make_batch(seed=6, step=0, vocab=1000, seq=256, lo=64, hi=256)
    patches.apply()
    loss, got = _grads(model, batch)
    assert engaged.RAN["window_attn"] == 2
    monkeypatch.setattr(fused_proj, "ATTN_BLOCK", False)
    monkeypatch.setattr(unpad, "window_takes", lambda *a: False)
    masked_loss, masked = _grads(model, batch)
    assert engaged.RAN["rows_attn"] == 2
    assert abs(loss - masked_loss) <= 1e-3 * abs(masked_loss)
    _near(got, masked, 0.02)
    model.config.attention_sinks = 0
    _, without = _grads(model, batch)
    assert (without[0] - masked[0]).norm() > 0.05 * masked[0].norm()
    model.config.attention_sinks = 4
    model.eval()
    with torch.no_grad(), torch.autocast("cuda", dtype=torch.float16), pytest.raises(ValueError, match="sinks"):
        model(input_ids=batch["input_ids"])


def _fixed_key(monkeypatch, *words):
    """Every key drawn is (a copy of) one tensor, so that two runs drop the same elements."""
    key = torch.tensor(words, dtype=torch.int64, device="cuda")
    for module in (fused_proj, lora):
        monkeypatch.setattr(module, "draw_key", lambda device: key.clone())
    return key


@pytest.mark.parametrize("path", ["block", "per_node", "lora_node"])
def test_adapter_dropout_on_mfma_matches_the_ops(monkeypatch, patched, path):
    """The step with counter-based dropout on the MFMA products against the same masks through the
    node's PyTorch ops (SOLUTION_DISABLE_QKV_MFMA's path)."""
    print(f"[case] adapter dropout path={path}", flush=True)
    monkeypatch.setattr(dropout, "COUNTER", True)
    if path != "block":
        monkeypatch.setattr(fused_proj, "ATTN_BLOCK", False)
    if path == "lora_node":
        monkeypatch.setenv("SOLUTION_DISABLE_FUSED_PROJ", "1")
    model = _model(lora_dropout=0.3)
    batch = qlora_model.make_batch(seed=7, step=0, vocab=1000, seq=256, lo=64, hi=256)
    patches.apply()
    _fixed_key(monkeypatch, 1234567, 89)
    loss, got = _grads(model, batch)
    assert engaged.RAN["counter_dropout"] and engaged.RAN["qkv_mfma"] and engaged.RAN["qkv_mfma_bwd"]
    ran = engaged.RAN["qkv_mfma"]
    monkeypatch.setattr(fused_proj, "QKV_MFMA", False)
    ops_loss, ops = _grads(model, batch)
    assert engaged.RAN["qkv_mfma"] == ran
    assert abs(loss - ops_loss) <= 1e-3 * abs(ops_loss)
    # a mask that differed on some elements would be off by the square root of their share
    _near(got, ops, 0.02)
    _fixed_key(monkeypatch, 1234568, 89)
    _, other = _grads(model, batch)
    assert (other[0] - ops[0]).norm() > 0.1 * ops[0].norm()


def test_adapter_dropout_keeps_native_masks_by_default(patched):
    """Without the switch a seed gives the masks it gave: the patched step draws PyTorch's own."""
    assert not dropout.COUNTER
    model = _model(lora_dropout=0.3)
    batch = qlora_model.make_batch(seed=7, step=0, vocab=1000, seq=256, lo=64, hi=256)
    patches.apply()
    _grads(model, batch)
    assert engaged.RAN["counter_dropout"] == 0 and engaged.RAN["qkv_mfma"] == 0


def test_graphed_steps_with_dropout_and_sliding_layers(monkeypatch, patched):
    """GraphedTrainer replays a model with adapter dropout and sliding layers: a replay takes the key
    in force (here one tensor whose contents change) and equals the eager step with the same packing
    and key; with keys of the generator's own, two replays of one batch differ."""
    from talm_amd.step_graph import GraphedTrainer

    model = _model(lora_dropout=0.2, **WINDOWED)
    trainer = qlora_model.Trainer(model, steps=64, lr=0.0, weight_decay=0.0, fused_adapters=True)
    batches = [qlora_model.make_batch(seed=8, step=i, vocab=1000, seq=256, lo=64, hi=256) for i in range(4)]
    patches.apply()
    graphed = GraphedTrainer(trainer, bucket=64)
    with monkeypatch.context() as m:
        m.setattr(dropout, "COUNTER", True)
        for batch in batches[:2]:
            graphed.step(batch)  # eager warm-up
        key = _fixed_key(m, 5, 6)
        for i, batch in enumerate(batches + batches):
            key.fill_(100 + i % 3)
            loss = graphed.step(batch).clone()
            torch.cuda.synchronize()
            n = graphed.bucket_of(int(batch["attention_mask"].sum()))
            with unpad.static_tokens(n, max_pad=graphed.bucket):
                want, _ = _grads(model, batch)
            assert abs(float(loss) - want) <= 1e-6 * abs(want), i
    assert graphed.replays == 8
    graphed.close()
    graphed = GraphedTrainer(trainer, bucket=64, warm_steps=2)
    for batch in batches[:2]:
        graphed.step(batch)
    losses = {float(graphed.step(batches[0])) for _ in range(4)}
    assert len(losses) == 4, losses  # lr is 0: only the masks differ
    graphed.close()


def test_unpacked_adapter_takes_the_branch(monkeypatch, patched):
    """A LoRA layer whose base is not part of a packed layer: its branch with counter-based dropout
    against PEFT's arithmetic under the same mask, outputs and adapter gradients. fp16 roundings in
    both of the base, t, the branch and the sum: 2^-10 of the output's scale, 1% of the gradients."""
    from oracle import philox
    from talm_amd.nf4_linear import Linear4bit

    torch.manual_seed(0)
    base = Linear4bit.from_weight(torch.randn(128, 256, device="cuda") * 0.05)
    layer = lora.LoraLinear(base, 16, 32, 0.25).cuda().train()
    with torch.no_grad():
        layer.lora_B["default"].weight.normal_(0, 0.05)
    x = torch.randn(3, 11, 256, device="cuda").half()
    dy = torch.randn(3, 11, 128, device="cuda").half()
    patches.apply()
    monkeypatch.setattr(dropout, "COUNTER", True)
    key = _fixed_key(monkeypatch, 42, 43)
    params = (layer.lora_A["default"].weight, layer.lora_B["default"].weight)
    with torch.autocast("cuda", dtype=torch.float16):
        y = layer(x)
    got = torch.autograd.grad(y, params, dy)
    assert engaged.RAN["lora_branch"] == 1
    keep = torch.from_numpy(philox.keep(key.tolist(), 33, 256, 0.25)).cuda().view(3, 11, 256)
    xd = x.float() * keep * float(philox.factor(0.25))
    want = base(x).float() + 2.0 * (xd @ params[0].t()) @ params[1].t()
    assert (y.float() - want).abs().max() <= 2.0 ** -9 * want.abs().max()
    _near(got, torch.autograd.grad(want, params, dy.float()), 0.01)


# -- generation ------------------------------------------------------------------------------------

def _logits(model, ids, steps):
    """Prefill, then `steps` single tokens through the cache; the logits of every position asked."""
    outs = []
    with torch.no_grad(), torch.autocast("cuda", dtype=torch.float16):
        out = model(input_ids=ids, use_cache=True)
        outs.append(out.logits[:, -1].float())
        for i in range(steps):
            out = model(input_ids=(ids[:, i:i + 1] * 7 + 11) % 1000, past_key_values=out.past_key_values,
                        use_cache=True)
            outs.append(out.logits[:, -1].float())
    return torch.stack(outs)


@pytest.mark.parametrize("batch,adapters", [(1, True), (3, True), (2, False)])
def test_token_by_token_on_the_nf4_codes(monkeypatch, patched, batch, adapters):
    """Cached generation with the few-token products against the same patched model without them:
    logits within fp16's rounding through three layers (the bar of the parity run, 0.5%)."""
    print(f"[case] generation batch={batch} adapters={adapters}", flush=True)
    model = _model().eval()
    if not adapters:
        for layer in model.model.layers:
            for name in ("q_proj", "v_proj"):
                setattr(layer.self_attn, name, getattr(layer.self_attn, name).base_layer)
    patches.apply()
    ids = torch.randint(0, 1000, (batch, 70), device="cuda", generator=torch.Generator("cuda").manual_seed(1))
    with monkeypatch.context() as m:
        m.setattr(few_tokens, "ENABLED", False)
        want = _logits(model, ids, 5)
        assert engaged.RAN["gemv"] == 0
    qgroup.release()
    engaged.reset()
    got = _logits(model, ids, 5)
    # per layer and token: q|k|v, o, gate|up, down
    assert engaged.RAN["gemv"] == 5 * 3 * 4
    assert engaged.RAN["group"] == 3  # the prefill's layers alone were dequantized
    assert (got - want).norm() <= 5e-3 * want.norm()


def test_few_tokens_leave_training_and_long_calls_alone(patched):
    model = _model()
    batch = qlora_model.make_batch(seed=9, step=0, vocab=1000, batch=1, seq=24, lo=20, hi=24)
    patches.apply()
    _grads(model, batch)
    assert engaged.RAN["gemv"] == 0
    ids = torch.randint(0, 1000, (1, qgroup.GEMV_TOKENS + 1), device="cuda")
    with torch.no_grad(), torch.autocast("cuda", dtype=torch.float16):
        model(input_ids=ids)
        assert engaged.RAN["gemv"] == 0
        model(input_ids=ids[:, :-1])
        assert engaged.RAN["gemv"] > 0


def test_a_failing_product_turns_itself_off(monkeypatch, patched):
    """The convention of every fast path: one failure, one line, the call reruns without it."""
    from talm_amd import state

    model = _model().eval()
    patches.apply()
    ids = torch.randint(0, 1000, (1, 70), device="cuda")
    with monkeypatch.context() as m:
        m.setattr(few_tokens, "ENABLED", False)
        want = _logits(model, ids, 2)
    monkeypatch.setattr(state, "STRICT", False)
    monkeypatch.setattr(qgroup.LayerGroup, "nf4_gemv", lambda *a: (_ for _ in ()).throw(RuntimeError("injected")))
    try:
        got = _logits(model, ids, 2)
        assert list(state.DISABLED) == ["gemv"]
        assert (got - want).norm() <= 5e-3 * want.norm()
    finally:
        state.DISABLED.clear()


def test_mlp_alone(patched):
    model = _model().eval()
    patches.apply()
    mlp = model.model.layers[1].mlp
    x = torch.randn(2, 3, 512, device="cuda").half()
    with torch.no_grad(), torch.autocast("cuda", dtype=torch.float16):
        model(input_ids=torch.zeros(1, 40, dtype=torch.int64, device="cuda"))  # packs the layers
        group = model.model.layers[1]._solution_layer_group
        y = fused_mlp.fused_mlp_forward(mlp, x)
    with torch.no_grad():
        gate, up = (group.dequantize_one(i).double() for i in (4, 5))
        a = x.double()
        want = (torch.nn.functional.silu(a @ gate.T) * (a @ up.T)) @ group.dequantize_one(6).double().T
    # gate, up, the activation and y rounded: a few 2^-11 of the magnitudes
    assert y.shape == x.shape and (y.double() - want).norm() <= 4 * 2.0 ** -11 * want.norm()


def test_few_tokens_of_a_layer_the_codes_do_not_serve_keep_the_mlp_node(monkeypatch, patched):
    """A group that the few-token products refuse (other NF4 blocks, other widths): the MLP stays the node
    that longer calls run, the results too."""
    model = _model(hidden_size=1024, intermediate_size=4096, num_hidden_layers=2).eval()
    patches.apply()
    ids = torch.randint(0, 1000, (1, 8), device="cuda")

    def run():
        engaged.reset()
        with torch.no_grad(), torch.autocast("cuda", dtype=torch.float16):
            logits = model(input_ids=ids).logits
        return logits, {name: engaged.RAN[name] for name in ("fused_mlp", "mlp_block", "gemv")}
    with monkeypatch.context() as m:
        m.setattr(few_tokens, "ENABLED", False)
        want, ran = run()
    assert ran["fused_mlp"] == 2 and ran["gemv"] == 0
    monkeypatch.setattr(qgroup.LayerGroup, "gemv_ok", lambda *a: False)
    got, now = run()
    assert now == ran and torch.equal(got, want)

def test_rows_that_share_memory_stay_on_the_codes(patched):
    """x given as an expanded row, or as overlapping ones: copied, not refused."""
    model = _model().eval()
    patches.apply()
    with torch.no_grad(), torch.autocast("cuda", dtype=torch.float16):
        model(input_ids=torch.zeros(1, 40, dtype=torch.int64, device="cuda"))  # packs the layers
        flat = torch.randn(1024, device="cuda").half()
        for x in (flat[:512].expand(4, 512), flat[:512].expand(2, 3, 512), flat.as_strided((4, 512), (8, 1))):
            ran = engaged.RAN["gemv"]
            got = model.model.layers[0].self_attn.o_proj(x)
            assert engaged.RAN["gemv"] == ran + 1
            assert torch.equal(got, model.model.layers[0].self_attn.o_proj(x.contiguous()))

def test_unpacked_adapter_on_a_base_of_another_type(monkeypatch, patched):
    """A base that answers in float32 (it leaves autocast): run once, its output kept in that type."""
    calls = []

    class Base(torch.nn.Linear):
        def forward(self, x):
            calls.append(1)
            with torch.autocast("cuda", enabled=False):
                return super().forward(x.float())

    torch.manual_seed(0)
    layer = lora.LoraLinear(Base(256, 128, device="cuda"), 16, 32, 0.25).cuda().train()
    with torch.no_grad():
        layer.lora_B["default"].weight.normal_(0, 0.05)
    x = torch.randn(9, 256, device="cuda").half()
    patches.apply()
    monkeypatch.setattr(dropout, "COUNTER", True)
    key = _fixed_key(monkeypatch, 42, 43)
    with torch.autocast("cuda", dtype=torch.float16):
        y = layer(x)
    assert len(calls) == 1 and y.dtype == torch.float32 and engaged.RAN["lora_branch"] == 1
    params = (layer.lora_A["default"].weight, layer.lora_B["default"].weight)
    branch = lora.adapter_branch(x, *params, 2.0, 0.25, key)
    assert torch.equal(y, layer.base_layer(x) + branch)


def test_adapter_branch_reads_its_weights_as_they_are(patched):
    """In a patched process, whose parameters have shared fp16 copies: weights that are views of other
    memory, that change through .data, and that are temporaries."""
    patches.apply()
    g = torch.Generator("cuda").manual_seed(3)
    x = torch.randn(12, 64, device="cuda", generator=g).half()
    key = torch.tensor([3, 4], device="cuda")
    a = torch.randn(16, 64, device="cuda", generator=g)
    b = torch.randn(32, 16, device="cuda", generator=g)

    def check(a, b):
        want = lora.adapter_branch(x, a.half().contiguous(), b.half().contiguous(), 2.0, 0.3, key)
        assert torch.equal(lora.adapter_branch(x, a, b, 2.0, 0.3, key), want)
        return want
    for views in ((a, b), (a.t().contiguous().t(), b.t().contiguous().t()), (a[:1].expand(16, 64), b[:1].expand(32, 16)),
                  (torch.randn(32, 128, device="cuda")[::2, ::2], b)):
        first = check(*views)
        views[0].data.mul_(2.0) if views[0].stride(0) else views[0][:1].data.mul_(2.0)
        second = check(*views)
        assert not torch.equal(first, second)
    for i in range(3):
        check(a * i, b + i)


@pytest.mark.parametrize("batch", [1, 9])
def test_adapters_of_single_projections_join_their_products(monkeypatch, patched, batch):
    """Generation with adapters on o_proj and down_proj beside q's and v's: each is added by its projection's
    product. Logits against the same patched model without the few-token products, as above."""
    print(f"[case] generation with adapters on o and down, batch={batch}", flush=True)
    torch.manual_seed(4)
    model = _model()
    for layer in model.model.layers:
        for owner, name in ((layer.self_attn, "o_proj"), (layer.mlp, "down_proj")):
            wrapped = lora.LoraLinear(getattr(owner, name), 16, 32)
            torch.nn.init.normal_(wrapped.lora_B["default"].weight, 0, 0.02)
            setattr(owner, name, wrapped)
    model.eval()
    patches.apply()
    ids = torch.randint(0, 1000, (batch, 70), device="cuda", generator=torch.Generator("cuda").manual_seed(1))
    with monkeypatch.context() as m:
        m.setattr(few_tokens, "ENABLED", False)
        want = _logits(model, ids, 3)
        assert engaged.RAN["gemv"] == 0
        for layer in model.model.layers:  # the adapters matter
            layer.mlp.down_proj.scaling["default"] = 0.0
        without = _logits(model, ids, 3)
        for layer in model.model.layers:
            layer.mlp.down_proj.scaling["default"] = 2.0
    assert (without - want).norm() > 0.05 * want.norm()
    engaged.reset()
    got = _logits(model, ids, 3)
    # per layer and token: q|k|v, o, gate, up, down
    assert engaged.RAN["gemv"] == 3 * 3 * 5
    assert (got - want).norm() <= 5e-3 * want.norm()
