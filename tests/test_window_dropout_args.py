"""Argument checks of the sliding-window attention, the counter-based dropout with the adapters'
products, and the few-token 4-bit products: rejected before anything touches a GPU. The
generator of the oracle against its authors' known answers, the masks' counters and shares."""

import numpy as np
import pytest
import torch

from oracle import philox
from talm_amd import _lib, _ops, dropout, few_tokens, lora, patches, unpad

PTR = 1 << 12  # a fake address: never dereferenced on rejection


def _status(name, *args):
    lib = _lib.lib()
    status = getattr(lib, name)(*args)
    return status, lib.talm_last_error().decode()


@pytest.mark.parametrize("counter,key,words", [
    ((0, 0, 0, 0), (0, 0), (0x6627e8d5, 0xe169c58d, 0xbc57ac4c, 0x9b00dbd8)),
    ((0xffffffff,) * 4, (0xffffffff,) * 2, (0x408f276d, 0x41c83b0e, 0xa20bc7c6, 0x6d5451fd)),
    ((0x243f6a88, 0x85a308d3, 0x13198a2e, 0x03707344), (0xa4093822, 0x299f31d0),
     (0xd16cfe09, 0x94fdcceb, 0x5001e420, 0x24126ea1)),
])
def test_oracle_generator_has_the_published_answers(counter, key, words):
    got = philox.philox4x32([np.array([c]) for c in counter], key)
    assert tuple(int(w[0]) for w in got) == words


def test_masks_differ_by_site_and_key_and_keep_the_stated_share():
    n, p = 1 << 15, 0.25
    a = philox.keep((5, 7), 32, n // 32, p, 0)
    # 2^15 draws of probability 3/4: five standard deviations are 5 sqrt(n p (1 - p)) = 392
    for other in (philox.keep((5, 7), 32, n // 32, p, 1), philox.keep((6, 7), 32, n // 32, p, 0),
                  philox.keep((5, 8), 32, n // 32, p, 0)):
        assert abs(int(other.sum()) - 0.75 * n) < 392
        # independent masks agree on p^2 + (1 - p)^2 = 0.625 of the elements: sd = sqrt(n .625 .375)
        assert abs(int((a == other).sum()) - 0.625 * n) < 5 * np.sqrt(n * 0.625 * 0.375)
    assert philox.keep((5, 7), 3, 13, 0.0).all()
    assert philox.threshold(0.99999999) == 65535  # never everything


# (position of the argument, its bad value, a word of the message) on an otherwise good call
def _window(**bad):
    v = dict(tok=256, cu=PTR, seqs=1, longest=8, n=8, hq=2, hkv=1, d=128, scale=1.0, window=4,
             sinks=0, dtype=_lib.TALM_F16, q=PTR)
    v.update(bad)
    return _status("talm_attn_window_fwd", v["q"], v["tok"], 128, PTR, 128, 128, PTR, 128, 128,
                   v["cu"], v["seqs"], v["longest"], v["n"], v["hq"], v["hkv"], v["d"], v["scale"],
                   v["window"], v["sinks"], v["dtype"], PTR, 256, 128, PTR, None)


@pytest.mark.parametrize("bad,word", [
    ({"window": 0}, "window"), ({"window": -3}, "window"), ({"sinks": -1}, "sinks"),
    ({"dtype": _lib.TALM_F32}, "dtype"), ({"scale": 0.0}, "scale"), ({"scale": -1.0}, "scale"),
    ({"scale": float("inf")}, "scale"), ({"scale": float("nan")}, "scale"), ({"d": 64}, "head_dim"),
    ({"hq": 3, "hkv": 2}, "shape"), ({"tok": 130}, "multiples of 8"), ({"q": None}, "null"),
    ({"q": PTR + 8}, "16-byte"), ({"cu": None}, "null"),
])
def test_window_forward_rejects(bad, word):
    status, message = _window(**bad)
    assert status == _lib.TALM_EINVAL and word in message and "attn_window_fwd" in message


def test_window_backward_rejects_a_short_workspace():
    need = _ops.attn_window_bwd_workspace_bytes(4096, 2, 1, 1, 4096, 64, 4)
    assert need > _ops.attn_bwd_workspace_bytes(4096, 2)
    assert _ops.attn_window_bwd_workspace_bytes(4096, 2, 1, 1, 4096, 64, 0) == \
        _ops.attn_bwd_workspace_bytes(4096, 2)
    with pytest.raises(ValueError):
        _ops.attn_window_bwd_workspace_bytes(4096, 2, 1, 1, 4096, 0, 4)
    rows = [PTR, 256, 128]
    status, message = _status(
        "talm_attn_window_bwd", *rows, *[PTR, 128, 128] * 2, *rows, *rows, PTR, PTR, 1, 4096, 4096, 2,
        1, 128, 1.0, 64, 4, _lib.TALM_F16, None, None, 0, *rows, *[PTR, 128, 128] * 2, PTR,
        need - 512, None)
    assert status == _lib.TALM_EINVAL and "workspace" in message


def test_window_workspace_of_many_sinks_is_bounded():
    """The sinks' partials stay within 64 MiB, or one chunk where that alone is more."""
    for seqs, longest, sinks in ((1, 100000, 4), (64, 4096, 200), (64, 8192, 4), (4, 4096, 4096)):
        n = seqs * longest // 2
        extra = _ops.attn_window_bwd_workspace_bytes(n, 12, 2, seqs, longest, 64, sinks) \
            - _ops.attn_bwd_workspace_bytes(n, 12)
        one = seqs * 12 * min(sinks, longest) * 128 * 8
        assert 0 < extra <= max(64 << 20, one)


def test_window_attention_rejects_cpu_tensors_and_bad_arguments():
    q = torch.zeros(1, 2, 8, 128, dtype=torch.float16)
    cu = torch.tensor([0, 8], dtype=torch.int32)
    with pytest.raises(ValueError, match="GPU"):
        unpad.window_attention(q, q[:, :1], q[:, :1], cu, 8, 1.0, 4)


@pytest.mark.parametrize("args,word", [
    ((PTR, 8, 4, 8, _lib.TALM_F16, 1.0, PTR, 0, PTR, 8), "p 1"),
    ((PTR, 8, 4, 8, _lib.TALM_F16, -0.1, PTR, 0, PTR, 8), "p -0.1"),
    ((PTR, 8, 4, 8, _lib.TALM_F16, float("nan"), PTR, 0, PTR, 8), "p nan"),
    ((PTR, 8, 4, 8, _lib.TALM_F16, 0.5, None, 0, PTR, 8), "key"),
    ((PTR, 8, 4, 8, _lib.TALM_F16, 0.5, PTR + 4, 0, PTR, 8), "key"),
    ((PTR, 7, 4, 8, _lib.TALM_F16, 0.5, PTR, 0, PTR, 8), "shape"),
    ((PTR, 8, 4, 8, 7, 0.5, PTR, 0, PTR, 8), "dtype"),
    ((None, 8, 4, 8, _lib.TALM_F16, 0.5, PTR, 0, PTR, 8), "null"),
])
def test_dropout_rejects(args, word):
    status, message = _status("talm_dropout", *args, None)
    assert status == _lib.TALM_EINVAL and word in message


def test_dropout_of_nothing_is_no_launch():
    assert _status("talm_dropout", None, 8, 0, 8, 1, 0.5, PTR, 0, None, 8, None)[0] == _lib.TALM_OK


def test_python_entries_reject():
    x = torch.zeros(4, 64, dtype=torch.float16)
    with pytest.raises(ValueError, match="GPU"):
        dropout.dropout(x, 0.5, torch.zeros(2, dtype=torch.int64))
    with pytest.raises(ValueError, match="adapter_branch"):
        lora.adapter_branch(x, torch.zeros(16, 64), torch.zeros(32, 16), 2.0)


@pytest.mark.parametrize("k,ldx,adapters,word", [(40, 40, 1, "multiple of 32"), (64, 60, 1, "shape"),
                                                 (64, 64, 3, "shape"), (64, 66, 1, "shape")])
def test_adapter_down_rejects(k, ldx, adapters, word):
    status, message = _status("talm_lora_down_drop", PTR, ldx, 4, k, PTR, PTR, adapters, 0.5, PTR, 0,
                              1, 1.0, 1.0, PTR, PTR, 32, None)
    assert status == _lib.TALM_EINVAL and word in message


@pytest.mark.parametrize("k,cols,ws,p,word", [
    (40, 32, 1 << 20, 0.5, "multiple of 32"), (64, 12, 1 << 20, 0.5, "columns"), (64, 32, 64, 0.5, "workspace"),
    (64, 32, 1 << 20, 1.0, "p 1"), (0, 32, 1 << 20, 0.5, "shape")])
def test_adapter_branch_forward_rejects(k, cols, ws, p, word):
    status, message = _status("talm_lora_branch_fwd", PTR, 64, 4, k, cols, PTR, PTR, p, PTR, 0, 2.0, PTR,
                              PTR, PTR, ws, None)
    assert status == _lib.TALM_EINVAL and word in message


def test_adapter_backward_rejects():
    def call(hidden=64, seg=32, ws=1 << 20, dtype=_lib.TALM_F32, lo=0, da=PTR, db=PTR, a0=PTR, dx=PTR, ldd=64,
             p=0.5):
        return _status("talm_lora_bwd_drop", PTR, 64, PTR, 32, PTR, 16, PTR, 16, 4, hidden, 1, p, PTR, 0, 1, dtype,
                       lo, seg, 1.0, da, db, 0, 0, 0.0, None, None, a0, None, None, 0, dx, ldd, PTR, ws, None)
    for kwargs, word in (({"hidden": 60}, "shape"), ({"seg": 40}, "shape"), ({"ws": 64}, "workspace"),
                         ({"dtype": 2}, "dtype"), ({"lo": 8}, "shape"), ({"db": None}, "all or none"),
                         ({"da": None}, "all or none"), ({"a0": None}, "null"), ({"ldd": 60}, "shape"),
                         ({"dx": PTR + 8}, "16-byte"), ({"p": 1.5}, "p 1.5")):
        status, message = call(**kwargs)
        assert status == _lib.TALM_EINVAL and word in message, kwargs
    assert call(da=None, db=None, dx=None)[0] == _lib.TALM_OK  # nothing wanted: no launch


@pytest.mark.parametrize("tokens,cols,qblock,qblock2,word", [
    (33, 128, 64, 256, "32 tokens"), (1, 96, 64, 256, "shape"), (1, 128, 32, 256, "blocks"),
    (1, 128, 64, 200, "blocks"), (-1, 128, 64, 256, "shape"), (1, (1 << 24) + 64, 64, 256, "shape")])
def test_gemv_rejects(tokens, cols, qblock, qblock2, word):
    status, message = _status("talm_nf4_gemv", PTR, 128, tokens, PTR, PTR, PTR, PTR, PTR, 128, cols,
                              qblock, qblock2, None, None, 0, None, 0, 0, None, 0, 0, PTR, 128, None)
    assert status == _lib.TALM_EINVAL and word in message


@pytest.mark.parametrize("ldt,b0,lo0,hi0,b1,lo1,hi1", [
    (15, PTR, 0, 64, None, 0, 0), (31, PTR, 0, 64, PTR, 64, 128), (32, None, 0, 64, None, 0, 0),
    (32, PTR, -1, 64, None, 0, 0), (32, PTR, 0, 129, None, 0, 0), (32, PTR, 0, 64, PTR, 64, 200),
    (32, PTR, 0, 64, PTR, 70, 64)])
def test_gemv_rejects_adapters_outside_the_weight(ldt, b0, lo0, hi0, b1, lo1, hi1):
    status, message = _status("talm_nf4_gemv", PTR, 128, 1, PTR, PTR, PTR, PTR, PTR, 128, 128, 64, 256,
                              None, PTR, ldt, b0, lo0, hi0, b1, lo1, hi1, PTR, 128, None)
    assert status == _lib.TALM_EINVAL and "adapters" in message


@pytest.mark.parametrize("x", [
    torch.zeros(64, dtype=torch.float16).expand(4, 64), torch.zeros(64, dtype=torch.float16).expand(2, 3, 64),
    torch.zeros(256, dtype=torch.float16).as_strided((4, 64), (8, 1)),
    torch.zeros(256, dtype=torch.float16).as_strided((4, 64), (56, 1)),
    torch.zeros(4, 68, dtype=torch.float16)[:, :64], torch.zeros(4, 80, dtype=torch.float16)[:, 4:68],
    torch.zeros(64, 4, dtype=torch.float16).t(),
    torch.zeros((1 << 25) + 64, dtype=torch.float16).as_strided((2, 64), (1 << 25, 1))])
def test_gemv_rows_are_ones_the_product_reads(x):
    """Rows that share memory, are not 16-byte aligned or lie further apart than the kernel's offsets reach
    are copied; others are taken where they lie."""
    rows = few_tokens._rows(x)
    assert rows.shape == (x.numel() // 64, 64) and rows.stride(1) == 1 and torch.equal(rows, x.reshape(-1, 64))
    assert 64 <= rows.stride(0) <= 1 << 24 and rows.stride(0) % 8 == 0 and rows.data_ptr() % 16 == 0


def test_gemv_rows_of_a_wider_buffer_stay():
    wide = torch.zeros(4, 128, dtype=torch.float16)
    assert few_tokens._rows(wide[:, 64:]).data_ptr() == wide[:, 64:].data_ptr()
    assert few_tokens._rows(wide[:1, 8:72]).data_ptr() == wide[:1, 8:72].data_ptr()


def test_dropout_is_native_where_no_gpu_is_in_use(monkeypatch):
    """A process without a GPU is not asked whether it captures a graph: a patched adapter layer on the CPU
    runs its own forward."""
    monkeypatch.setattr(dropout, "COUNTER", False)
    monkeypatch.setattr(torch.cuda, "is_initialized", lambda: False)
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: pytest.fail("asked"))
    assert not dropout.counter_dropout()
    layer = lora.LoraLinear(torch.nn.Linear(64, 32), 16, 32, 0.5).eval()
    x = torch.randn(3, 64)
    want = layer(x)
    monkeypatch.setattr(lora, "install_cast_cache", lambda: None)
    lora.patch_lora()
    try:
        assert torch.equal(layer(x), want)
    finally:
        patches.unapply()


def test_adapter_branch_keeps_nothing_of_its_weights(monkeypatch):
    """The shared fp16 copies belong to a model's contiguous parameters, kept by identity until an optimizer
    steps: any tensor may be given here, a view or one that changes through .data."""
    monkeypatch.setattr(lora, "_hooks", [None])  # as in a patched process
    monkeypatch.setattr(lora.COPIES, "half", lambda w: pytest.fail("kept"))
    with pytest.raises(ValueError, match="adapter_branch"):  # the refusal of CPU operands
        lora.adapter_branch(torch.zeros(4, 64, dtype=torch.float16), torch.zeros(1, 64).expand(16, 64),
                            torch.zeros(32, 16), 2.0)


def test_windowed_calls_of_modules_without_a_config_pass(monkeypatch):
    """The "sdpa" interface is the process's: a module that names no config has no sinks, one whose config
    does is refused off the packed rows."""
    from types import SimpleNamespace

    from transformers.modeling_utils import ALL_ATTENTION_FUNCTIONS

    q = torch.randn(1, 2, 5, 16, generator=torch.Generator().manual_seed(0))
    plain = ALL_ATTENTION_FUNCTIONS["sdpa"]
    unpad.patch_sdpa_rows()
    try:
        call = ALL_ATTENTION_FUNCTIONS["sdpa"]
        assert call is not plain
        for module in (SimpleNamespace(is_causal=True), SimpleNamespace(is_causal=True, config=None),
                       SimpleNamespace(is_causal=True, config=SimpleNamespace()),
                       SimpleNamespace(is_causal=True, config=SimpleNamespace(attention_sinks=None))):
            want = plain(module, q, q, q, None, sliding_window=3)[0]
            assert torch.equal(call(module, q, q, q, None, sliding_window=3)[0], want)
        module = SimpleNamespace(is_causal=True, config=SimpleNamespace(attention_sinks=2))
        with pytest.raises(ValueError, match="sinks"):
            call(module, q, q, q, None, sliding_window=3)
    finally:
        patches.unapply()


def test_a_longest_length_beyond_the_rows_is_the_rows():
    """The kernels add rows, windows and sinks in 32 bits: none may count as longer than all rows."""
    for window in (64, 2 ** 31 - 1):
        for sinks in (0, 4, 4096, 2 ** 31 - 1):
            want = _ops.attn_window_bwd_workspace_bytes(4096, 2, 1, 1, 4096, window, sinks)
            for longest in (5000, 2 ** 31 - 1):
                assert _ops.attn_window_bwd_workspace_bytes(4096, 2, 1, 1, longest, window, sinks) == want
    with pytest.raises(ValueError):
        _ops.attn_window_bwd_workspace_bytes(1 << 30, 1, 1, 1, 4096, 64, 0)
    status, message = _window(n=1 << 30)
    assert status == _lib.TALM_EINVAL and "shape" in message


@pytest.mark.parametrize("tokens,heads,kv,seqs,longest,window,sinks", [
    (1 << 30, 1, 1, 1, 4096, 64, 4),           # rows
    (1 << 20, 2, 1, 65536, 64, 64, 4),         # sequences
    (1 << 29, 1, 1, 1, 4194177, 64, 0),        # a longer sequence than the tiles' axis holds
    (1 << 29, 1, 1, 2, 4194176, 64, 4194176),  # sinks' tiles beside the others
    (1 << 29, 64, 64, 65535, 4096, 64, 4096),  # sinks' partials
    (1 << 20, 1 << 16, 1, 1, 4096, 64, 0),     # heads
])
def test_window_workspace_of_a_call_that_would_be_rejected(tokens, heads, kv, seqs, longest, window, sinks):
    """The size query answers -1 exactly where the call says TALM_EINVAL for its sizes."""
    assert _lib.lib().talm_attn_window_bwd_workspace(tokens, heads, kv, seqs, longest, window, sinks) == -1
    rows = [PTR, 256, 128]
    status, message = _status(
        "talm_attn_window_bwd", *rows, *rows, *rows, *rows, *rows, PTR, PTR, seqs, longest, tokens, heads, kv, 128,
        1.0, window, sinks, _lib.TALM_F16, None, None, 0, *rows, *rows, *rows, PTR, 0, None)
    assert status == _lib.TALM_EINVAL and "workspace" not in message


def test_adapter_backward_of_no_tokens_wants_nothing_for_dx():
    """dx of no tokens has no element, and A may be absent: without weight gradients nothing is launched."""
    status, message = _status("talm_lora_bwd_drop", None, 64, None, 32, None, 16, None, 16, 0, 64, 1, 0.5, PTR, 0, 1,
                              _lib.TALM_F32, 0, 32, 1.0, None, None, 0, 0, 0.0, None, None, None, None, None, 0, PTR,
                              64, PTR, 1 << 20, None)
    assert status == _lib.TALM_OK, message


def test_window_remainder_has_to_be_aligned():
    rows = [PTR, 256, 128]
    status, message = _status("talm_attn_window_fwd_lo", *rows, *rows, *rows, PTR, 1, 8, 8, 2, 2, 128, 1.0, 4, 0,
                              _lib.TALM_F16, PTR, 256, 128, PTR + 8, PTR, None)
    assert status == _lib.TALM_EINVAL and "out_lo" in message
    status, message = _status("talm_attn_window_bwd_lo", *rows, *rows, *rows, PTR, 256, 128, PTR + 8, *rows, PTR, PTR, 1,
                              8, 8, 2, 2, 128, 1.0, 4, 0, _lib.TALM_F16, None, None, 0, *rows, *rows, *rows, PTR,
                              1 << 20, None)
    assert status == _lib.TALM_EINVAL and "out_lo" in message
