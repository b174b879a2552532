"""The projections of a packed 4-bit layer for calls of a few tokens without autograd: what a
generating model does token by token.

A training forward dequantizes a layer once (94 MB written) for products of a thousand tokens; one
token's products cost a fraction of that. Here each projection is one launch on the layer's NF4
codes (talm_nf4_gemv, LayerGroup.nf4_gemv; nothing is dequantized and no layer becomes resident):
q|k|v as one product with the LoRA adapters of q and v added before the one rounding, o, gate|up
and down. The same fp16 weights and fp32 sums as the products they replace (GroupLinear,
solution/qgroup.py:346-355; the adapters as PEFT adds them, solution/lora.py:183-186).

A token of the 28-layer Qwen2.5-1.5B shape in 4 bits, batch 1 / 8 / 32 (MI355X, transformers' cache, the host sets
the time): 8.0 / 8.7 / 8.7 ms, against 10.9 / 13.3 / 13.3 through whole layers' dequantization.

Used by the patched Linear4bit, LoraLinear, Qwen2Attention and Qwen2MLP forwards for at most
GEMV_TOKENS rows while gradients are off; SOLUTION_DISABLE_GEMV=1 keeps the other paths.
"""

import os

import torch

from .engaged import RAN
from .state import DISABLED, fallback

ENABLED = os.environ.get("SOLUTION_DISABLE_GEMV") != "1"

# the most rows of x that talm_nf4_gemv takes, and the most elements from one to the next
GEMV_TOKENS, MAX_STRIDE = 32, 1 << 24


def few(x):
    """Whether x [..., C] is a call this module is for, by its rows and the grad mode."""
    return (ENABLED and not torch.is_grad_enabled() and "gemv" not in DISABLED
            and "qgroup" not in DISABLED and x.is_cuda and x.dim() >= 1
            and 0 < x.numel() <= GEMV_TOKENS * x.shape[-1])


def takes(x, group, first, last):
    """Whether `linear` takes fp16 x for projections first .. last - 1 of the group."""
    return (few(x) and x.dtype == torch.float16 and group.gemv_ok(first, last)
            and group.shapes[first][1] == x.shape[-1])


def serves(group, x):
    """Whether every projection of the group runs here for x's rows: the layer's forward then need
    not dequantize it."""
    return few(x) and all(group.gemv_ok(i, i + 1) for i in range(len(group.shapes)))


def _rows(x):
    x2 = x.reshape(-1, x.shape[-1])
    (n, cols), (step, unit) = x2.shape, x2.stride()
    # the kernel's rows do not overlap, and lie at most MAX_STRIDE elements apart
    if unit != 1 or x2.data_ptr() % 16 or n > 1 and (step % 8 or not cols <= step <= MAX_STRIDE):
        x2 = x2.clone(memory_format=torch.contiguous_format)
    return x2


def _adapters_take(group, first, last, adapters, halves):
    """Whether the adapters ((segment, scaling, p), ..) with fp16 (A, B) per adapter can be added by
    the product: one or two of rank 16 without dropout."""
    size = group.shapes[first][1]
    return (len(adapters) <= 2 and size % 32 == 0
            and all(p == 0 and tuple(a.shape) == (16, size) and a.is_contiguous() and b.is_contiguous()
                    and tuple(b.shape) == (group.shapes[first + seg][0], 16)
                    for (seg, _s, p), (a, b) in zip(adapters, halves)))


def linear(x, group, first, last, adapters=(), halves=()):
    """x [..., in] through projections first .. last - 1 side by side, with their biases and LoRA
    adapters: [..., sum of out]. None where the product does not take the call, or failed (it is then
    off, state.py): the caller's other path runs."""
    if not takes(x, group, first, last) or not _adapters_take(group, first, last, adapters, halves):
        return None
    try:
        return _linear(x, group, first, last, adapters, halves)
    except Exception as exc:  # noqa: BLE001 - state.py convention
        if not fallback("gemv", exc):
            raise
        return None


def _linear(x, group, first, last, adapters, halves):
    x2 = _rows(x)
    n, sizes = x2.shape[0], [group.shapes[i][0] for i in range(first, last)]
    added = None
    if adapters:
        t = torch.empty(n, 16 * len(adapters), dtype=torch.float16, device=x.device)
        ts = torch.empty_like(t)
        size, two = x2.shape[1], len(adapters) > 1
        torch.ops.talm.lora_down(x2, halves[0][0], halves[1][0] if two else None, size, size, 0, 0, 0,
                                 adapters[0][1], adapters[1][1] if two else 0.0, t, ts)
        added = (ts, [(b, sum(sizes[:seg]), sum(sizes[:seg + 1]))
                      for (seg, _s, _p), (_a, b) in zip(adapters, halves)])
    out = torch.empty(n, sum(sizes), dtype=torch.float16, device=x.device)
    group.nf4_gemv(x2, first, last, out, added)
    RAN["gemv"] += 1
    return out.view(*x.shape[:-1], out.shape[1])


def mlp_takes(x, group, gate, down):
    """Whether `mlp` takes fp16 x."""
    return takes(x, group, gate, down) and group.gemv_ok(down, down + 1)


def mlp(x, group, gate, down):
    """down(silu(gate(x)) * up(x)), gate and up adjacent projections, in three launches; None as
    `linear`."""
    if not group.gemv_ok(down, down + 1):
        return None
    gu = linear(x, group, gate, down)
    if gu is None:
        return None
    inter = gu.shape[-1] // 2
    gu2 = gu.view(-1, 2 * inter)
    act = torch.empty(gu2.shape[0], inter, dtype=torch.float16, device=x.device)
    torch.ops.talm.swiglu_fwd_rows(gu2[:, :inter], gu2[:, inter:], act)
    y = linear(act, group, down, down + 1)
    return None if y is None else y.view(*x.shape[:-1], -1)
