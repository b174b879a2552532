"""Dropout whose mask is computed from a counter-based generator and never stored.

`dropout(x, p, key, site)` keeps element (r, c) of x (as rows of its last dimension) when its 16
bits of the generator are at least round(65536 p), and multiplies kept elements by the reciprocal
of the exact share kept; the backward computes the same mask again (talm_dropout; the generator
and its counters are described in include/talm.h). `key` is an int64 [2] tensor on x's device,
`site` tells the dropouts that share a key apart: the same key, site and shape give the same
mask. `draw_key(device)` draws a key from PyTorch's generator of the device, so
`torch.manual_seed` and saved generator states repeat the masks; a key is read on the device, so
a HIP graph that draws one draws a new one on every replay.

The reference's adapters with dropout keep a mask, or the generator's state to draw it again
(solution/lora.py:183-186, :209-216; solution/fused_proj.py:139-153, :188-193). Reading a
generator's state is not possible while a graph is captured; a key is.
"""

import os

import torch

from . import _ops  # noqa: F401 - registers torch.ops.talm.*

# The q|k|v and single-projection LoRA nodes take their adapters' dropout from this generator
# (fused_proj.py) instead of PyTorch's native_dropout. Off by default: a seed then gives PEFT's masks.
# While a graph is captured they do so in any case.
COUNTER = os.environ.get("SOLUTION_COUNTER_DROPOUT") == "1"


def draw_key(device):
    """A fresh key, int64 [2] on `device`, from PyTorch's generator of the device."""
    return torch.randint(-2 ** 63, 2 ** 63 - 1, (2,), dtype=torch.int64, device=device)


def check(x, p, key, site):
    """The arguments' common checks (ValueError)."""
    if not 0.0 <= p < 1.0:
        raise ValueError(f"dropout: p {p} (0 <= p < 1)")
    if key is None and p > 0.0:
        raise ValueError("dropout: a key is needed (draw_key)")
    if key is not None and (key.dtype != torch.int64 or key.numel() != 2
                            or key.device != x.device or not key.is_contiguous()):
        raise ValueError("dropout: key int64 [2], contiguous, on x's device")
    if not 0 <= site < 2 ** 32:
        raise ValueError(f"dropout: site {site} (0 .. 2^32 - 1)")


def _apply(x, p, key, site):
    if x.numel() == 0:
        return torch.empty_like(x, memory_format=torch.contiguous_format)
    x2 = x.reshape(-1, x.shape[-1] if x.dim() else 1)
    if x2.shape[1] > 1 and x2.stride(1) != 1 or x2.shape[0] > 1 and x2.stride(0) < x2.shape[1]:
        x2 = x2.contiguous()
    y = torch.empty(x2.shape, dtype=x.dtype, device=x.device)
    torch.ops.talm.dropout(x2, p, key, site, y)
    return y.view(x.shape)


class Dropout(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, p, key, site):
        ctx.p, ctx.site = p, site
        ctx.save_for_backward(key)
        return _apply(x, p, key, site)

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, grad):
        (key,) = ctx.saved_tensors
        return _apply(grad, ctx.p, key, ctx.site), None, None, None


def dropout(x, p, key=None, site=0):
    """x with each element dropped with probability p (in steps of 2^-16) and the others scaled by
    the reciprocal of the share kept; float32, float16 or bfloat16 on the GPU."""
    if not x.is_cuda or x.dtype not in (torch.float32, torch.float16, torch.bfloat16):
        raise ValueError("dropout: a float32, float16 or bfloat16 tensor on the GPU")
    p, site = float(p), int(site)
    check(x, p, key, site)
    return Dropout.apply(x, p, key, site)
