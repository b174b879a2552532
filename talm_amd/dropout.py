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


def counter_dropout():
    """Whether the LoRA nodes' dropout comes from this generator now."""
    return COUNTER or torch.cuda.is_initialized() and torch.cuda.is_current_stream_capturing()


def draw_key(device):
    """A fresh key, int64 [2] on `device`, from PyTorch's generator of the device."""
    return torch.randint(-2 ** 63, 2 ** 63 - 1, (2,), dtype=torch.int64, device=device)


def dropout(x, p, key=None, site=0):
    """x with each element dropped with probability p (in steps of 2^-16) and the others scaled by
    the reciprocal of the share kept; float32, float16 or bfloat16 on the GPU, of any shape and
    strides. An autograd node of the C++ op layer, differentiable once."""
    return torch.ops.talm.counter_dropout(x, p, key, site)
