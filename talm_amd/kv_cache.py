"""An attention layer's keys and values in 8 bits, for a model that answers token by token.

`CacheLayer` holds the buffers of one layer and has three operators on the HIP kernels (kvcache.hip,
talm_cache_write / _read / _attn): new tokens' keys and values are written, quantized block by block
and turned by their rotary positions on the way; tokens are read back in 16 bits; new tokens' queries
attend to the cache. No counterpart in the reference, which trains.

A sequence's tokens form blocks of 64 (`BLOCK`). A complete block is a page of the layer's pool: per KV
head its keys, and its values, as 8-bit floats (e4m3) times one power of two, the smallest that takes
the block's largest magnitude to at most 448. The tokens behind the last complete block stay in 16
bits, so a cache's contents do not depend on how its tokens were split over calls. `table` names the
page of each of a sequence's blocks: pages may lie in any order, and sequences with a common
beginning may share complete ones.
"""

import torch

from . import _ops  # noqa: F401 - registers torch.ops.talm.*
from .engaged import RAN

BLOCK = 64


class CacheLayer:
    """The buffers of one attention layer's cache, on one GPU, contiguous:

      codes   float8_e4m3fn [pages, 2, Hkv, 64 D]   keys, values; D 64 or 128
      scales  float32 [pages, 2, Hkv]
      tail    float16 or bfloat16 [sequences, 2, Hkv, 64 D]   each sequence's open block
      table   int32 [sequences, width]   pages of blocks; an entry that is no page of the pool holds
              none (its block's tokens are dropped, read as zeros and not attended to)

    A page's order is the kernels' (include/talm.h). The operators take new tokens as rows of packed
    operands [1, H, N, D] (any strides; fp16 or bf16 as the tail): sequence b's are rows bounds[b, 0] to
    bounds[b, 1] - 1, its tokens past[b], past[b] + 1, ..; `bounds` int32 [sequences, 2] and `past` int32
    [sequences] lie on the device, `max_new` is at least the largest count of rows. Rows that no sequence
    holds, that lie past max_new or do not fit the table are not written. The operators run on the
    current stream, wait for nothing and can be captured in a HIP graph; they have no gradient and
    refuse operands that need one."""

    def __init__(self, codes, scales, tail, table):
        self.codes, self.scales, self.tail, self.table = codes, scales, tail, table

    @classmethod
    def allocate(cls, sequences, kv_heads, head_dim, capacity, dtype=torch.float16, device="cuda"):
        """Buffers for `sequences` of up to `capacity` tokens, sequence b's pages one behind the other."""
        if min(sequences, kv_heads, capacity) < 0 or head_dim not in (64, 128) \
                or dtype not in (torch.float16, torch.bfloat16):
            raise ValueError(f"CacheLayer: {sequences} sequences of {capacity} tokens, {kv_heads} KV heads of "
                             f"{head_dim} (64 or 128) in {dtype} (float16 or bfloat16)")
        width = -(-capacity // BLOCK)
        pages, size = sequences * width, BLOCK * head_dim
        return cls(torch.empty(pages, 2, kv_heads, size, dtype=torch.float8_e4m3fn, device=device),
                   torch.empty(pages, 2, kv_heads, dtype=torch.float32, device=device),
                   torch.empty(sequences, 2, kv_heads, size, dtype=dtype, device=device),
                   torch.arange(pages, dtype=torch.int32, device=device).view(sequences, width))

    @property
    def capacity(self):
        """The most tokens of a sequence."""
        return self.table.shape[1] * BLOCK

    def write(self, key, value, bounds, past, max_new, query=None, rope=None):
        """Append key and value [1, Hkv, N, D]. With `rope` = (cos, sin) float32 [N, D] the keys are turned
        first, and the query [1, Hq, N, D]: returns it turned, as a new tensor (every row of it), or
        None. A call reads the open block that the call before it left: writes to one sequence stay in
        order."""
        cos, sin = rope if rope is not None else (None, None)
        out = torch.ops.talm.cache_write(key, value, bounds, past, max_new, self.codes, self.scales, self.tail,
                                         self.table, query, cos, sin)
        RAN["cache_write"] += 1
        return out

    def read(self, length, bounds, past, max_new, rows, out=None):
        """Tokens past[b] + i of a cache whose sequences hold `length` (int32 [sequences]) tokens, as rows
        bounds[b, 0] + i of (key, value), each [1, Hkv, rows, D] in the tail's type. `out`: two contiguous
        [rows, Hkv, D] buffers to take them (rows that no sequence holds keep their contents there, and
        are undefined without it). Tokens behind a sequence's length read as zeros."""
        if out is None:
            shape = (rows, self.codes.shape[2], self.codes.shape[3] // BLOCK)
            out = (self.tail.new_empty(shape), self.tail.new_empty(shape))
        elif any(t.shape[0] != rows for t in out):
            raise ValueError(f"cache_read: out of {[t.shape[0] for t in out]} rows, {rows} asked")
        torch.ops.talm.cache_read(self.codes, self.scales, self.tail, self.table, length, bounds, past, max_new,
                                  *out)
        RAN["cache_read"] += 1
        return tuple(t.transpose(0, 1)[None] for t in out)

    def attention(self, query, bounds, past, max_new, max_len, scale, window=None, sinks=0):
        """softmax(scale q K^T) V of query [1, Hq, N, D] over the cache, which holds the rows' own tokens
        already: the row of token p sees the tokens up to p, in a `window` only the last `window` ones
        (itself among them) and the sequence's first `sinks`. `max_len` is at least the longest sequence
        with its new tokens. Returns [1, N, Hq, D]; a row that sees nothing is zero, a row that no
        sequence holds undefined."""
        if window is not None and window < 1:
            raise ValueError(f"cache_attention: window {window} (at least 1, or None)")
        out = torch.ops.talm.cache_attention(query, bounds, past, max_new, max_len, self.codes, self.scales,
                                             self.tail, self.table, scale, window or 0, sinks)
        RAN["cache_attn"] += 1
        return out
