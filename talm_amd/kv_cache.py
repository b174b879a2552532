"""An attention layer's keys and values in 8 bits, for a model that answers token by token.

`QuantizedCache` is a model's cache: given as `past_key_values` to a patched Qwen2 (`generate`, or its
forward), which then keeps its keys and values in 8 bits and attends to them with the kernels here;
sliding layers with sinks (config.attention_sinks), which transformers' own masks do not know, are
answered with it too.

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

import contextlib
import functools

import torch
from transformers import Cache

from . import _ops, unpad  # noqa: F401 - _ops registers torch.ops.talm.*
from .engaged import ON, RAN
from .state import DISABLED, fallback

BLOCK = 64
_HALVES = (torch.float16, torch.bfloat16)


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
    current stream, wait for nothing and can be captured in a HIP graph; they have no derivative and
    refuse operands that need one (that require a gradient, or are dual). A row belongs to one sequence,
    and a page that a call writes to one block of one sequence."""

    def __init__(self, codes, scales, tail, table):
        self.codes, self.scales, self.tail, self.table = codes, scales, tail, table

    @classmethod
    def allocate(cls, sequences, kv_heads, head_dim, capacity, dtype=torch.float16, device="cuda"):
        """Buffers for `sequences` of up to `capacity` tokens, sequence b's pages one behind the other."""
        if min(sequences, kv_heads, capacity) < 0 or head_dim not in (64, 128) \
                or dtype not in _HALVES:
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
        key, value = out if out is not None else (None, None)
        out = torch.ops.talm.cache_read(self.codes, self.scales, self.tail, self.table, length, bounds, past, max_new,
                                        rows, key, value)
        RAN["cache_read"] += 1
        return out

    def attention(self, query, bounds, past, max_new, max_len, scale, window=None, sinks=0):
        """softmax(scale q K^T) V of query [1, Hq, N, D] over the cache, which holds the rows' own tokens
        already and none behind them (past[b] and b's rows are all that it has): the row of token p sees the
        tokens up to p, in a `window` only the last `window` ones (itself among them) and the sequence's
        first `sinks`. `max_len` is at least the longest sequence with its new tokens (in a graph: with those
        of any replay). Values of tokens that a row does not see must be finite, since a weight of 0 does
        not hide NaN; its keys may be anything. Returns [1, N, Hq, D], means of values and none past the
        type's largest number; a row that sees nothing is zero, a row that no sequence holds undefined."""
        if window is not None and window < 1:
            raise ValueError(f"cache_attention: window {window} (at least 1, or None)")
        out = torch.ops.talm.cache_attention(query, bounds, past, max_new, max_len, self.codes, self.scales,
                                             self.tail, self.table, scale, window or 0, sinks)
        RAN["cache_attn"] += 1
        return out


def _packed(x):
    """[B, H, T, D] -> its rows as [1, H, B T, D], a view where the strides allow one."""
    b, h, t, d = x.shape
    return x.transpose(1, 2).reshape(b * t, h, d).transpose(0, 1)[None]


class QuantizedCache(Cache):
    """The keys and values of a patched Qwen2 in 8 bits, for `batch` sequences of up to `capacity` tokens:

        cache = QuantizedCache(model.config, batch=4, capacity=4096)
        model.generate(**inputs, past_key_values=cache)

    Each call's new tokens are those that its attention mask names, one run per sequence (left-padded
    prompts, as generation has them); padding is neither stored nor attended to. A first call attends to
    its own 16-bit keys and values where the packed rows' kernels take them (fp16 or bfloat16 heads of
    128), later ones, and first ones of heads of 64, to the cache. `dtype`, of its 16-bit parts and its
    attention, is by default that of the first call's keys: float32 ones count as autocast's type, and
    without autocast as bfloat16, which has their range. A named float16 makes numbers past 65504
    infinite. Models that run inside of its calls (a hook's) are answered on their own.

    It needs solution.apply(), the "sdpa" attention, no gradient, and every layer's call (no checkpointed
    ones); it does not reorder, repeat or crop its sequences (beam search, assisted generation), and its
    calls run eagerly (a step to capture in a HIP graph takes CacheLayer)."""

    is_compileable = False

    def __init__(self, config, batch, capacity, dtype=None, device="cuda"):
        super().__init__(layers=[])
        heads = config.num_attention_heads
        dim = getattr(config, "head_dim", None) or config.hidden_size // heads
        self.cache_layers = [CacheLayer.allocate(batch, config.num_key_value_heads, dim, capacity,
                                                 torch.float16 if dtype is None else dtype, device)
                             for _ in range(config.num_hidden_layers)]
        self.batch, self.capacity = batch, capacity
        self.named_dtype = self.dtype = dtype
        self.device = torch.device(device)
        self.lengths, self.columns = [0] * batch, 0
        self._step = self._broken = None

    # -- what transformers asks of a cache

    def get_seq_length(self, layer_idx=0):
        """Columns of the attention mask so far, padding among them."""
        return self.columns

    def get_mask_sizes(self, query_length, layer_idx=0):
        return self.columns + int(query_length), 0

    def get_max_length(self, layer_idx=0):
        return self.capacity

    get_max_cache_shape = get_max_length

    def reset(self):
        """Empty again, also after a call that failed part-way."""
        self.lengths, self.columns = [0] * self.batch, 0
        self._step = self._broken = None
        self.dtype = self.named_dtype

    def _unsupported(self, *args, **kwargs):
        raise NotImplementedError("QuantizedCache does not reorder, repeat, select, crop or offload its sequences")

    reorder_cache = crop = batch_repeat_interleave = batch_select_indices = offload = _unsupported

    # -- one call of the model

    @contextlib.contextmanager
    def step(self, config, batch, rows, mask=None):
        """One forward of `rows` new columns a sequence; `mask` [batch, columns so far + rows] or None (all
        of them tokens). The sequences grow when it ends; one that fails part-way leaves the cache unusable
        until `reset`, since some layers hold its tokens."""
        from .fused_proj import _rows_attention

        if self._broken:
            raise RuntimeError("QuantizedCache: a call failed part-way, reset() empties the cache")
        if self._step is not None:
            raise RuntimeError("QuantizedCache: one call of the model at a time")
        if torch.is_grad_enabled():
            raise ValueError("QuantizedCache: the cache has no gradient, call the model under torch.no_grad()")
        if not _rows_attention(config):
            raise ValueError('QuantizedCache: the model must be patched (solution.apply()) and use "sdpa" attention')
        if self.device.type == "cuda" and torch.cuda.is_current_stream_capturing():
            raise RuntimeError("QuantizedCache: its calls run eagerly; capture CacheLayer's operators")
        if batch != self.batch or rows < 1:
            raise ValueError(f"QuantizedCache: {rows} tokens of {batch} sequences, made for {self.batch}")
        runs, padded = _runs(mask, batch, self.columns, rows)
        new = [end - start for start, end in runs]
        lengths = [n + m for n, m in zip(self.lengths, new)]
        if max(lengths) > self.capacity:
            raise ValueError(f"QuantizedCache: a sequence of {max(lengths)} tokens, made for {self.capacity}")
        first = not any(self.lengths)
        # one copy: bounds, past, and for a first call the rows' sequences, padding as sequences of its own
        bounds = [b * rows + at for b, run in enumerate(runs) for at in run]
        values = bounds + self.lengths + ([0] + bounds + [batch * rows] if first else [])
        device = torch.tensor(values, dtype=torch.int32).pin_memory().to(self.device, non_blocking=True)
        self._step = _Step(device[:2 * batch].view(batch, 2), device[2 * batch:3 * batch], max(new), max(lengths),
                           device[3 * batch:] if first else None, rows,
                           _real(runs, rows, self.device) if padded else None)
        outer, unpad._cached.step = getattr(unpad._cached, "step", None), self
        try:
            yield
            self._settled()
            if len(self._step.written) != len(self.cache_layers):
                raise RuntimeError(f"QuantizedCache: layers {sorted(self._step.written)} of {len(self.cache_layers)} "
                                   "wrote their tokens (a checkpointed layer is not given the cache)")
        except BaseException:
            self._broken = True
            raise
        finally:
            unpad._cached.step, self._step = outer, None
        self.lengths, self.columns = lengths, self.columns + rows

    def _layer(self, layer_idx):
        if self._step is None:
            raise RuntimeError("QuantizedCache: outside of a patched Qwen2 model's forward (solution.apply())")
        return self.cache_layers[layer_idx]

    def _writes(self, layer_idx):
        """The layer, about to be written in this call."""
        layer = self._layer(layer_idx)
        self._settled()
        if layer_idx in self._step.written:
            raise RuntimeError(f"QuantizedCache: layer {layer_idx} wrote its tokens already in this call")
        self._step.written.add(layer_idx)
        return layer

    def _take_type(self, key):
        """The cache's type from its first keys, unless it was named; later ones must be of the same."""
        if self.named_dtype is not None:
            return
        dtype = key.dtype
        if dtype not in _HALVES:
            kind = key.device.type
            dtype = torch.get_autocast_dtype(kind) if torch.is_autocast_enabled(kind) else None
            dtype = dtype if dtype in _HALVES else torch.bfloat16
        if self.dtype is None:
            self.dtype = dtype
            for layer in self.cache_layers:
                layer.tail = layer.tail.view(dtype)
        elif self.dtype != dtype:
            raise ValueError(f"QuantizedCache: keys of {dtype} behind ones of {self.dtype}: name the cache's dtype")

    def _settled(self):
        """The attention of what the last `update` returned must have been asked for here."""
        if self._step.kept is not None:
            raise RuntimeError("QuantizedCache: a layer's attention was not of the keys and values that the cache "
                               "returned to it")

    def update(self, key_states, value_states, layer_idx, *args, **kwargs):
        """New keys and values [B, Hkv, T, D] of one layer; returns them (the attention reads the cache)."""
        layer, s = self._writes(layer_idx), self._step
        self._take_type(key_states)
        key_states, value_states = key_states.to(self.dtype), value_states.to(self.dtype)
        if key_states.shape[0] != self.batch or key_states.shape[2] != s.rows:
            raise ValueError(f"QuantizedCache: keys of {key_states.shape[0]} sequences of {key_states.shape[2]} tokens "
                             f"in a call of {self.batch} of {s.rows}")
        layer.write(_packed(key_states), _packed(value_states), s.bounds, s.past, s.max_new)
        s.kept = key_states, value_states
        return s.kept

    def asked(self, key, value):
        """Whether an attention call is of the keys and values that the last `update` returned: a model that runs
        inside of this one's call, a probe or a guard, has others."""
        kept = self._step.kept
        return kept is not None and key is kept[0] and value is kept[1]

    def takes(self, dtype, dim):
        """Whether `answer` serves the call: not a first one (its keys are needed in 16 bits), with heads of
        the cache's type and size."""
        return (self._step is not None and self._step.cu is None and dtype == self.dtype
                and dim == self.cache_layers[0].tail.shape[3] // BLOCK)

    def answer(self, query, key, value, layer_idx, tables, scale, window, sinks, dropout=0.0):
        """Attention of new rows [1, H, N, D] that are not turned yet, tables (cos, sin) float32 [N, D]: written
        with their rotary positions in one launch, then attended. Returns [1, N, Hq, D]."""
        if dropout:
            raise ValueError("QuantizedCache: no dropout of attention weights")
        layer, s = self._writes(layer_idx), self._step
        turned = layer.write(key, value, s.bounds, s.past, s.max_new, query, tables)
        return self._clean(layer.attention(turned, s.bounds, s.past, s.max_new, s.max_len, scale, window, sinks))

    def attend(self, module, query, key, value, dropout, scaling, window):
        """The attention interface of a call with this cache: query [B, Hq, T, D] against the layer's tokens;
        returns [B, T, Hq, D] in the query's type."""
        if dropout:
            raise ValueError("QuantizedCache: no dropout of attention weights")
        layer, s = self._layer(module.layer_idx), self._step
        b, heads, t, d = query.shape
        if b != self.batch or t != s.rows:
            raise ValueError(f"QuantizedCache: queries of {b} sequences of {t} tokens in a call of {self.batch} of "
                             f"{s.rows}")
        s.kept = None
        scale = scaling if scaling is not None else d ** -0.5
        sinks = unpad.attention_sinks(module) if window is not None else 0
        q = _packed(query.to(self.dtype))
        out = None
        if s.cu is not None:
            out = self._first(q, _packed(key), _packed(value), scale, window, sinks)
        if out is None:
            out = self._clean(layer.attention(q, s.bounds, s.past, s.max_new, s.max_len, scale, window, sinks))
        return out.view(b, t, heads, d).to(query.dtype)

    def _first(self, q, k, v, scale, window, sinks):
        """A first call's attention to its own keys and values in the packed rows' kernels; None where they do
        not take it, are off or failed (state.py): the cache answers then."""
        s = self._step
        if "varlen_attention" in DISABLED or not unpad.window_takes(q, k, v):
            return None
        try:
            # without a window: the fp16 kernels of training, or a window that no sequence is longer than
            if window is None and q.dtype == torch.float16:
                out = unpad.VarlenAttention.apply(q, k, v, s.cu, s.rows, scale)
                RAN["varlen_attn"] += 1
                return out
            return unpad.window_attention(q, k, v, s.cu, s.rows, scale, window or s.rows, sinks)
        except Exception as exc:  # noqa: BLE001 - state.py convention
            if not fallback("varlen_attention", exc):
                raise
        return None

    def _clean(self, out):
        """Padding's rows, which no sequence holds, as zeros."""
        real = self._step.real
        return out if real is None else torch.where(real, out, 0.0)


class _Step:
    """What the layers of one call share."""

    def __init__(self, bounds, past, max_new, max_len, cu, rows, real):
        self.bounds, self.past, self.max_new, self.max_len = bounds, past, max_new, max_len
        self.cu, self.rows, self.real = cu, rows, real
        self.written = set()  # the layers that hold the call's tokens
        self.kept = None  # the keys and values that `update` returned, until their attention


def _runs(mask, batch, columns, rows):
    """Where each sequence's new tokens lie among its `rows` new columns, [(start, end)], and whether any
    column is padding. Reads the mask on the host."""
    if mask is None:
        return [(0, rows)] * batch, False
    if not isinstance(mask, torch.Tensor) or tuple(mask.shape) != (batch, columns + rows):
        raise ValueError(f"QuantizedCache: an attention mask [{batch}, {columns + rows}] of the tokens so far and "
                         "the new ones, or none")
    new = mask[:, columns:] != 0
    count = new.sum(1)
    start = new.to(torch.int8).argmax(1)
    # a run: as many tokens between the first and the last as there are
    span = torch.where(count > 0, rows - new.flip(1).to(torch.int8).argmax(1) - start, 0)
    values = torch.stack((count, start, span)).tolist()
    if values[0] != values[2]:
        raise ValueError("QuantizedCache: a sequence's new tokens must be one run of its mask")
    return [(lo, lo + n) for n, lo in zip(values[0], values[1])], any(n < rows for n in values[0])


def _real(runs, rows, device):
    """[1, B T, 1, 1]: the rows that are tokens."""
    at = torch.arange(rows)
    lo, hi = torch.tensor(runs).unbind(1)
    return ((at >= lo[:, None]) & (at < hi[:, None])).view(1, -1, 1, 1).to(device)


def patch_qwen2_cache():
    """`Qwen2Model.forward` opens the step of a QuantizedCache that it is given, and makes no masks then."""
    from transformers.models.qwen2 import modeling_qwen2

    cls = modeling_qwen2.Qwen2Model
    forward = cls.forward
    ON.add("kv_cache")
    if getattr(forward, "_talm_cache", False):
        return

    @functools.wraps(forward)
    def forward_cached(self, input_ids=None, attention_mask=None, position_ids=None, past_key_values=None,
                       inputs_embeds=None, **kwargs):
        if not isinstance(past_key_values, QuantizedCache):
            return forward(self, input_ids=input_ids, attention_mask=attention_mask, position_ids=position_ids,
                           past_key_values=past_key_values, inputs_embeds=inputs_embeds, **kwargs)
        tokens = input_ids if input_ids is not None else inputs_embeds
        with past_key_values.step(self.config, tokens.shape[0], tokens.shape[1], attention_mask):
            return forward(self, input_ids=input_ids, attention_mask={"full_attention": None, "sliding_attention": None},
                           position_ids=position_ids, past_key_values=past_key_values, inputs_embeds=inputs_embeds,
                           **kwargs)

    forward_cached._talm_cache = True
    cls.forward = forward_cached
