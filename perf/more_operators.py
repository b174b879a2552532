"""Operators of an 8-bit key and value cache, each as a program that answers with it calls it
(Qwen2.5-1.5B shape: 12 query / 2 KV heads of 128; the smaller models' 14 / 2 heads of 64).

Kinds of case:
  write  new tokens' keys and values into the cache, quantized block by block, queries and keys
         turned by their rotary positions on the way (kv_cache.CacheLayer.write)
  read   tokens of the cache back in 16 bits (kv_cache.CacheLayer.read)
  attn   attention of new tokens over the cache (kv_cache.CacheLayer.attention)

The cache of a layer. A sequence's tokens form blocks of 64. A complete block is a page: its keys
and its values, per KV head, are 8-bit floats (e4m3) times one power of two, the smallest that takes
the block's largest magnitude to at most 448. The tokens behind the last complete block stay in 16
bits. Buffers: codes [pages, 2, Hkv, 64 D] (keys, values), scales [pages, 2, Hkv], tail [sequences,
2, Hkv, 64 D] and table [sequences, width], the page of each of a sequence's blocks. A page's keys
lie as [16 tokens' tile 4, D / 64, quarter of 64 columns 4, token 16, column 16], its values as [tile
of 16 columns D / 16, quarter of a tile of tokens 4, column 16, tile of tokens 4, token 4]; a tail's
keys as [64, D], its values as [D, 64]. New tokens are rows of packed buffers, `bounds` [sequences,
2] their first and end row for each sequence, `past` the tokens it had before.

With `own` false a pass computes the same in elementary torch operations, in 32 bits, rounded where
the cache or an output is; `exact` restates each kind in 64 bits.
"""

import math

import numpy as np
import torch

own = False

BLOCK = 64
DEV = "cuda"


def listed():
    return [
        # the token that one conversation is at: launch latency
        {"name": "write_1", "kind": "write", "count": 1, "past": "1999 1999", "new": "1 1",
         "heads": 12, "kv": 2, "dim": 128, "dtype": "float16"},
        # a step of 64 sequences answered together, some of which complete a block
        {"name": "write_64", "kind": "write", "count": 64, "past": "200 2047", "new": "1 1",
         "heads": 12, "kv": 2, "dim": 128, "dtype": "float16"},
        # four prompts that arrive together
        {"name": "write_prompts", "kind": "write", "count": 4, "past": "0 0", "new": "1531 4096",
         "heads": 12, "kv": 2, "dim": 128, "dtype": "float16"},
        # a long document
        {"name": "write_document", "kind": "write", "count": 1, "past": "0 0",
         "new": "32001 32001", "heads": 12, "kv": 2, "dim": 128, "dtype": "bfloat16"},
        # a few short conversations handed to code that takes 16-bit keys and values
        {"name": "read_8", "kind": "read", "count": 8, "past": "0 0", "new": "100 500",
         "heads": 14, "kv": 2, "dim": 64, "dtype": "float16"},
        # a batch's whole cache
        {"name": "read_16", "kind": "read", "count": 16, "past": "0 0", "new": "4000 8191",
         "heads": 12, "kv": 2, "dim": 128, "dtype": "bfloat16"},
        # one conversation's next token
        {"name": "attn_1", "kind": "attn", "count": 1, "past": "4000 4000", "new": "1 1",
         "heads": 12, "kv": 2, "dim": 128, "window": 0, "sinks": 0, "dtype": "float16"},
        # 64 sequences answered together, short and long ones
        {"name": "attn_64", "kind": "attn", "count": 64, "past": "200 8190", "new": "1 1",
         "heads": 12, "kv": 2, "dim": 128, "window": 0, "sinks": 0, "dtype": "float16"},
        # a question about a book: one token over the longest context
        {"name": "attn_book", "kind": "attn", "count": 1, "past": "131000 131000", "new": "1 1",
         "heads": 12, "kv": 2, "dim": 128, "window": 0, "sinks": 0, "dtype": "float16"},
        # a sliding layer with sinks, 32 long sequences, bfloat16
        {"name": "attn_window", "kind": "attn", "count": 32, "past": "9000 17000", "new": "1 1",
         "heads": 12, "kv": 2, "dim": 128, "window": 4096, "sinks": 4, "dtype": "bfloat16"},
        # a long prompt that goes through in pieces: its 512 next tokens
        {"name": "attn_piece", "kind": "attn", "count": 1, "past": "7777 7777", "new": "512 512",
         "heads": 12, "kv": 2, "dim": 128, "window": 0, "sinks": 0, "dtype": "float16"},
        # the next turns of 12 conversations
        {"name": "attn_turns", "kind": "attn", "count": 12, "past": "300 3500", "new": "1 300",
         "heads": 12, "kv": 2, "dim": 128, "window": 0, "sinks": 0, "dtype": "float16"},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _span(rng, lo, hi):
    top = _log(rng, lo, hi)
    return rng.randint(max(lo, top // 8), top), top


def draw(rng):
    kind = rng.choice(("write", "read", "attn", "attn"))
    heads, kv, dim = rng.choice(((12, 2, 128), (12, 2, 128), (14, 2, 64), (16, 8, 128),
                                 (8, 8, 64), (8, 1, 128)))
    case = {"kind": kind, "heads": heads, "kv": kv, "dim": dim,
            "dtype": rng.choice(("float16", "float16", "bfloat16"))}
    steps = rng.random() < 0.5  # single tokens, or longer pieces
    count = _log(rng, 1, 64) if steps else _log(rng, 1, 12)
    width = 256 / (kv * dim)  # so many tokens of the listed cases' width are one of these
    if kind == "read":
        new = _span(rng, 1, int(min(30000, 100000 * width / count)))
        return {**case, "count": count, "past": "0 0", "new": "%d %d" % new}
    if kind == "write":
        # pieces begin at a block's border, so that a pass can be repeated on one state
        past = _span(rng, 1, 4000) if steps else (BLOCK * rng.randint(0, 20),) * 2
        new = (1, 1) if steps else _span(rng, 1, int(min(30000, 60e6 / (heads + 2 * kv) / dim) / count))
    else:
        past = _span(rng, 1, int(min(130000, 270000 * width / count)))
        new = (1, 1) if steps else _span(rng, 1, 300)
        while count * new[1] * (past[1] + new[1]) * heads * dim > 6e9 and new[1] > 1:
            new = (max(1, new[0] // 2), new[1] // 2)
        window = rng.choice((0, 0, _log(rng, 1, 8192)))
        case.update(window=window, sinks=rng.choice((0, 1, 4, 64, 200)) if window else 0)
    return {**case, "count": count, "past": "%d %d" % past, "new": "%d %d" % new}


# -- inputs ----------------------------------------------------------------------------------------

def _spread(case, name):
    """The case's `count` lengths between its two ends, in no order."""
    lo, hi = (int(n) for n in case[name].split())
    n = [lo + i * 2654435761 % 2 ** 32 * (hi - lo + 1) // 2 ** 32
         for i in range(1, case["count"] + 1)]
    n[0] = hi
    return n


def _randn(g, *shape, dtype=torch.float32, std=1.0):
    return torch.randn(*shape, generator=g, device=DEV).mul_(std).to(dtype)


def _inputs(case, seed):
    g, dtype = torch.Generator(DEV).manual_seed(seed), getattr(torch, case["dtype"])
    heads, kv, dim, count = case["heads"], case["kv"], case["dim"], case["count"]
    past, new = _spread(case, "past"), _spread(case, "new")
    ends = np.cumsum(new)
    total, rows = [p + n for p, n in zip(past, new)], int(ends[-1])
    blocks = [-(-t // BLOCK) for t in total]
    pages = sum(blocks)
    # the pool's pages were handed out in any order
    order = torch.randperm(pages, generator=g, device=DEV).to(torch.int32)
    where = torch.full((count, max(blocks)), -1, dtype=torch.int64)
    first = 0
    for i, n in enumerate(blocks):
        where[i, :n] = torch.arange(first, first + n)
        first += n
    where = where.to(DEV)
    table = torch.where(where >= 0, order[where.clamp_min(0)], -1).to(torch.int32)
    # the projections' output: q, k and v are column views of one [N, q + k + v] buffer
    qkv = _randn(g, rows, heads + 2 * kv, dim)
    # a few columns of the keys are several times the others, as biases of k_proj make them
    loud = (1 + 7 * (torch.rand(kv, dim, generator=g, device=DEV) < 0.05)).float()
    qkv[:, heads:heads + kv] *= loud
    qkv = qkv.to(dtype)
    views = [t.transpose(0, 1)[None] for t in qkv.split((heads, kv, kv), 1)]
    s = {"kind": case["kind"], "query": views[0], "key": views[1], "value": views[2],
         "bounds": torch.tensor(np.stack((ends - new, ends), 1), dtype=torch.int32, device=DEV),
         "past": torch.tensor(past, dtype=torch.int32, device=DEV),
         "length": torch.tensor(total, dtype=torch.int32, device=DEV), "table": table,
         "rows": rows, "max_new": max(new), "max_len": max(total),
         "window": case.get("window", 0), "sinks": case.get("sinks", 0)}
    if case["kind"] == "write":
        s["codes"] = torch.zeros(pages, 2, kv, BLOCK * dim, device=DEV).to(torch.float8_e4m3fn)
        s["scales"] = torch.ones(pages, 2, kv, device=DEV)
        s["tail"] = _randn(g, count, 2, kv, BLOCK * dim, dtype=dtype)
        place = torch.cat([torch.arange(p, p + n) for p, n in zip(past, new)]).to(DEV)
        freq = 1e6 ** -(torch.arange(dim // 2, device=DEV, dtype=torch.float64) / (dim // 2))
        angle = place[:, None] * torch.cat((freq, freq))
        s["rope"] = (angle.cos().float(), angle.sin().float())
    else:
        held = _randn(g, pages, 2, kv, BLOCK, dim)
        held[:, 0] *= loud[:, None]
        codes, s["scales"] = _quantize(held.to(dtype).float())
        s["codes"] = _page_order(codes).to(torch.float8_e4m3fn)
        tail = _randn(g, count, 2, kv, BLOCK, dim)
        tail[:, 0] *= loud[:, None]
        s["tail"] = _tail_order(tail).to(dtype)
    # the plain form's indices, on the host known with the lengths: every block that the new tokens
    # touch, and each row's sequence, place in it and place among its new tokens
    touched = [(i, b) for i, (p, t) in enumerate(zip(past, total))
               for b in range(p // BLOCK, -(-t // BLOCK))]
    whole = [(b + 1) * BLOCK <= total[i] for i, b in touched]
    s["touched"] = tuple(torch.tensor(t, device=DEV) for t in zip(*touched))
    s["whole"] = torch.tensor([i for i, w in enumerate(whole) if w], dtype=torch.int64, device=DEV)
    s["part"] = torch.tensor([i for i, w in enumerate(whole) if not w], dtype=torch.int64, device=DEV)
    s["row_seq"] = torch.repeat_interleave(torch.arange(count), torch.tensor(new)).to(DEV)
    s["row_at"] = torch.cat([torch.arange(n) for n in new]).to(DEV)
    return s


def prepare(case, seed):
    s = _inputs(case, seed)
    if own:
        from talm_amd.kv_cache import CacheLayer

        s["layer"] = CacheLayer(s["codes"], s["scales"], s["tail"], s["table"])
    return s


# -- one pass --------------------------------------------------------------------------------------

def run(state):
    return (_OWN if own else _PLAIN)[state["kind"]](state)


def _own_write(s):
    query = s["layer"].write(s["key"], s["value"], s["bounds"], s["past"], s["max_new"], s["query"],
                             s["rope"])
    return {"codes": s["codes"], "scales": s["scales"], "tail": s["tail"], "query": query}


def _own_read(s):
    return s["layer"].read(s["length"], s["bounds"], s["past"], s["max_new"], s["rows"])


def _own_attn(s):
    return s["layer"].attention(s["query"], s["bounds"], s["past"], s["max_new"], s["max_len"],
                                s["query"].shape[3] ** -0.5, s["window"] or None, s["sinks"])


def _page_order(x):
    """[P, 2, H, 64, D] keys and values in the order of a page."""
    p, _, h, _, d = x.shape
    k = x[:, 0].view(p, h, 4, 16, d // 64, 4, 16).permute(0, 1, 2, 4, 5, 3, 6)
    v = x[:, 1].view(p, h, 4, 4, 4, d // 16, 16).permute(0, 1, 5, 3, 6, 2, 4)
    return torch.stack((k.flatten(2), v.flatten(2)), 1)


def _page_tokens(codes):
    """`_page_order` undone."""
    p, _, h, size = codes.shape
    d = size // BLOCK
    k = codes[:, 0].view(p, h, 4, d // 64, 4, 16, 16).permute(0, 1, 2, 5, 3, 4, 6)
    v = codes[:, 1].view(p, h, d // 16, 4, 16, 4, 4).permute(0, 1, 5, 3, 6, 2, 4)
    return torch.stack((k.reshape(p, h, BLOCK, d), v.reshape(p, h, BLOCK, d)), 1)


def _tail_order(x):
    """[S, 2, H, 64, D] keys and values in the order of a tail."""
    return torch.stack((x[:, 0].flatten(2), x[:, 1].transpose(2, 3).flatten(2)), 1)


def _tail_tokens(tail):
    s, _, h, size = tail.shape
    d = size // BLOCK
    return torch.stack((tail[:, 0].view(s, h, BLOCK, d),
                        tail[:, 1].view(s, h, d, BLOCK).transpose(2, 3)), 1)


def _quantize(x):
    """[P, 2, H, 64, D] in 32 bits -> codes as 32-bit values, scales [P, 2, H]."""
    top = x.abs().amax((3, 4))
    share, power = torch.frexp(top)  # 448 = 0.875 * 2^9
    power = torch.where(share <= 0.875, power - 9, power - 8)
    scale = torch.where(top > 0, ((power + 127) << 23).view(torch.float32), 1.0)
    return (x / scale[..., None, None]).to(torch.float8_e4m3fn).float(), scale


def _turn(x, cos, sin):
    half = x.shape[-1] // 2
    return x * cos[:, None] + torch.cat((-x[..., half:], x[..., :half]), -1) * sin[:, None]


def _plain_write(s):
    dtype = s["key"].dtype
    q, k, v = (s[name][0].transpose(0, 1).float() for name in ("query", "key", "value"))
    q, k = (_turn(t, *s["rope"]).to(dtype) for t in (q, k))
    x = torch.stack((k, v.to(dtype)), 1)  # [N, 2, H, D]
    seq, block = s["touched"]
    place = block[:, None] * BLOCK + torch.arange(BLOCK, device=DEV)
    at = place - s["past"][seq][:, None]
    before = _tail_tokens(s["tail"])[seq]
    row = (s["bounds"][seq, :1] + at).clamp(0, s["rows"] - 1)
    now = torch.where((at < 0)[:, None, None, :, None], before, x[row].permute(0, 2, 3, 1, 4))
    codes, scales = _quantize(now[s["whole"]].float())
    pages = s["table"][seq[s["whole"]], block[s["whole"]]].long()
    s["codes"].view(torch.uint8)[pages] = _page_order(codes).to(torch.float8_e4m3fn).view(torch.uint8)
    s["scales"][pages] = scales
    part = s["part"]
    there = (place < s["length"][seq][:, None])[part][:, None, None, :, None]
    s["tail"][seq[part]] = _tail_order(torch.where(there, now[part], before[part]))
    return {"codes": s["codes"], "scales": s["scales"], "tail": s["tail"],
            "query": q.transpose(0, 1)[None]}


def _values(s):
    """Every sequence's keys and values, [S, width of the table, 2, H, 64, D] in 32 bits; what lies
    behind a sequence's tokens is no value."""
    codes = _page_tokens(s["codes"].float()) * s["scales"][..., None, None]
    x = codes[s["table"].clamp_min(0).long()]
    block = torch.arange(x.shape[1], device=DEV)
    last = (block == (s["length"] // BLOCK)[:, None])[:, :, None, None, None, None]
    return torch.where(last, _tail_tokens(s["tail"]).float()[:, None], x)


def _plain_read(s):
    x = _values(s).permute(2, 0, 1, 4, 3, 5).flatten(2, 3)  # [2, S, tokens, H, D]
    x = x[:, s["row_seq"], s["past"][s["row_seq"]] + s["row_at"]].to(s["tail"].dtype)
    return tuple(t.transpose(0, 1)[None] for t in x)


def _plain_attn(s):
    _, heads, rows, dim = s["query"].shape
    k, v = _values(s).permute(2, 0, 3, 1, 4, 5).flatten(3, 4).unbind(0)  # [S, H, tokens, D]
    count, kv, tokens = k.shape[:3]
    most = s["max_new"]
    # each sequence's rows, to the longest's count; those behind its own are left out at the end
    at = torch.arange(most, device=DEV)
    row = (s["bounds"][:, :1] + at).clamp_max(rows - 1)
    q = s["query"][0].transpose(0, 1).float()[row].view(count, most, kv, heads // kv, dim)
    q = q.permute(0, 2, 3, 1, 4).reshape(count, kv, -1, dim)
    place, key = (s["past"][:, None] + at)[:, :, None], torch.arange(tokens, device=DEV)
    seen = (key <= place) & (key < s["length"][:, None, None])
    if s["window"]:
        seen &= (place - key < s["window"]) | (key < s["sinks"])
    p = torch.matmul(q, k.transpose(2, 3).contiguous()).mul_(dim ** -0.5)
    p = p.view(count, kv, heads // kv, most, tokens)
    p.masked_fill_(~seen[:, None, None], -math.inf)
    p = p.sub_(p.amax(-1, keepdim=True)).exp_()
    p = p.div_(p.sum(-1, keepdim=True)).view(count, kv, -1, tokens)
    v = torch.where((key < s["length"][:, None])[:, None, :, None], v, 0.0)
    o = torch.matmul(p, v).view(count, heads, most, dim).transpose(1, 2)
    return o[s["row_seq"], s["row_at"]].to(s["query"].dtype)[None]


_OWN = {"write": _own_write, "read": _own_read, "attn": _own_attn}
_PLAIN = {"write": _plain_write, "read": _plain_read, "attn": _plain_attn}


# -- what a pass cannot do without -----------------------------------------------------------------

def work(case):
    heads, kv, dim = case["heads"], case["kv"], case["dim"]
    past, new = _spread(case, "past"), _spread(case, "new")
    size, rows = 2 * kv * dim, sum(new)  # a token's keys and values

    def held(tokens, before=0):
        """The cache's bytes of tokens before .. tokens - 1 of one sequence."""
        whole = tokens // BLOCK * BLOCK
        return size * max(0, whole - before) + 2 * size * (tokens - max(whole, before))

    if case["kind"] == "write":
        # q, k, v, cos and sin; the turned q, the new tokens' place, and a completed block's rest
        n = sum(held(p + n, p) + (3 * size * (p % BLOCK) if (p + n) // BLOCK > p // BLOCK else 0)
                for p, n in zip(past, new))
        return {"bytes": n + rows * (4 * heads * dim + 2 * size + 8 * dim),
                "flops": rows * (3 * (heads + kv) * dim + 2 * size)}
    if case["kind"] == "read":
        return {"bytes": sum(held(n) for n in new) + 2 * size * rows, "flops": size * rows}
    window, sinks, pairs, cache = case["window"], case["sinks"], 0, 0
    for p, n in zip(past, new):
        at = np.arange(p, p + n, dtype=np.int64)
        if not window:
            pairs += int((at + 1).sum())
            cache += held(p + n)
            continue
        pairs += int((np.minimum(at + 1, window) + np.minimum(np.maximum(at + 1 - window, 0), sinks)).sum())
        start = max(0, p + 1 - window)
        cache += held(p + n, start) + size * min(start, sinks)
    return {"bytes": cache + 4 * rows * heads * dim, "flops": 4 * dim * heads * pairs}


# -- the definition in 64 bits ---------------------------------------------------------------------

def exact(case, seed):
    s = _inputs(case, seed)
    return {"write": _exact_write, "read": _exact_read, "attn": _exact_attn}[case["kind"]](case, s)


def _two_to(n):
    return ((n.long() + 1023) << 52).view(torch.float64)


def _nearest_code(x):
    """Values of magnitude at most 448 to the nearest number of the type with 3 bits behind the
    point from 2^-6 on and steps of 2^-9 below, ties to the even one."""
    _, power = torch.frexp(x)
    step = _two_to((power - 1).clamp_min(-6) - 3)
    return torch.round(x / step) * step


def _token(x, b):
    """Which numbers of a page's keys and of its values are token b's columns."""
    d = np.arange(x // BLOCK)
    tile, row, quarter, rest = b // 16, b % 16, b % 16 // 4, b % 4
    keys = tile * 16 * len(d) + d // 64 * 1024 + d % 64 // 16 * 256 + row * 16 + d % 16
    values = d // 16 * 1024 + quarter * 256 + d % 16 * 16 + tile * 4 + rest
    return torch.from_numpy(keys).to(DEV), torch.from_numpy(values).to(DEV)


def _exact_write(case, s):
    kv, dim = case["kv"], case["dim"]
    cos, sin = (t.double()[:, None] for t in s["rope"])
    turned = []
    for name in ("query", "key"):
        a, b = s[name][0].transpose(0, 1).double().chunk(2, -1)
        (ca, cb), (sa, sb) = cos.chunk(2, -1), sin.chunk(2, -1)
        turned.append(torch.cat((a * ca - b * sa, b * cb + a * sb), -1))
    q, k = turned
    v = s["value"][0].transpose(0, 1).double()
    codes, scales, tail = s["codes"].double(), s["scales"].double(), s["tail"].double()
    order = [_token(BLOCK * dim, t) for t in range(BLOCK)]
    keys, values = (torch.stack(t) for t in zip(*order))
    first = 0
    for i, (past, new) in enumerate(zip(_spread(case, "past"), _spread(case, "new"))):
        # the sequence's tokens from its open block on, as [kv, token, dim]
        r, base = past % BLOCK, past // BLOCK
        mine = slice(first, first + new)
        first += new
        for j, x in enumerate((k, v)):
            old = tail[i, j].view(kv, BLOCK, dim) if j == 0 else tail[i, j].view(kv, dim, BLOCK).transpose(1, 2)
            x = torch.cat((old[:, :r], x[mine].transpose(0, 1)), 1)
            n = (r + new) // BLOCK
            if n:
                pages = s["table"][i, base:base + n].long()
                y = x[:, :n * BLOCK].to(s["tail"].dtype).double().reshape(kv, n, BLOCK, dim).transpose(0, 1)
                scale = _two_to(torch.ceil(torch.log2(y.abs().amax((2, 3)) / 448)))
                y = _nearest_code(y / scale[..., None, None])
                scales[pages, j] = scale
                page = torch.empty(n, kv, BLOCK * dim, dtype=torch.float64, device=DEV)
                page[:, :, (keys, values)[j].flatten()] = y.flatten(2)
                codes[pages, j] = page
            left = x[:, n * BLOCK:]
            m = left.shape[1]
            if j == 0:
                tail[i, 0].view(kv, BLOCK, dim)[:, :m] = left
            else:
                tail[i, 1].view(kv, dim, BLOCK)[:, :, :m] = left.transpose(1, 2)
    return {"codes": codes, "scales": scales, "tail": tail, "query": q.transpose(0, 1)[None]}


def _sequence(case, s, i):
    """Keys and values of sequence i, [2, kv, tokens, dim] in 64 bits."""
    kv, dim, length = case["kv"], case["dim"], int(s["length"][i])
    n = length // BLOCK
    pages = s["table"][i, :n].long()
    x = s["codes"][pages].double() * s["scales"][pages].double()[..., None]
    order = [_token(BLOCK * dim, t) for t in range(BLOCK)]
    out = []
    for j, places in enumerate(zip(*order)):
        y = x[:, j][:, :, torch.stack(places).flatten()].view(n, kv, BLOCK, dim)
        end = s["tail"][i, j].double()
        end = end.view(kv, BLOCK, dim) if j == 0 else end.view(kv, dim, BLOCK).transpose(1, 2)
        out.append(torch.cat((y.transpose(0, 1).reshape(kv, n * BLOCK, dim), end[:, :length % BLOCK]), 1))
    return torch.stack(out)


def _exact_read(case, s):
    x = torch.cat([_sequence(case, s, i) for i in range(case["count"])], 2)
    return x[0][None], x[1][None]


def _exact_attn(case, s):
    heads, kv, dim = case["heads"], case["kv"], case["dim"]
    out, first = torch.empty(s["rows"], heads, dim, dtype=torch.float64, device=DEV), 0
    for i, (past, new) in enumerate(zip(_spread(case, "past"), _spread(case, "new"))):
        keys, values = _sequence(case, s, i)
        q = s["query"][0, :, first:first + new].double()
        row = torch.arange(past, past + new, device=DEV)[:, None]
        col = torch.arange(past + new, device=DEV)[None]
        hide = col > row
        if case["window"]:
            hide |= (col <= row - case["window"]) & (col >= case["sinks"])
        for h in range(heads):
            z = (q[h] @ keys[h * kv // heads].T) / math.sqrt(dim)
            w = torch.softmax(torch.where(hide, -math.inf, z), 1)
            out[first:first + new, h] = w @ values[h * kv // heads]
        first += new
    return out[None]
