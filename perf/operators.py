"""Operators around the attention half of a QLoRA decoder layer, each as a program calls it
(Qwen2.5-1.5B shape: hidden 1536, 12 query / 2 KV heads of 128, MLP 8960, packed rows).

Kinds of case:
  window  causal attention of packed rows in a sliding window, the first tokens (sinks) always
          visible: forward, or forward and backward (unpad.window_attention)
  drop    dropout from a counter-based generator, forward and backward (dropout.dropout)
  lora    a LoRA adapter's branch with dropout on its input, forward and all gradients
          (lora.adapter_branch)
  gemv    projections of a 4-bit layer for a few tokens (LayerGroup.nf4_gemv)

With `own` false a pass computes the same in elementary torch operations, in 32 bits, rounded
once at the end; `exact` restates each kind in 64 bits.
"""

import math

import numpy as np
import torch

own = False

HIDDEN, INTER, DIM, RANK = 1536, 8960, 128, 16
LAYER = ((1536, 1536), (256, 1536), (256, 1536), (1536, 1536), (8960, 1536), (8960, 1536),
         (1536, 8960))  # q, k, v, o, gate, up, down: (out, in)
BLOCK, BLOCK2 = 64, 256
SCALING = 2.0  # LoRA alpha / r = 32 / 16
SITE = 3       # which of a program's dropouts this is
NF4 = (-1.0, -0.6961928009986877, -0.5250730514526367, -0.39491748809814453,
       -0.28444138169288635, -0.18477343022823334, -0.09105003625154495, 0.0,
       0.07958029955625534, 0.16093020141124725, 0.24611230194568634, 0.33791524171829224,
       0.44070982933044434, 0.5626170039176941, 0.7229568362236023, 1.0)
DEV = "cuda"


def listed():
    return [
        # a batch of short prompts on a model of small windows: launch latency
        {"name": "window_short", "kind": "window", "lengths": "128 77 1 200", "heads": 12,
         "kv": 2, "window": 64, "sinks": 4, "dtype": "float16", "train": True},
        # the attention of 16 fine-tuning rows of 128..512 tokens on a sliding layer
        {"name": "window_sft", "kind": "window",
         "lengths": "245 503 280 139 512 128 377 461 190 333 256 418 299 147 505 222",
         "heads": 12, "kv": 2, "window": 256, "sinks": 0, "dtype": "float16", "train": True},
        # long-context fine-tuning: rows several windows long, the first tokens kept visible
        {"name": "window_long", "kind": "window", "lengths": "4096 3001 2222 1531", "heads": 12,
         "kv": 2, "window": 1000, "sinks": 4, "dtype": "float16", "train": True},
        # evaluation of one long document in bfloat16: forward only
        {"name": "window_eval", "kind": "window", "lengths": "8192", "heads": 12, "kv": 2,
         "window": 2047, "sinks": 128, "dtype": "bfloat16", "train": False},
        # dropout on a short batch's hidden states
        {"name": "drop_131", "kind": "drop", "rows": 131, "cols": HIDDEN, "p": 0.05,
         "dtype": "float16"},
        # dropout on the MLP activations of a full 4 x 512 batch
        {"name": "drop_act", "kind": "drop", "rows": 2048, "cols": INTER, "p": 0.1,
         "dtype": "bfloat16"},
        # q_proj's adapter for a typical batch of 4 rows of 128..512
        {"name": "lora_q_1312", "kind": "lora", "tokens": 1312, "in": HIDDEN, "out": 1536,
         "p": 0.05},
        # down_proj's adapter of a full batch
        {"name": "lora_down_2048", "kind": "lora", "tokens": 2048, "in": INTER, "out": 1536,
         "p": 0.1},
        # q|k|v of the one token a generating model is at
        {"name": "gemv_qkv_1", "kind": "gemv", "tokens": 1, "first": 0, "last": 3},
        # its MLP's gate|up
        {"name": "gemv_gate_up_1", "kind": "gemv", "tokens": 1, "first": 4, "last": 6},
        # the down projection of five sequences answered together
        {"name": "gemv_down_5", "kind": "gemv", "tokens": 5, "first": 6, "last": 7},
        # gate|up of a batch of 32 sequences
        {"name": "gemv_gate_up_32", "kind": "gemv", "tokens": 32, "first": 4, "last": 6},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(("window", "window", "drop", "lora", "gemv"))
    if kind == "window":
        count, longest = rng.randint(1, 8), _log(rng, 1, 3500)
        lengths = [longest] + [rng.randint(max(0, longest // 4), longest)
                               for _ in range(count - 1)]
        heads, kv = rng.choice(((12, 2), (12, 2), (14, 2), (16, 8), (8, 8)))
        while len(lengths) > 1 and heads * sum(n * n for n in lengths) > 2e8:
            lengths.pop()
        return {"kind": kind, "lengths": " ".join(map(str, lengths)), "heads": heads, "kv": kv,
                "window": _log(rng, 1, 4096), "sinks": rng.choice((0, 1, 4, 4, 16, 65, 200)),
                "dtype": rng.choice(("float16", "float16", "bfloat16")),
                "train": rng.random() < 0.7}
    if kind == "drop":
        return {"kind": kind, "rows": _log(rng, 1, 2048),
                "cols": rng.choice((HIDDEN, HIDDEN, INTER, 4864, 1001, 13)),
                "p": rng.choice((0.0, 0.05, 0.1, 0.3, 0.5)),
                "dtype": rng.choice(("float16", "bfloat16", "float32"))}
    if kind == "lora":
        rows, cols = rng.choice(LAYER + ((896, 896), (128, 896), (896, 4864)))
        return {"kind": kind, "tokens": _log(rng, 1, 2048), "in": cols, "out": rows,
                "p": rng.choice((0.05, 0.05, 0.1, 0.5))}
    first, last = rng.choice(((0, 3), (0, 1), (1, 2), (3, 4), (4, 6), (5, 6), (6, 7)))
    return {"kind": kind, "tokens": rng.choice((1, 1, 2, 3, rng.randint(4, 32))),
            "first": first, "last": last}


# -- inputs ----------------------------------------------------------------------------------------

def _gen(seed):
    return torch.Generator(DEV).manual_seed(seed)


def _randn(g, *shape, dtype=torch.float16, std=1.0, mean=0.0):
    return torch.randn(*shape, generator=g, device=DEV).mul_(std).add_(mean).to(dtype)


def _lengths(case):
    return [int(n) for n in case["lengths"].split()]


def _key(g):
    return torch.randint(0, 2 ** 62, (2,), generator=g, device=DEV)


def _second_level_table():
    """The 256 values of the second quantization: per decade 10^(i - 6), the midpoints of 2^i + 1
    points on [0.1, 1], both signs; 0 and 1."""
    values = [0.0, 1.0]
    for i in range(7):
        points = torch.linspace(0.1, 1.0, 2 ** i + 1, dtype=torch.float32)
        for sign in (1.0, -1.0):
            values += (sign * 10.0 ** (i - 6) * ((points[1:] + points[:-1]) / 2.0)).tolist()
    return torch.tensor(sorted(values), dtype=torch.float32)


def _window_inputs(case, seed):
    g, n, h, kv = _gen(seed), sum(_lengths(case)), case["heads"], case["kv"]
    dtype = getattr(torch, case["dtype"])
    # the projections' output: q, k and v are column views of one [N, q + k + v] buffer
    qkv = _randn(g, n, (h + 2 * kv) * DIM, dtype=dtype)
    bounds, views = (0, h, h + kv, h + 2 * kv), []
    for lo, hi in zip(bounds, bounds[1:]):
        view = qkv[:, lo * DIM:hi * DIM].view(n, hi - lo, DIM).transpose(0, 1)[None]
        views.append(view.detach().requires_grad_(case["train"]))
    lengths = torch.tensor([0] + _lengths(case))
    return {"views": views, "grad": _randn(g, 1, n, h, DIM, dtype=dtype, std=0.02),
            "lengths": _lengths(case), "longest": max(_lengths(case)),
            "cu": lengths.cumsum(0).to(DEV, torch.int32), "window": case["window"],
            "sinks": case["sinks"], "train": case["train"]}


def _drop_inputs(case, seed):
    g, shape, dtype = _gen(seed), (case["rows"], case["cols"]), getattr(torch, case["dtype"])
    return {"x": _randn(g, *shape, dtype=dtype).requires_grad_(),
            "grad": _randn(g, *shape, dtype=dtype, std=0.02), "key": _key(g), "p": case["p"]}


def _lora_inputs(case, seed):
    g, n = _gen(seed), case["tokens"]
    a = (torch.rand(RANK, case["in"], generator=g, device=DEV) * 2 - 1) * case["in"] ** -0.5
    return {"x": _randn(g, n, case["in"]).requires_grad_(),
            # an adapter in mid-training, in the fp16 copies that a forward reads
            "a": a.half().requires_grad_(), "b": _randn(g, case["out"], RANK, std=0.02)
            .requires_grad_(), "grad": _randn(g, n, case["out"], std=0.02), "key": _key(g),
            "p": case["p"]}


def _gemv_inputs(case, seed):
    g, parts = _gen(seed), []
    for rows, cols in LAYER:  # NF4 weights of std about 0.02
        n = rows * cols
        packed = torch.randint(0, 256, (n // 2,), generator=g, device=DEV, dtype=torch.uint8)
        absmax8 = torch.randint(0, 256, (n // BLOCK,), generator=g, device=DEV,
                                dtype=torch.uint8)
        scale2 = torch.rand(n // BLOCK // BLOCK2, generator=g, device=DEV) * 0.008 + 0.008
        parts.append((packed, absmax8, scale2, 0.04))
    return {"parts": parts, "biases": [_randn(g, LAYER[i][0], std=0.1) for i in range(3)],
            "code": _second_level_table().to(DEV),
            "x": _randn(g, case["tokens"], LAYER[case["first"]][1]),
            "first": case["first"], "last": case["last"]}


_INPUTS = {"window": _window_inputs, "drop": _drop_inputs, "lora": _lora_inputs,
           "gemv": _gemv_inputs}


def prepare(case, seed):
    s = {"kind": case["kind"], **_INPUTS[case["kind"]](case, seed)}
    if own and case["kind"] == "gemv":
        from talm_amd.nf4_linear import Linear4bit, QuantState, State2
        from talm_amd.qgroup import LayerGroup

        modules = []
        for i, ((rows, cols), (packed, absmax8, absmax2, offset)) in enumerate(
                zip(LAYER, s.pop("parts"))):
            m = Linear4bit(cols, rows, bias=i < 3, device=DEV)
            m.weight.data = packed.view(-1, 1)
            m.weight.quant_state = QuantState(absmax8, (rows, cols), s["code"], BLOCK,
                                              torch.tensor(offset, device=DEV),
                                              State2(absmax2, s["code"], BLOCK2))
            if i < 3:
                m.bias.data = s["biases"][i]
            modules.append(m)
        s["group"], s["modules"] = LayerGroup(modules), modules
    return s


# -- one pass --------------------------------------------------------------------------------------

def run(state):
    return (_OWN if own else _PLAIN)[state["kind"]](state)


def _own_window(s):
    from talm_amd.unpad import window_attention

    def call():
        return window_attention(*s["views"], s["cu"], s["longest"], DIM ** -0.5, s["window"],
                                s["sinks"])
    if not s["train"]:
        with torch.no_grad():
            return call()
    out = call()
    return (out, *torch.autograd.grad(out, s["views"], s["grad"]))


def _own_drop(s):
    from talm_amd.dropout import dropout

    y = dropout(s["x"], s["p"], s["key"], SITE)
    return (y, *torch.autograd.grad(y, s["x"], s["grad"]))


def _own_lora(s):
    from talm_amd.lora import adapter_branch

    y = adapter_branch(s["x"], s["a"], s["b"], SCALING, s["p"], s["key"], SITE)
    return (y, *torch.autograd.grad(y, (s["x"], s["a"], s["b"]), s["grad"]))


def _own_gemv(s):
    x, first, last = s["x"], s["first"], s["last"]
    out = torch.empty(x.shape[0], sum(LAYER[i][0] for i in range(first, last)),
                      dtype=torch.float16, device=DEV)
    s["group"].nf4_gemv(x, first, last, out)
    return out


def _plain_window(s):
    q, k, v = (t[0] for t in s["views"])  # [H, N, D]
    heads, kv, scale = q.shape[0], k.shape[0], DIM ** -0.5
    grad = s["grad"][0].transpose(0, 1)
    outs, start = [], 0
    for n in s["lengths"]:
        if n == 0:
            continue
        rows = slice(start, start + n)
        start += n
        i = torch.arange(n, device=DEV)
        seen = (i[None] <= i[:, None]) & ((i[:, None] - i[None] < s["window"])
                                          | (i[None] < s["sinks"]))
        parts = []
        for j in range(kv):  # the query heads of one KV head at a time
            span = slice(j * heads // kv, (j + 1) * heads // kv)
            qj, kj, vj = (t.detach().float() for t in (q[span, rows], k[j, rows], v[j, rows]))
            p = torch.matmul(qj, kj.t()).mul_(scale).masked_fill_(~seen, -math.inf)
            p = p.sub_(p.amax(-1, keepdim=True)).exp_()
            p = p.div_(p.sum(-1, keepdim=True))
            o = torch.matmul(p, vj)
            if not s["train"]:
                parts.append((o,))
                continue
            g = grad[span, rows].float()
            dv = torch.matmul(p.transpose(1, 2), g).sum(0, keepdim=True)
            ds = torch.matmul(g, vj.t()).sub_((g * o).sum(-1, keepdim=True)).mul_(p)
            parts.append((o, torch.matmul(ds, kj).mul_(scale),
                          torch.matmul(ds.transpose(1, 2), qj).sum(0, keepdim=True).mul_(scale),
                          dv))
        outs.append([torch.cat(t, 0) for t in zip(*parts)])
    o, *grads = (torch.cat(t, 1).to(q.dtype) for t in zip(*outs))
    o = o.transpose(0, 1)[None]
    return (o, *(t[None] for t in grads)) if s["train"] else o


def _keep(key, rows, cols, p):
    """Which elements of a [rows, cols] matrix stay: 16 random bits each, eight elements of a row
    from one 128-bit block of Philox-4x32 with ten rounds (Salmon, Moraes, Dror and Shaw, 2011),
    its counter (block low, block high, site, key[1] low), its key key[0]."""
    mask, per_row = 0xffffffff, (cols + 7) // 8
    block = torch.arange(rows * per_row, device=key.device)
    c = [block & mask, block >> 32, torch.full_like(block, SITE),
         (key[1] & mask).expand_as(block)]
    k0, k1 = key[0] & mask, (key[0] >> 32) & mask
    for _ in range(10):
        a, b = c[0] * 0xD2511F53, c[2] * 0xCD9E8D57
        c = [((b >> 32) & mask) ^ c[1] ^ k0, b & mask, ((a >> 32) & mask) ^ c[3] ^ k1, a & mask]
        k0, k1 = (k0 + 0x9E3779B9) & mask, (k1 + 0xBB67AE85) & mask
    bits = torch.stack([part for w in c for part in (w & 0xffff, w >> 16)], 1)
    return bits.view(rows, -1)[:, :cols] >= _threshold(p)


def _threshold(p):
    return min(int(round(p * 65536)), 65535)


def _plain_drop(s):
    x, factor = s["x"].detach(), 65536 / (65536 - _threshold(s["p"]))
    keep = _keep(s["key"], *x.shape, s["p"])
    return tuple(torch.where(keep, t.float() * factor, 0.0).to(t.dtype) for t in (x, s["grad"]))


def _plain_lora(s):
    x, a, b, g = (s[name].detach().float() for name in ("x", "a", "b", "grad"))
    keep, factor = _keep(s["key"], *x.shape, s["p"]), 65536 / (65536 - _threshold(s["p"]))
    xd = torch.where(keep, x * factor, 0.0)
    t = torch.mm(xd, a.t())
    u = torch.mm(g, b) * SCALING
    dx = torch.where(keep, torch.mm(u, a) * factor, 0.0)
    outs = (torch.mm(t, b.t()) * SCALING, dx, torch.mm(u.t(), xd), torch.mm(g.t(), t) * SCALING)
    return tuple(o.half() for o in outs)


def _weights(packed, absmax8, absmax2, offset, code):
    """The fp16 weights of NF4 codes: every product and sum rounded to fp32, then the weight to
    fp16, as the format defines them."""
    levels = torch.tensor(NF4, dtype=torch.float32, device=DEV)
    codes = torch.stack((packed >> 4, packed & 15), 1).reshape(-1).long()
    scale = code[absmax8.long()] * absmax2.repeat_interleave(BLOCK2)
    scale = scale + torch.tensor(offset, dtype=torch.float32, device=DEV)
    return (levels[codes].view(-1, BLOCK) * scale[:, None]).half().reshape(-1)


def _plain_gemv(s):
    x, outs = s["x"].float(), []
    for i in range(s["first"], s["last"]):
        y = torch.mm(x, _weights(*s["parts"][i], s["code"]).view(LAYER[i]).float().t())
        outs.append(y + s["biases"][i].float() if i < 3 else y)
    return torch.cat(outs, 1).half()


_OWN = {"window": _own_window, "drop": _own_drop, "lora": _own_lora, "gemv": _own_gemv}
_PLAIN = {"window": _plain_window, "drop": _plain_drop, "lora": _plain_lora,
          "gemv": _plain_gemv}


# -- what a pass cannot do without -----------------------------------------------------------------

def _pairs(case):
    """Visible (row, key) pairs of one head."""
    w, s, total = case["window"], case["sinks"], 0
    for n in _lengths(case):
        i = np.arange(n, dtype=np.int64)
        # the window's keys, and the sinks before the window
        total += int((np.minimum(i + 1, w) + np.minimum(np.maximum(i + 1 - w, 0), s)).sum())
    return total


def work(case):
    kind = case["kind"]
    if kind == "window":
        n, h, kv = sum(_lengths(case)), case["heads"], case["kv"]
        pairs, q, k = _pairs(case) * h, n * h * DIM * 2, n * kv * DIM * 2
        if not case["train"]:
            return {"bytes": 2 * q + 2 * k, "flops": 4 * DIM * pairs}
        # q, k, v, dout -> out, dq, dk, dv; two products forward, five backward
        return {"bytes": 4 * q + 4 * k, "flops": 14 * DIM * pairs}
    if kind == "drop":
        n = case["rows"] * case["cols"]
        return {"bytes": 4 * n * (4 if case["dtype"] == "float32" else 2), "flops": 2 * n}
    if kind == "lora":
        n, i, o = case["tokens"], case["in"], case["out"]
        # x, dy -> y, dx; A, B -> dA, dB
        return {"bytes": 4 * n * (i + o) + 4 * RANK * (i + o),
                "flops": 2 * n * RANK * (3 * i + 3 * o)}
    n = sum(LAYER[i][0] for i in range(case["first"], case["last"]))
    k, m = LAYER[case["first"]][1], case["tokens"]
    return {"bytes": n * k // 2 + n * k // BLOCK + 8 * (n * k // BLOCK // BLOCK2)
            + 2 * m * (n + k), "flops": 2 * m * n * k}


# -- the definition in 64 bits ---------------------------------------------------------------------

def exact(case, seed):
    return {"window": _exact_window, "drop": _exact_drop, "lora": _exact_lora,
            "gemv": _exact_gemv}[case["kind"]](case, seed)


def _exact_window(case, seed):
    s = _window_inputs(case, seed)
    q, k, v = (t.detach()[0].double() for t in s["views"])
    group = q.shape[0] // k.shape[0]
    grad = s["grad"][0].double()
    out = torch.empty_like(grad)
    dq, dk, dv = torch.empty_like(q), torch.zeros_like(k), torch.zeros_like(v)
    ends = np.cumsum(s["lengths"])
    for lo, hi in zip(ends - np.array(s["lengths"]), ends):
        for head in range(q.shape[0]):
            kh = head // group
            for r0 in range(int(lo), int(hi), 1024):  # 1024 rows against every key up to them
                r1 = min(r0 + 1024, int(hi))
                row = torch.arange(r0 - int(lo), r1 - int(lo), device=DEV)[:, None]
                col = torch.arange(r1 - int(lo), device=DEV)[None]
                hide = (col > row) | ((col <= row - case["window"]) & (col >= case["sinks"]))
                keys, values = k[kh, lo:r1], v[kh, lo:r1]
                z = (q[head, r0:r1] @ keys.T) / math.sqrt(DIM)
                w = torch.softmax(torch.where(hide, -math.inf, z), 1)
                out[r0:r1, head] = w @ values
                if case["train"]:
                    d = grad[r0:r1, head]
                    dw = d @ values.T
                    dz = w * (dw - (dw * w).sum(1, keepdim=True)) / math.sqrt(DIM)
                    dq[head, r0:r1] = dz @ keys
                    dk[kh, lo:r1] += dz.T @ q[head, r0:r1]
                    dv[kh, lo:r1] += w.T @ d
    return (out[None], dq[None], dk[None], dv[None]) if case["train"] else out[None]


def _exact_keep(key, rows, cols, p):
    """`_keep` from its definition, on the host in unsigned 64-bit words."""
    low, word = np.uint64(0xffffffff), np.uint64(32)
    key = key.cpu().numpy().astype(np.uint64)
    n = np.arange(rows * -(-cols // 8), dtype=np.uint64)
    x0, x1, x2, x3 = n & low, n >> word, np.full_like(n, SITE), np.full_like(n, key[1] & low)
    k0, k1 = int(key[0] & low), int(key[0] >> word)
    for step in range(10):
        a, b = x0 * np.uint64(0xD2511F53), x2 * np.uint64(0xCD9E8D57)
        r0 = np.uint64((k0 + step * 0x9E3779B9) % 2 ** 32)
        r1 = np.uint64((k1 + step * 0xBB67AE85) % 2 ** 32)
        x0, x1, x2, x3 = (b >> word) ^ x1 ^ r0, b & low, (a >> word) ^ x3 ^ r1, a & low
    words = np.stack((x0, x1, x2, x3), 1).astype("<u4")
    bits = words.view("<u2").reshape(rows, -1)[:, :cols].astype(np.int64)
    return torch.from_numpy(bits >= min(round(p * 65536), 65535)).to(DEV)


def _exact_drop(case, seed):
    s = _drop_inputs(case, seed)
    keep = _exact_keep(s["key"], case["rows"], case["cols"], case["p"]).double()
    share = 1 - min(round(case["p"] * 65536), 65535) / 65536
    return s["x"].detach().double() * keep / share, s["grad"].double() * keep / share


def _exact_lora(case, seed):
    s = _lora_inputs(case, seed)
    x, a, b, g = (s[name].detach().double() for name in ("x", "a", "b", "grad"))
    share = 1 - min(round(case["p"] * 65536), 65535) / 65536
    m = _exact_keep(s["key"], case["tokens"], case["in"], case["p"]).double() / share
    dt = SCALING * (g @ b)
    t = (x * m) @ a.T
    return SCALING * (t @ b.T), (dt @ a) * m, dt.T @ (x * m), SCALING * (g.T @ t)


def _exact_gemv(case, seed):
    s = _gemv_inputs(case, seed)
    x, outs = s["x"].double(), []
    for i in range(case["first"], case["last"]):
        packed, absmax8, absmax2, offset = s["parts"][i]
        # the weights are fp16 values that the format defines through fp32 products and sums
        scale = (s["code"][absmax8.long()].view(-1, BLOCK2) * absmax2[:, None]).view(-1) \
            + np.float32(offset).item()
        level = torch.tensor(NF4, device=DEV)
        w = torch.empty(packed.numel(), 2, device=DEV)
        w[:, 0], w[:, 1] = level[(packed // 16).long()], level[(packed % 16).long()]
        w = (w.view(-1, BLOCK) * scale[:, None]).half().double().view(LAYER[i])
        outs.append(x @ w.T + (s["biases"][i].double() if i < 3 else 0.0))
    return torch.cat(outs, 1)
