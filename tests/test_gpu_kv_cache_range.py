"""The 8-bit cache's attention (kv_cache.CacheLayer) at the ends of its ranges: values as large as their type
holds, and long sequences whose every part shows in the output. Tolerances are those of
test_gpu_kv_cache.py unless a test derives its own."""

import numpy as np
import pytest
import torch

from oracle import kv_cache as oracle
from talm_amd import _lib
from test_gpu_kv_cache import U, Case

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("dim,heads,past,new", [
    (128, 4, [70, 20, 1000], [1, 1, 1]),        # tiles of 16 rows in one part
    (64, 4, [3000, 500], [1, 2]),               # in parts, which are joined
    (128, 1, [20000], [1]),                     # in many
    (128, 6, [300, 2000], [40, 20]),            # tiles of 32 rows
    (64, 16, [130, 8700], [150, 450])])         # and of 64, in parts
def test_values_of_the_types_largest_magnitudes(dim, heads, past, new, dtype):
    """Outputs are means of values and no larger than the type's largest number, also where a code rounds
    past it (its values read as that number) and sums of many are past float32's."""
    most = torch.finfo(dtype).max
    c = Case(len(past), 1, dim, max(p + n for p, n in zip(past, new)), dtype, heads=heads)
    sign = torch.where(torch.arange(dim) % 3 == 0, -1.0, 1.0)

    def top(n):
        return (sign.expand(n, dim) * most).to(dtype).cuda()[None, None]

    def loud(n):
        return ((2 * torch.rand(n, dim, generator=c.g) - 1).double() * most).to(dtype).cuda()[None, None]

    for make in (top, loud):
        c.tokens = [t[:, :, :0] for t in c.tokens]
        c.append(past, v=make(sum(past)))
        c.append(new, v=make(sum(new)))
        out = c.check_attention(new)
        assert out.isfinite().all()
        if make is top:
            assert (out[0].sign().cpu() == sign).all()


@pytest.mark.parametrize("new", [1, 40])
def test_infinite_values_stay_infinite(new):
    """What is not finite in 16 bits is no large number: rows that see it are not finite."""
    for dtype in (torch.float16, torch.bfloat16):
        c = Case(1, 1, 64, 200, dtype, heads=2)
        v = c.rows(100 + new, 1)
        v[0, 0, 90, 5] = float("inf")
        c.append([100], v=v[:, :, :100])
        c.append([new], v=v[:, :, 100:])
        past = torch.tensor([100], dtype=torch.int32).cuda()
        out = c.layer.attention(c.rows(new, 2), torch.tensor([[0, new]], dtype=torch.int32).cuda(), past, new, 200, 0.125)
        assert not out[..., 5].isfinite().any() and out[..., :5].isfinite().all()


def test_operands_with_derivatives_are_refused():
    """Whoever wants a derivative, backwards or forwards, gets an error and not a result without one."""
    import torch.autograd.forward_ad as forward

    c = Case(2, 2, 64, 128, heads=4)
    c.append([70, 3])
    bounds, _ = c.spans([1, 1])
    past, k, q = torch.tensor([70, 3], dtype=torch.int32).cuda(), c.rows(2, 2), c.rows(2, 4)
    table = torch.zeros(2, 64, device="cuda")
    out = torch.empty(2, 2, 64, dtype=torch.float16, device="cuda")
    layer = c.layer

    def write(k=k, v=k, q=q, cos=table, sin=table, **parts):
        with_parts(parts).write(k, v, bounds, past, 1, q, (cos, sin))

    def attend(q=q, **parts):
        with_parts(parts).attention(q, bounds, past, 1, 128, 1.0)

    def read(out=out, **parts):
        with_parts(parts).read(past, bounds, past * 0, 1, 2, (out, out.detach().clone()))

    def with_parts(parts):
        names = ("codes", "scales", "tail", "table")
        return type(layer)(**{n: parts.get(n, getattr(layer, n)) for n in names})

    asked = [(write, "k", k), (write, "v", k), (write, "q", q), (write, "cos", table), (write, "sin", table),
             (attend, "q", q), (read, "out", out)]
    asked += [(f, n, getattr(layer, n)) for f in (write, attend, read) for n in ("scales", "tail")]
    for call, name, x in asked:
        call()
        wanted = x.detach().clone().requires_grad_()
        with pytest.raises(ValueError, match="gradient"):
            call(**{name: wanted})
        with torch.no_grad():
            call(**{name: wanted})
        with forward.dual_level():
            dual = forward.make_dual(x.detach().clone(), torch.ones_like(x))
            with pytest.raises(ValueError, match="gradient"):
                call(**{name: dual})
            with torch.no_grad(), pytest.raises(ValueError, match="gradient"):
                call(**{name: dual})
            with forward._set_fwd_grad_enabled(False):
                call(**{name: dual})


def test_more_workgroups_than_a_launch_takes():
    """600 sequences of 8 heads, the last of which brings 131072 tokens at once: 19.7 million workgroups of a write,
    and of a read, most of them of sequences that have one token. The same as that sequence alone."""
    from talm_amd.kv_cache import CacheLayer

    count, kv, dim, long = 600, 8, 64, 131072
    width, rows = long // 64 + 1, count - 1 + long
    i32 = {"dtype": torch.int32, "device": "cuda"}
    g = torch.Generator("cuda").manual_seed(0)
    k, v = (torch.randn(rows, kv, dim, generator=g, device="cuda").half().transpose(0, 1)[None] for _ in range(2))

    def layer(sequences, tables, pages):
        new = CacheLayer.allocate(sequences, kv, dim, 64)
        new.tail.zero_()
        return CacheLayer(torch.zeros(pages, 2, kv, 64 * dim, dtype=torch.uint8, device="cuda")
                          .view(torch.float8_e4m3fn), torch.zeros(pages, 2, kv, device="cuda"), new.tail, tables)

    table = torch.full((count, width), -1, **i32)
    table[-1] = torch.arange(width, **i32)
    table[:-1, 0] = width + torch.arange(count - 1, **i32)
    many = layer(count, table, width + count - 1)
    alone = layer(1, table[-1:], width)
    first = torch.arange(count, **i32)
    bounds, past = torch.stack((first, first + 1), 1), torch.zeros(count, **i32)
    bounds[-1, 1] = rows
    past[:-1] = 63  # their one token completes a block of what the tail held
    many.write(k, v, bounds, past, long)
    at = bounds[-1:] * 1
    alone.write(k, v, at, past[-1:], long)
    assert torch.equal(many.codes.view(torch.uint8)[:width], alone.codes.view(torch.uint8))
    assert torch.equal(many.scales[:width], alone.scales) and torch.equal(many.tail[-1], alone.tail[0])
    assert (many.codes.view(torch.uint8)[width:] != 0).flatten(2).any(2).all()
    length = torch.full((count,), 64, **i32)
    length[-1] = long
    got = many.read(length, bounds, past, long, rows)
    want = alone.read(length[-1:], at - (count - 1), past[-1:], long, long)
    for x, y, new in zip(got, want, (k, v)):
        assert torch.equal(x[:, :, count - 1:], y)
        # the short ones' scale is that of their one token: within half a step of a code
        few = x[:, :, :count - 1].float() - new[:, :, :count - 1].float()
        assert (few.abs() <= 2.0 ** -4 * new[:, :, :count - 1].float().abs() + 2.0 ** -17).all()


class Visible:
    """A sequence of T tokens whose 64-token blocks each have a key of their own, D random signs: a query of the same
    signs gives its block's tokens scores of 20 and others' about 20 / sqrt(D), so that nearly all of its weight
    lies there, and an output that lost, doubled or misplaced the block is off by hundreds of tolerances (planted()).

    Tolerance, without terms that grow with T. A wavefront sums n keys of at most one part, with weights relative to a
    reference of its own that is no larger than its largest score: rounded to fp16 they are off by 2^-11 of themselves,
    or 2^-25 where they are subnormal, which is n 2^-25 max|V| of an output, since a reference's weight is part of
    the sum; so is their sum. fp32 sums: n products, 4 wavefronts and at most 256 parts, 2^-24 each. Scores: D 2^-24
    of the sum of their magnitudes, exponents up to 2^5 twice (a weight's and its part's) 2^-19 each. The output: u."""

    def __init__(self, length, dim, dtype, heads, kv=1, new=1, seed=0):
        self.c = Case(1, kv, dim, length, dtype, seed=seed, heads=heads)
        self.blocks, self.length, self.new, g = -(-length // 64), length, new, self.c.g
        self.sign = torch.where(torch.rand(self.blocks, dim, generator=g) < 0.5, -1.0, 1.0)
        k = self.sign.repeat_interleave(64, 0)[:length, None].expand(length, kv, dim).to(dtype).cuda().transpose(0, 1)[None]
        v = self.c.rows(length, kv)
        for lo, hi in ((0, length - new), (length - new, length)):
            self.c.append([hi - lo], k=k[:, :, lo:hi], v=v[:, :, lo:hi])

    def parts(self, window=0, sinks=0):
        c = self.c
        size = _lib.lib().talm_cache_attn_workspace(self.new, c.heads, c.kv, c.dim, 1, self.new, self.length, window, sinks)
        return max(1, size // (self.new * c.heads * (c.dim + 2) * 4))

    def attend(self, targets, window=None, sinks=0):
        """targets [new, heads]: the block that each row and head looks at. Returns (query, output) [new, heads, D]."""
        c = self.c
        q = (self.sign[targets] * (20.0 / c.dim ** 0.5)).to(c.dtype).cuda()
        past = torch.tensor([self.length - self.new], dtype=torch.int32).cuda()
        bounds = torch.tensor([[0, self.new]], dtype=torch.int32).cuda()
        out = c.layer.attention(q.transpose(0, 1)[None], bounds, past, self.new, self.length, c.dim ** -0.5, window, sinks)
        return q.double().cpu().numpy(), out[0].double().cpu().numpy()

    def check(self, q, got, target, past, head=0, window=None, sinks=0):
        """Rows q, got [n, D] of one KV head that look at blocks `target` [n], at places past, past + 1, .."""
        c = self.c
        k, v = (x[head] for x in self.held)
        scale = c.dim ** -0.5
        want, size, score = oracle.attention(q, k, v, past, scale, window, sinks)
        visits = self.blocks if window is None else min(self.blocks, (window + 63) // 64 + 2 + (sinks + 63) // 64)
        n = 64 * -(-visits // self.parts(window or 0, sinks))
        rel = 2.0 ** -11 + 2 * (c.dim * 2.0 ** -24 * score + 2.0 ** -18) + (n + 260) * 2.0 ** -24
        tol = rel * (size + np.abs(want)) + U[c.dtype] * np.abs(want) + 2.0 ** -25 * (n * np.abs(v).max() + 1)
        worst = float((np.abs(got - want) / tol).max())
        planted = min(self.planted(x, w, t, k, v, y, p) for x, w, t, y, p in zip(q, want, tol, target, past + np.arange(len(q))))
        print(f"[case] {self.length} tokens, {self.parts(window or 0, sinks)} parts, D={c.dim} {c.dtype} window={window}: "
              f"worst {worst:.3f} of its tolerance, a lost block {planted:.0f}", flush=True)
        assert not np.isnan(got).any() and worst <= 1.0
        assert planted >= 20

    def planted(self, q, want, tol, k, v, block, place):
        """How many tolerances the output would be off without the block that the row looks at."""
        at = slice(64 * block, min(64 * block + 64, place + 1))
        s = q @ k[at].T * self.c.dim ** -0.5
        if not len(s):
            return np.inf
        # nearly all of the weight is the block's: what is left without it is a mean of the others, taken as 0
        p = np.exp(s - s.max())
        return float((np.abs(p @ v[at] / p.sum()) / tol).max())

    @property
    def held(self):
        if not hasattr(self, "_held"):
            self._held = self.c.values(0)
        return self._held


@pytest.mark.parametrize("length,parts", [(1500, 6), (3000, 12), (8999, 36), (65536, 256), (100001, 224)])
@pytest.mark.parametrize("dim,dtype", [(128, torch.float16), (64, torch.float16), (128, torch.bfloat16), (64, torch.bfloat16)])
def test_every_part_of_a_long_sequence_shows(length, parts, dim, dtype):
    """One token's 16 heads, in all of the join's forms; a block of every part, and every wavefront's in turn."""
    x = Visible(length, dim, dtype, 16)
    assert x.parts() == parts
    per = -(-x.blocks // parts)
    targets = np.array([min(r * per + r % per, x.blocks - 1) for r in range(-(-parts // 16) * 16)])
    outs = [x.attend(torch.from_numpy(targets[lo:lo + 16])[None]) for lo in range(0, len(targets), 16)]
    q, got = (np.concatenate([o[i][0] for o in outs]) for i in range(2))
    # each at the last token's place: as rows behind it they see the same keys
    x.check(q, got, targets, length - 1)


@pytest.mark.parametrize("dim,dtype", [(128, torch.float16), (64, torch.bfloat16)])
def test_every_part_of_a_long_window_shows(dim, dtype):
    length, window, sinks = 50001, 30000, 200
    x = Visible(length, dim, dtype, 16)
    seen = np.r_[0:3, (length - window) // 64 + 1:x.blocks]  # whole blocks but for the sinks' last and the newest
    targets = seen[np.linspace(0, len(seen) - 1, 16 * 12).astype(int)]
    for lo in range(0, len(targets), 16):
        q, got = x.attend(torch.from_numpy(targets[lo:lo + 16])[None], window, sinks)
        for h in range(16):
            x.check(q[:, h], got[:, h], targets[lo + h:lo + h + 1], length - 1, 0, window, sinks)


@pytest.mark.parametrize("length,new,heads,kv,dim,dtype", [
    (9000, 200, 12, 2, 128, torch.float16), (9000, 600, 12, 2, 128, torch.bfloat16), (7001, 20, 8, 2, 64, torch.float16),
    (700, 300, 4, 2, 64, torch.bfloat16)])
@pytest.mark.parametrize("window,sinks", [(None, 0), (3000, 100)])
def test_every_block_of_a_piece_shows(length, new, heads, kv, dim, dtype, window, sinks):
    """Tiles of 32 and 64 rows: every row and head looks at a block that it sees."""
    x = Visible(length, dim, dtype, heads, kv, new)
    past, g = length - new, np.random.default_rng(0)
    place = past + np.arange(new)[:, None]
    first = np.maximum(place - (window or length) + 1, 0) // 64 + 1  # whole blocks of a window
    first = np.minimum(first, place // 64)
    targets = first + (g.random((new, heads)) * (place // 64 - first + 1)).astype(int)
    q, got = x.attend(torch.from_numpy(targets), window, sinks)
    for h in range(heads):
        x.check(q[:, h], got[:, h], targets[:, h], past, h * kv // heads, window, sinks)


@pytest.mark.parametrize("dim,heads,length", [(64, 4, 300), (128, 16, 300), (64, 16, 3000), (128, 6, 5000), (64, 2, 40)])
def test_single_tokens_weights_are_of_32_bits(dim, heads, length):
    """Weights of a single token's rows are no coarser than fp32 sums: keys and queries of few bits, whose scores are
    exact, leave exponents below 2^4 with a product's and a subtraction's rounding (2^-20 of a weight, with exp2), two
    parts of 11 bits (2^-22, or 2^-25 of a reference's weight), sums of at most 128 tokens a wavefront, 4 of them and
    a few parts (256 2^-24 in all), and the output's half step."""
    c = Case(1, 1, dim, length, heads=heads)
    few = torch.tensor([-1.0, -0.5, 0.0, 0.5, 1.0])
    k = few[torch.randint(5, (length, dim), generator=c.g)].half().cuda()[None, None]
    c.append([length - 1], k=k[:, :, :-1])
    c.append([1], k=k[:, :, -1:])
    q = (torch.randint(-8, 9, (1, heads, 1, dim), generator=c.g) / 4).half().cuda()
    past = torch.tensor([length - 1], dtype=torch.int32).cuda()
    out = c.layer.attention(q, torch.tensor([[0, 1]], dtype=torch.int32).cuda(), past, 1, length, 0.125)
    (k,), (v,) = c.values(0)
    want, size, _ = oracle.attention(q[0, :, 0].double().cpu().numpy(), k, v, length - 1, 0.125)
    rel = 2.0 ** -20 + 2.0 ** -22 + 256 * 2.0 ** -24
    tol = rel * (size + np.abs(want)) + 2.0 ** -11 * np.abs(want) + 2.0 ** -25 * (128 * 2.0 ** -8 * np.abs(v).max() + 1)
    worst = (np.abs(out[0, 0].double().cpu().numpy() - want) / tol).max()
    print(f"[case] D={dim} {length} tokens: worst {worst:.3f} of its tolerance", flush=True)
    assert worst <= 1.0
