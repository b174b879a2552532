"""The 8-bit key and value cache (kv_cache.CacheLayer) against its definition on the CPU: what it holds
bit for bit, what is read back, and attention over it in float64.

Attention's tolerance counts roundings, u half a step of the operands' type (fp16 2^-11, bf16 2^-8):
P enters its product in fp16 (2^-11 relative, or 2^-25 where it is subnormal; a row's sum is at least 1
where P is formed), the tail's in two bfloat16 parts or fp16, no coarser, and so does its sum: with weights
p (1 + d), |d| <= 2^-11, the output is off by (sum p d v - out sum p d) / sum p (1 + d), at most
2^-11 (P|V| + |out|) (1 + 2^-10); the output is rounded (u, or 2^-25 where fp16 is subnormal); a score is
an fp32 sum of D products (D 2^-24 of the sum of their magnitudes, and P relatively so much) with exp2 and
the scale's product (2^-19 for exponents up to 2^5); P V sums at most T tokens (T 2^-24):
(2^-11 + 2 (D 2^-24 max sum |q k| scale + 2^-19) + T 2^-24) (P|V| + |out|) + u |out| + 2^-25 T max|V| + 2^-25."""

import numpy as np
import pytest
import torch

from oracle import kv_cache as oracle

pytestmark = pytest.mark.gpu

U = {torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}


class Case:
    """A cache on the GPU beside the 16-bit tokens that went into it. Its buffers begin as NaN and its
    pages lie in no order."""

    def __init__(self, sequences, kv, dim, capacity, dtype=torch.float16, seed=0, heads=None, spare=3):
        from talm_amd.kv_cache import CacheLayer

        self.g = torch.Generator().manual_seed(seed)
        self.kv, self.dim, self.dtype, self.heads = kv, dim, dtype, heads or kv
        layer = CacheLayer.allocate(sequences, kv, dim, capacity, dtype)
        width = layer.table.shape[1]
        pages = sequences * width + spare
        order = torch.randperm(pages, generator=self.g)[:sequences * width].to(torch.int32)
        codes = torch.full((pages, 2, kv, 64 * dim), 0x7f, dtype=torch.uint8, device="cuda")
        self.layer = CacheLayer(codes.view(torch.float8_e4m3fn),
                                torch.full((pages, 2, kv), float("nan"), device="cuda"),
                                torch.full_like(layer.tail, float("nan")), order.view(sequences, width).cuda())
        self.tokens = [np.zeros((2, kv, 0, dim)) for _ in range(sequences)]

    @property
    def past(self):
        return [t.shape[2] for t in self.tokens]

    def rows(self, n, heads, std=1.0, strided=True):
        """[1, heads, n, D] rows, as a column view of a wider buffer."""
        x = torch.randn(n, heads + (2 if strided else 0), self.dim, generator=self.g) * std
        return x.to(self.dtype).cuda()[:, :heads].transpose(0, 1)[None]

    def spans(self, new, gap=0):
        """bounds of `new` rows per sequence with `gap` rows between them; the rows in all."""
        ends = np.cumsum([n + gap for n in new])
        return torch.tensor([[e - n, e] for e, n in zip(ends, new)], dtype=torch.int32).reshape(-1, 2).cuda(), \
            int(ends[-1]) if len(new) else 0

    def write(self, new, gap=0, k=None, v=None, **more):
        bounds, n = self.spans(new, gap)
        k = self.rows(n, self.kv) if k is None else k
        v = self.rows(n, self.kv) if v is None else v
        past = torch.tensor(self.past, dtype=torch.int32).cuda()
        out = self.layer.write(k, v, bounds, past, max(new, default=0), **more)
        return out, k, v, bounds, past

    def keep(self, new, k, v, bounds):
        for b, (lo, hi) in enumerate(bounds.tolist()):
            x = torch.stack((k[0, :, lo:hi], v[0, :, lo:hi])).double().cpu().numpy()
            self.tokens[b] = np.concatenate((self.tokens[b], x), 2)

    def append(self, new, **more):
        _, k, v, bounds, _ = self.write(new, **more)
        self.keep(new, k, v, bounds)

    def check_held(self):
        """Codes, scales and tail bit for bit."""
        codes, scales = self.layer.codes.float().cpu().double().numpy(), self.layer.scales.cpu().numpy()
        tail, table = self.layer.tail.double().cpu().numpy(), self.layer.table.cpu().numpy()
        for b, t in enumerate(self.tokens):
            n = t.shape[2] // 64
            for which in range(2):
                for h in range(self.kv):
                    for block in range(n):
                        want, scale = oracle.quantize(t[which, h, block * 64:(block + 1) * 64])
                        want = (oracle.value_order if which else oracle.key_order)(want)
                        page = table[b, block]
                        assert scales[page, which, h] == scale, (b, block, which, h)
                        np.testing.assert_array_equal(codes[page, which, h], want)
                    rest = t[which, h, n * 64:]
                    got = tail[b, which, h].reshape(self.dim, 64).T if which else \
                        tail[b, which, h].reshape(64, self.dim)
                    np.testing.assert_array_equal(got[:len(rest)], rest)

    def values(self, b, top=None):
        t = self.tokens[b]
        return np.stack([[oracle.held(t[i, h], top) for h in range(self.kv)] for i in range(2)])

    def check_attention(self, new, window=None, sinks=0, gap=0, std=1.0, q=None):
        """Attention of the last `new` tokens of each sequence."""
        print(f"[case] attention lengths={self.past} new={new} heads={self.heads}/{self.kv} D={self.dim} "
              f"{self.dtype} window={window} sinks={sinks}", flush=True)
        bounds, n = self.spans(new, gap)
        past = [t - n_ for t, n_ in zip(self.past, new)]
        q = self.rows(n, self.heads, std) if q is None else q
        scale = self.dim ** -0.5
        out = self.layer.attention(q, bounds, torch.tensor(past, dtype=torch.int32).cuda(), max(new), max(self.past),
                                   scale, window, sinks)
        assert out.shape == (1, n, self.heads, self.dim) and out.dtype == self.dtype
        got, worst = out[0].double().cpu().numpy(), 0.0
        sub = 2.0 ** -25
        for b, (lo, hi) in enumerate(bounds.tolist()):
            k, v = self.values(b)
            for h in range(self.heads):
                j = h * self.kv // self.heads
                x = q[0, h, lo:hi].double().cpu().numpy()
                want, size, score = oracle.attention(x, k[j], v[j], past[b], scale, window, sinks)
                length = k.shape[1]
                rel = 2.0 ** -11 + 2 * (self.dim * 2.0 ** -24 * score + 2.0 ** -19) + length * 2.0 ** -24
                tol = rel * (size + np.abs(want)) + U[self.dtype] * np.abs(want) \
                    + sub * (length * np.abs(v[j]).max(initial=0.0) + 1)
                err = np.abs(got[lo:hi, h] - want)
                assert not np.isnan(err).any()
                worst = max(worst, float((err / tol).max(initial=0.0)))
        print(f"  worst {worst:.3f} of its tolerance", flush=True)
        assert worst <= 1.0
        return out


SHAPES = [(2, 128, torch.float16), (1, 64, torch.bfloat16), (3, 64, torch.float16), (8, 128, torch.bfloat16)]


@pytest.mark.parametrize("kv,dim,dtype", SHAPES)
def test_pages_and_tails_bit_for_bit(kv, dim, dtype):
    """Calls that begin and end anywhere in a block, of none, one and many tokens, with rows between the
    sequences'."""
    c = Case(4, kv, dim, 400, dtype)
    for new in ([0, 1, 63, 64], [1, 62, 1, 1], [63, 1, 64, 127], [130, 0, 129, 5], [1, 1, 1, 1], [2, 65, 7, 0]):
        print(f"[case] write {new} behind {c.past} kv={kv} D={dim} {dtype}", flush=True)
        c.append(new, gap=2)
        c.check_held()


def test_contents_do_not_depend_on_the_calls():
    a, b = Case(1, 2, 128, 512, seed=4), Case(1, 2, 128, 512, seed=4)
    k, v = (a.rows(333, 2, s) for s in (3.0, 1.0))
    a.append([333], k=k, v=v)
    lo = 0
    for n in (1, 62, 1, 1, 64, 100, 0, 27, 77):
        b.append([n], k=k[:, :, lo:lo + n], v=v[:, :, lo:lo + n])
        lo += n
    assert lo == 333
    page = a.layer.table[0, :5].long()
    assert torch.equal(a.layer.table, b.layer.table)
    for name in ("codes", "scales"):
        x, y = (getattr(c.layer, name)[page] for c in (a, b))
        assert torch.equal(x.float(), y.float()), name
    for which, shape in ((0, (2, 64, 128)), (1, (2, 128, 64))):
        x, y = (c.layer.tail[0, which].view(shape) for c in (a, b))
        x, y = (t[:, :13] if which == 0 else t[:, :, :13] for t in (x, y))
        assert torch.equal(x, y)


def _magnitudes(dtype, g):
    """Ten blocks [640, 64]: of zeros, of subnormals, of the type's largest numbers, with one loud value, on
    the border of a scale, and every value of a code and halfway between two."""
    k = torch.randn(64 * 10, 64, generator=g)
    big = torch.finfo(dtype).max
    k[0:64] = 0
    k[64:128] *= 2.0 ** -20 if dtype == torch.float16 else 2.0 ** -120
    k[128:192] = big * torch.linspace(-1, 1, 64)
    k[192:256] *= 2.0 ** -6
    k[200, 5] = 300.0
    k[256:320] = 448.0 * torch.rand(64, 64, generator=g)  # a scale of 1 exactly
    k[256, 0] = 448.0
    k[320:384] = k[256:320]
    k[330, 1] = 448.5 if dtype == torch.float16 else 450.0  # the next scale
    codes = torch.arange(256, dtype=torch.uint8).view(torch.float8_e4m3fn).float()
    codes = codes[codes.isfinite()].sort().values
    k[384:448].view(-1)[:254] = codes                       # every code, and the ties between them
    k[384:448].view(-1)[300:553] = (codes[1:] + codes[:-1]) / 2
    k[448:512] = -0.0
    k[512:576] = torch.finfo(dtype).smallest_normal * torch.rand(64, 64, generator=g)
    return k.to(dtype).cuda()[None, None]


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
def test_codes_of_every_magnitude(dtype):
    c = Case(1, 1, 64, 64 * 16, dtype)
    k = _magnitudes(dtype, c.g)
    v = k.flip(2).contiguous()
    c.append([640], k=k, v=v)
    c.check_held()
    one = torch.tensor([640], dtype=torch.int32).cuda()
    got = c.layer.read(one, torch.tensor([[0, 640]], dtype=torch.int32).cuda(), one * 0, 640, 640)
    for x, want in zip(got, c.values(0, torch.finfo(dtype).max)):
        np.testing.assert_array_equal(x[0].double().cpu().numpy(), want)


def test_values_that_are_not_finite_are_nan_in_a_page():
    c = Case(1, 1, 64, 256)
    k = c.rows(128, 1, strided=False).clone()
    k[0, 0, 3, 4], k[0, 0, 70, 1], k[0, 0, 71, 2] = float("inf"), float("nan"), float("-inf")
    c.append([128], k=k)
    want = [oracle.quantize(k[0, 0, lo:lo + 64].double().cpu().numpy()) for lo in (0, 64)]
    for block, (codes, scale) in enumerate(want):
        page = int(c.layer.table[0, block])
        assert c.layer.scales[page, 0, 0].item() == scale
        got = c.layer.codes[page, 0, 0].float().cpu().double().numpy()
        np.testing.assert_array_equal(got, oracle.key_order(codes))
        assert np.isnan(got).sum() == block + 1


@pytest.mark.parametrize("dim,dtype", [(128, torch.float16), (64, torch.bfloat16)])
def test_rotary_positions_on_the_way(dim, dtype):
    """The turned queries and keys: in fp16 bit for bit those of rope_ and a plain write; in both types at
    most a rounding (u) and fp32's two (2^-23 of the terms) from float64."""
    from talm_amd.rope import rope_

    c, d = Case(3, 2, dim, 300, dtype, seed=7), Case(3, 2, dim, 300, dtype, seed=7)
    for step, new in enumerate(([70, 1, 127], [1, 1, 1], [60, 64, 0])):
        n = sum(new)
        q, k, v = c.rows(n, 6), c.rows(n, 2), c.rows(n, 2)
        angle = torch.rand(n, dim, generator=c.g) * 6.3
        # tables with a row stride of their own
        cos, sin = (torch.cat((t, t), 1).cuda()[:, :dim] for t in (angle.cos(), angle.sin()))
        got, _, _, bounds, _ = c.write(new, k=k, v=v, query=q, rope=(cos, sin))
        turned = []
        for x in (q, k):
            a, b = x[0].transpose(0, 1).double().chunk(2, 2)
            (ca, cb), (sa, sb) = (t.double()[:, None].chunk(2, 2) for t in (cos, sin))
            want = torch.cat((a * ca - b * sa, b * cb + a * sb), 2)
            size = torch.cat((a.abs() * ca.abs() + b.abs() * sa.abs(), b.abs() * cb.abs() + a.abs() * sb.abs()), 2)
            turned.append((want, U[dtype] * want.abs() + 2.0 ** -23 * size + 2.0 ** -25))
        assert got.shape == q.shape and got.dtype == dtype
        assert ((got[0].transpose(0, 1).double() - turned[0][0]).abs() <= turned[0][1]).all()
        if dtype == torch.float16:
            q2, k2 = q[0].transpose(0, 1).clone(), k[0].transpose(0, 1).clone()
            rope_(q2, k2, cos, sin)
            assert torch.equal(got[0].transpose(0, 1), q2)
        else:
            # the keys as the kernel rounded them, from a cache whose tail holds them all
            k2 = Case(1, 2, dim, 64, dtype)
            flat = torch.empty(n, 2, dim, dtype=dtype, device="cuda")
            for lo in range(0, n, 63):
                m = min(63, n - lo)
                k2.tokens[0] = np.zeros((2, 2, 0, dim))
                k2.write([m], k=k[:, :, lo:lo + m], v=v[:, :, lo:lo + m], rope=(cos[lo:lo + m], sin[lo:lo + m]))
                flat[lo:lo + m] = k2.layer.tail[0, 0].view(2, 64, dim)[:, :m].transpose(0, 1)
            k2 = flat
        assert ((k2.double() - turned[1][0]).abs() <= turned[1][1]).all()
        k2 = k2.transpose(0, 1)[None]
        d.write(new, k=k2, v=v)
        c.keep(new, k2, v, bounds)
        d.tokens = c.tokens
        c.check_held()
        for name in ("codes", "scales", "tail"):
            a, b = (getattr(x.layer, name).contiguous().view(torch.uint8) for x in (c, d))
            assert torch.equal(a, b), (step, name)


@pytest.mark.parametrize("kv,dim,dtype", SHAPES)
def test_read_back(kv, dim, dtype):
    """Whole caches, and pieces from anywhere to anywhere, over the end of a sequence too."""
    c = Case(4, kv, dim, 320, dtype)
    c.append([0, 61, 64, 200])
    c.append([1, 3, 64, 99])
    top = 65504.0 if dtype == torch.float16 else None
    length = torch.tensor(c.past, dtype=torch.int32).cuda()
    for past, new in (([0] * 4, c.past), ([0, 10, 63, 130], [1, 53, 2, 150]), ([0, 60, 120, 290], [3, 10, 20, 30])):
        print(f"[case] read {new} from {past} of {c.past}", flush=True)
        bounds, n = c.spans(new, gap=1)
        out = tuple(torch.full((n, kv, dim), 7.0, dtype=dtype, device="cuda") for _ in range(2))
        start = torch.tensor(past, dtype=torch.int32).cuda()
        got = c.layer.read(length, bounds, start, max(new), n, out)
        assert all(g.shape == (1, kv, n, dim) and g.data_ptr() == o.data_ptr() for g, o in zip(got, out))
        free = np.ones(n, bool)
        for b, (lo, hi) in enumerate(bounds.tolist()):
            free[lo:hi] = False
            want = np.zeros((2, kv, new[b], dim))
            there = max(0, min(new[b], c.past[b] - past[b]))
            want[:, :, :there] = c.values(b, top)[:, :, past[b]:past[b] + there]
            for i in range(2):
                np.testing.assert_array_equal(got[i][0, :, lo:hi].double().cpu().numpy(), want[i])
        assert all((o[torch.from_numpy(free).cuda()] == 7.0).all() for o in out)


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
def test_read_saturates_at_the_largest_number(dtype):
    c, most = Case(1, 1, 64, 64, dtype), torch.finfo(dtype).max
    c.append([64], k=torch.full((1, 1, 64, 64), most, dtype=dtype, device="cuda"))
    one = torch.tensor([64], dtype=torch.int32).cuda()
    k, _ = c.layer.read(one, torch.tensor([[0, 64]], dtype=torch.int32).cuda(), one * 0, 64, 64)
    assert (k == most).all()


@pytest.mark.parametrize("heads,kv,dim,dtype", [
    (12, 2, 128, torch.float16), (14, 2, 64, torch.bfloat16), (8, 8, 128, torch.bfloat16), (16, 1, 64, torch.float16),
    (40, 2, 128, torch.float16)])
def test_attention_of_single_tokens(heads, kv, dim, dtype):
    """Lengths around the borders of a page and of a workgroup's part, with sequences that have no new token."""
    c = Case(9, kv, dim, 1100, dtype, heads=heads)
    c.append([0, 62, 63, 64, 65, 127, 255, 1000, 0])
    c.append([1, 1, 1, 1, 1, 1, 1, 1, 0])
    c.check_attention([1, 1, 1, 1, 1, 1, 1, 1, 0])
    c.check_attention([1, 0, 1, 1, 0, 1, 1, 1, 0], gap=3, std=8.0)


@pytest.mark.parametrize("heads,kv,dim,dtype", [
    (12, 2, 128, torch.float16), (14, 2, 64, torch.float16), (4, 4, 128, torch.bfloat16), (8, 1, 64, torch.bfloat16)])
def test_attention_of_pieces(heads, kv, dim, dtype):
    c = Case(5, kv, dim, 700, dtype, heads=heads)
    c.append([0, 100, 63, 500, 128])
    new = [130, 37, 2, 64, 1]
    c.append(new)
    c.check_attention(new)
    c.check_attention([130, 5, 0, 1, 70], gap=1)


@pytest.mark.parametrize("window,sinks", [(1, 0), (1, 1), (5, 2), (64, 0), (65, 4), (200, 70), (333, 0), (2 ** 31 - 1, 5)])
@pytest.mark.parametrize("new", [1, 50])
def test_attention_in_a_window(window, sinks, new):
    c = Case(4, 2, 128, 900, torch.bfloat16 if window == 65 else torch.float16, heads=6)
    c.append([10, 64, 300, 800])
    c.append([new, new, 3, new])
    c.check_attention([new, new, 3, new], window, sinks)


@pytest.mark.parametrize("length,dim,dtype", [
    (500, 128, torch.float16), (1100, 64, torch.float16), (3000, 128, torch.bfloat16), (3000, 64, torch.float16), (20000, 128, torch.float16),
    (20000, 64, torch.bfloat16)])
def test_attention_of_long_sequences(length, dim, dtype):
    """Keys split over a few, over some and over many workgroups, whose parts are joined in three ways."""
    c = Case(2, 1, dim, length + 1, dtype, heads=3)
    c.append([length, length // 5])
    c.append([1, 1])
    c.check_attention([1, 1])
    c.check_attention([1, 1], window=length // 2, sinks=100)


@pytest.mark.parametrize("heads,kv,dim,dtype", [
    (16, 8, 64, torch.float16), (16, 8, 128, torch.bfloat16), (12, 2, 128, torch.float16)])
def test_attention_of_long_pieces(heads, kv, dim, dtype):
    """Tiles of 32 rows, and of 64 in parts; a sequence without new tokens; masks of windows inside a tile."""
    c = Case(3, kv, dim, 9400, dtype, heads=heads)
    c.append([2000, 300, 8700])
    new = [130, 0, 650 if kv == 2 else 450]
    c.append(new)
    c.check_attention(new)
    c.check_attention([3, 1, new[2]], window=700, sinks=5)


@pytest.mark.parametrize("dim,dtype", [
    (64, torch.float16), (64, torch.bfloat16), (128, torch.float16), (128, torch.bfloat16)])
def test_attention_of_prompts(dim, dtype):
    """Tiles of 64 rows, more than the CUs hold at once, of sequences of other lengths and of none."""
    c = Case(6, 4, dim, 460, dtype, heads=16)
    c.append([0, 40, 0, 17, 0, 0])
    new = [400, 390, 256, 400, 0, 400]
    c.append(new)
    c.check_attention(new)
    c.check_attention(new, window=70, sinks=3)


@pytest.mark.parametrize("new", [1, 9])
def test_attention_of_more_sequences_than_a_wavefront_counts(new):
    c = Case(131, 1, 64, 200, heads=4)
    c.append([(i * 37) % 150 for i in range(131)])
    rows = [0 if i % 7 == 3 else 1 + i % new for i in range(131)]
    c.append(rows)
    c.check_held()
    c.check_attention(rows)


def test_attention_of_loud_keys_and_quiet_values():
    """Scales far from 1, and different from page to page."""
    c = Case(2, 2, 128, 700, torch.float16, heads=4)
    for i in range(10):
        n = 64
        c.append([n, n], k=c.rows(2 * n, 2, 2.0 ** (i - 6)), v=c.rows(2 * n, 2, 2.0 ** (3 * i - 18)))
    c.append([1, 5])
    c.check_attention([1, 5], std=0.1)


@pytest.mark.parametrize("dim,dtype,heads", [
    (128, torch.bfloat16, 4), (64, torch.float16, 12), (128, torch.float16, 16), (64, torch.bfloat16, 16)])
def test_pieces_over_loud_keys_and_quiet_values(dim, dtype, heads):
    """The same in tiles of 32 rows, from loud pages to quiet ones and back."""
    c = Case(2, 2, dim, 1200, dtype, heads=heads)
    for i in range(11):
        n, loud = 64 if i % 3 else 50, 5 - abs(i - 5)
        c.append([n, n], k=c.rows(2 * n, 2, 2.0 ** -loud), v=c.rows(2 * n, 2, 2.0 ** (12 - 3 * (i % 7))))
    c.append([90, 400])
    c.check_attention([90, 400], std=0.3)
    c.check_attention([90, 30], window=100, sinks=70, std=0.3)


@pytest.mark.parametrize("bad", [float("nan"), float("inf")])
@pytest.mark.parametrize("dim,dtype,new", [
    (128, torch.float16, [1, 60]), (64, torch.bfloat16, [3, 150]), (128, torch.bfloat16, [130, 1]),
    (64, torch.float16, [1, 1])])
def test_keys_that_are_not_finite(dim, dtype, new, bad):
    """A key that is not finite, in a page and in the tail: rows that see it are NaN (an infinity in the tail
    keeps its sign there: a row whose query turns it into a score of -inf gives it no weight), rows that do
    not see it have the bits that they have without it, other heads too."""
    bounds, n = Case(2, 2, dim, 1).spans(new)
    (_, one), (_, two) = bounds.tolist()
    q = Case(1, 1, dim, 1, dtype, seed=9).rows(n, 8)

    def spoiled(lo, hi, column, place, total):
        """[rows, 4] of the second KV head's heads: which rows' outputs are NaN."""
        held_as_nan = bad != bad or place // 64 < total // 64
        return torch.ones(hi - lo, 4, dtype=torch.bool) if held_as_nan else (q[0, 4:, lo:hi, column] > 0).T.cpu()

    def both(past, window=None, sinks=0):
        past = torch.tensor(past, dtype=torch.int32).cuda()
        return (x.layer.attention(q, bounds, past, max(new), 2300, dim ** -0.5, window, sinks) for x in (c, d))

    def check(got, want, nan):
        assert want.isfinite().all() and torch.equal(got[:, :, :4], want[:, :, :4])
        assert torch.equal(got[0, :, 4:].isnan().all(2).cpu(), nan)
        assert torch.equal(got[0, :, 4:].isnan().any(2).cpu(), nan)

    c, d = (Case(2, 2, dim, 2300, dtype, seed=5, heads=8) for _ in range(2))
    long = 2170
    for i, x in enumerate((c, d)):
        k, v = x.rows(long + 100, 2), x.rows(long + 100, 2)
        if i == 0:
            k[0, 1, 40, 7] = k[0, 1, long + 99, 0] = bad
        x.append([long, 100], k=k, v=v)
        x.append(new)
    nan = torch.cat((spoiled(0, one, 7, 40, long + new[0]), spoiled(one, two, 0, 99, 100 + new[1])))
    check(*both([long, 100]), nan)
    got, want = both([long, 100], window=200, sinks=3)  # leaves the first sequence's out
    nan[:one] = False
    check(got, want, nan)
    assert torch.equal(got[:, :one], want[:, :one])

    # among the new tokens: the rows in front of it do not see it
    c, d = (Case(2, 2, dim, 400, dtype, seed=6, heads=8) for _ in range(2))
    nan = torch.zeros(n, 4, dtype=torch.bool)
    for i, x in enumerate((c, d)):
        x.append([130, 100])
        k, v = x.rows(n, 2), x.rows(n, 2)
        if i == 0:
            for (lo, hi), past in zip(bounds.tolist(), (130, 100)):
                at = (lo + hi) // 2
                k[0, 1, at, 3] = bad
                nan[at:hi] = spoiled(at, hi, 3, past + at - lo, past + hi - lo)
        x.append(new, k=k, v=v)
    got, want = both([130, 100])
    check(got, want, nan)
    for lo, hi in bounds.tolist():
        assert torch.equal(got[:, lo:(lo + hi) // 2], want[:, lo:(lo + hi) // 2])


def test_attention_over_shared_pages():
    """Two sequences with a common beginning whose complete pages are the same."""
    c = Case(2, 1, 128, 300, heads=2)
    c.append([130, 0])
    c.layer.table[1, :2] = c.layer.table[0, :2]
    c.layer.tail[1] = c.layer.tail[0]
    c.tokens[1] = c.tokens[0]
    c.append([3, 90])
    c.check_held()
    c.check_attention([3, 90])


def test_places_that_hold_no_page():
    """Table entries outside the pool: their tokens are dropped, read as zeros and seen by nobody."""
    c = Case(1, 1, 64, 320, heads=2, spare=0)
    pages = c.layer.codes.shape[0]
    whole = c.layer.table.clone()
    for bad in (-1, pages, 2 ** 31 - 1, -2 ** 31):
        c.tokens[0] = np.zeros((2, 1, 0, 64))
        c.layer.table.copy_(whole)
        c.layer.table[0, 1] = bad
        before = c.layer.codes.view(torch.uint8).clone()
        c.append([200])
        lost = whole[0, 1].long()
        assert torch.equal(c.layer.codes.view(torch.uint8)[lost], before[lost])
        one = torch.tensor([200], dtype=torch.int32).cuda()
        k, v = c.layer.read(one, torch.tensor([[0, 200]], dtype=torch.int32).cuda(), one * 0, 200, 200)
        assert (k[0, 0, 64:128] == 0).all() and (v[0, 0, 64:128] == 0).all() and (k[0, 0, :64] != 0).any()
        q = c.rows(1, 2)
        out = c.layer.attention(q, torch.tensor([[0, 1]], dtype=torch.int32).cuda(), one - 1, 1, 200, 0.125)
        held = c.values(0)[:, 0]
        there = np.r_[0:64, 128:200]
        for h in range(2):
            want, size, _ = oracle.attention(q[0, h].double().cpu().numpy(), held[0][there], held[1][there],
                                             len(there) - 1, 0.125)
            # the rounding of P and of the output, and 2^-12 for the rest of the module's bound
            assert (np.abs(out[0, :, h].double().cpu().numpy() - want) <= 2.0 ** -10 * size + 2.0 ** -12).all()


def test_rows_that_see_nothing_are_zero():
    c = Case(1, 1, 64, 192, heads=2)
    c.append([130])
    c.layer.table[0] = -1
    one = torch.tensor([63], dtype=torch.int32).cuda()
    out = c.layer.attention(c.rows(1, 2), torch.tensor([[0, 1]], dtype=torch.int32).cuda(), one, 1, 64, 0.125)
    assert (out == 0).all()


def test_what_does_not_fit_is_left_out():
    """Bounds outside the rows, counts past max_new or past the table, and negative pasts write nothing
    out of place."""
    c = Case(6, 1, 64, 128, heads=2, spare=0)
    n = 200
    k, v, q = c.rows(n, 1), c.rows(n, 1), c.rows(n, 2)
    bounds = torch.tensor([[0, 5], [-7, 3], [190, 400], [60, 50], [10, 2 ** 31 - 1], [-2 ** 31, 2 ** 31 - 1]],
                          dtype=torch.int32).cuda()
    past = torch.tensor([-1, 0, 126, 0, 2 ** 31 - 1, 127], dtype=torch.int32).cuda()
    tail, codes = c.layer.tail.clone(), c.layer.codes.view(torch.uint8).clone()
    c.layer.write(k, v, bounds, past, 64)
    # sequence 1: rows 0 .. 2 as tokens 0 .. 2; 2: rows 190, 191 as tokens 126, 127, which complete its
    # second block; 5: row 0 as token 127, which does too; the others nothing
    got = c.layer.tail[1, 0, 0].view(64, 64)
    assert torch.equal(got[:3], k[0, 0, :3]) and got[3:].isnan().all()
    for b in (0, 2, 3, 4, 5):
        assert torch.equal(c.layer.tail[b].view(torch.int16), tail[b].view(torch.int16)), b
    changed = (c.layer.codes.view(torch.uint8) != codes).flatten(1).any(1).nonzero().flatten().tolist()
    assert set(changed) <= {int(c.layer.table[2, 1]), int(c.layer.table[5, 1])}
    out = c.layer.attention(q, bounds, past, 64, 128, 0.125)
    want = torch.nn.functional.scaled_dot_product_attention(
        q[0, :, :3].float(), k[0, :, :3].float().expand(2, 3, 64), v[0, :, :3].float().expand(2, 3, 64),
        is_causal=True, scale=0.125)
    # sequence 5's row 0 overlaps sequence 1's; rows 1 and 2 are its own
    torch.testing.assert_close(out[0, 1:3].transpose(0, 1).float(), want[:, 1:], rtol=2e-3, atol=2e-3)
    k2, v2 = (torch.full((n, 1, 64), 7.0, dtype=torch.float16, device="cuda") for _ in range(2))
    length = torch.tensor([5, 3, 128, -1, 2 ** 31 - 1, 128], dtype=torch.int32).cuda()
    c.layer.read(length, bounds[:5].clone().resize_(6, 2).copy_(torch.tensor(
        [[0, 5], [-7, 3], [190, 400], [60, 50], [10, 2 ** 31 - 1], [7, 7]])), past, 64, n, (k2, v2))
    assert torch.equal(k2[:3, 0], k[0, 0, :3]) and (k2[3:190] == 7).all() and (k2[192:] == 7).all()


def test_pools_past_32_bit_offsets():
    """Pages whose codes lie more than 4 GiB into the pool."""
    from talm_amd.kv_cache import CacheLayer

    c = Case(1, 2, 128, 300, heads=4)
    pages = 135000
    layer = CacheLayer(torch.empty(pages, 2, 2, 64 * 128, dtype=torch.uint8, device="cuda")
                       .view(torch.float8_e4m3fn), torch.empty(pages, 2, 2, device="cuda"), c.layer.tail,
                       torch.tensor([[pages - 1, 3, pages - 2, 132000, 70000]], dtype=torch.int32).cuda())
    c.layer = layer
    c.append([290])
    c.append([1])
    codes = layer.codes[layer.table[0].long()]  # the few that are looked at
    c.layer = CacheLayer(codes.contiguous(), layer.scales[layer.table[0].long()].contiguous(), layer.tail,
                         torch.arange(5, dtype=torch.int32).cuda()[None])
    c.check_held()
    c.layer = layer
    c.check_attention([1])
    one = torch.tensor([291], dtype=torch.int32).cuda()
    k, v = layer.read(one, torch.tensor([[0, 291]], dtype=torch.int32).cuda(), one * 0, 291, 291)
    for got, want in zip((k, v), c.values(0)):
        np.testing.assert_array_equal(got[0].double().cpu().numpy(), want)


def test_operands_of_other_strides_and_alignment():
    c, d = Case(2, 2, 64, 200, seed=3, heads=4), Case(2, 2, 64, 200, seed=3, heads=4)
    n = 75
    bounds, _ = c.spans([70, 5])
    k, v, q = (torch.randn(n, h, 64, generator=c.g).half().cuda() for h in (2, 2, 4))

    def odd(t):  # columns apart, rows that do not begin on 16 bytes
        wide = torch.zeros(n, t.shape[1], 131, dtype=t.dtype, device="cuda")
        wide[:, :, 1:129:2] = t
        return wide[:, :, 1:129:2].transpose(0, 1)[None]

    def flat(t):
        return t.transpose(0, 1).contiguous()[None]

    past = torch.zeros(2, dtype=torch.int32).cuda()
    angle = torch.rand(n, 64, generator=c.g)
    rope = (angle.cos().cuda(), angle.sin().cuda())
    steps = torch.zeros(n, 3, 64, device="cuda")
    steps[:, 1] = rope[0]
    a = c.layer.write(odd(k), odd(v), bounds, past, 70, odd(q), (steps[:, 1], rope[1].t().contiguous().t()))
    b = d.layer.write(flat(k), flat(v), bounds, past, 70, flat(q), rope)
    assert torch.equal(a, b)
    for name in ("codes", "scales", "tail"):
        x, y = (getattr(z.layer, name).contiguous().view(torch.uint8) for z in (c, d))
        assert torch.equal(x, y), name
    same = [z.layer.attention(x, bounds, past, 70, 70, 0.125) for z, x in ((c, odd(q)), (d, flat(q)))]
    assert torch.equal(*same)
    # one head's rows for every head
    one = flat(k[:, :1])
    assert torch.equal(c.layer.attention(one.expand(1, 4, n, 64), bounds, past, 70, 70, 0.125),
                       c.layer.attention(one.expand(1, 4, n, 64).contiguous(), bounds, past, 70, 70, 0.125))


def test_nothing_to_do():
    from talm_amd.kv_cache import CacheLayer

    i32 = {"dtype": torch.int32, "device": "cuda"}
    for sequences, capacity in ((0, 64), (2, 0), (0, 0)):
        layer = CacheLayer.allocate(sequences, 2, 64, capacity)
        bounds, past = torch.zeros(sequences, 2, **i32), torch.zeros(sequences, **i32)
        for n in (0, 3):
            x = torch.zeros(1, 2, n, 64, dtype=torch.float16, device="cuda")
            angle = torch.zeros(n, 64, device="cuda")
            assert layer.write(x, x, bounds, past, n) is None
            turned = layer.write(x, x, bounds, past, 0, x, (angle, angle))
            assert turned.shape == x.shape and (turned == 0).all()
            assert layer.attention(x, bounds, past, n, capacity, 1.0).shape == (1, n, 2, 64)
            assert layer.read(past, bounds, past, n, n)[0].shape == (1, 2, n, 64)
    torch.cuda.synchronize()


def test_captured_steps_replay():
    """A step of write and attention in a HIP graph: replayed with other tokens and places, between eager
    calls, beside a second graph on the same buffers."""
    c = Case(3, 2, 128, 400, heads=12)
    c.append([60, 100, 5])
    scale = 128 ** -0.5
    k, v, q = (torch.zeros(1, h, 3, 128, dtype=torch.float16, device="cuda") for h in (2, 2, 12))
    bounds = torch.tensor([[0, 1], [1, 2], [2, 3]], dtype=torch.int32).cuda()
    past = torch.zeros(3, dtype=torch.int32).cuda()
    angle = torch.zeros(3, 128, device="cuda")
    tables = (angle.clone(), angle.clone())

    def step():
        turned = c.layer.write(k, v, bounds, past, 1, q, tables)
        return c.layer.attention(turned, bounds, past, 1, c.layer.capacity, scale)

    step()  # as a program warms up; nothing of it is kept: past says 0
    c.tokens = [t[:, :, :0] for t in c.tokens]
    c.append([60, 100, 5])
    graphs = []
    for _ in range(2):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = step()
        graphs.append((graph, out))
    for i in range(9):
        graph, out = graphs[i % 2]
        for t in (k, v, q):
            t.copy_(c.rows(3, t.shape[1]))
        a = torch.rand(3, 128, generator=c.g)
        tables[0].copy_(a.cos())
        tables[1].copy_(a.sin())
        past.copy_(torch.tensor(c.past, dtype=torch.int32))
        graph.replay()
        got = out.clone()
        torch.cuda.synchronize()
        assert torch.equal(step(), got), i
        k2 = k[0].transpose(0, 1).clone()
        from talm_amd.rope import rope_

        rope_(q[0].transpose(0, 1).clone(), k2, *tables)
        c.keep([1, 1, 1], k2.transpose(0, 1)[None], v, bounds)
    c.check_held()


@pytest.mark.parametrize("dim,dtype", [(128, torch.float16), (64, torch.bfloat16)])
def test_calls_on_other_streams_and_in_graphs_are_the_same(dim, dtype):
    """Many calls on several streams at once, and in two graphs that are replayed beside each other and
    beside an eager call: the same bits."""
    c = Case(5, 2, dim, 5000, dtype, heads=12)
    c.append([4500, 300, 2000, 0, 64])
    c.append([1, 1, 1, 0, 1])
    bounds, n = c.spans([1, 1, 1, 0, 1])
    q, past = c.rows(n, 12), torch.tensor([4500, 300, 2000, 0, 64], dtype=torch.int32).cuda()

    def call():
        return c.layer.attention(q, bounds, past, 1, 4501, 0.1)

    want = call()
    streams = [torch.cuda.Stream() for _ in range(3)]
    torch.cuda.synchronize()
    outs = []
    for _ in range(20):
        for s in streams:
            with torch.cuda.stream(s):
                outs.append(call())
    outs += [call() for _ in range(20)]
    torch.cuda.synchronize()
    assert all(torch.equal(o, want) for o in outs)
    graphs = []
    for _ in range(2):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = call()
        graphs.append((graph, out))
    for _ in range(3):
        for (graph, _), s in zip(graphs, streams):
            with torch.cuda.stream(s):
                graph.replay()
        eager = call()
        torch.cuda.synchronize()
        assert all(torch.equal(o, want) for o in (eager, *(out for _, out in graphs)))


def test_operands_that_are_refused():
    from talm_amd.kv_cache import CacheLayer

    c = Case(2, 2, 64, 128, heads=4)
    bounds, _ = c.spans([1, 1])
    past = torch.zeros(2, dtype=torch.int32).cuda()
    k, q = c.rows(2, 2), c.rows(2, 4)
    table = torch.zeros(2, 64, device="cuda")
    ok = dict(k=k, v=k, bounds=bounds, past=past, q=None, rope=None)

    def write(**bad):
        a = {**ok, **bad}
        return c.layer.write(a["k"], a["v"], a["bounds"], a["past"], 1, a["q"], a["rope"])

    for bad in (dict(k=k.float()), dict(k=k.bfloat16()), dict(k=k[:, :1]), dict(v=k[:, :, :1]), dict(k=k[..., :32]),
                dict(k=k.cpu()), dict(bounds=bounds.long()), dict(bounds=bounds[:1]), dict(past=past.cpu()),
                dict(past=past.float()), dict(q=q), dict(q=q, rope=(table, None)), dict(rope=(table[:1], table[:1])),
                dict(q=q[:, :, :1], rope=(table, table)), dict(rope=(table.half(), table.half())),
                dict(k=k.detach().clone().requires_grad_())):
        with pytest.raises(ValueError):
            write(**bad)
    with pytest.raises(ValueError):
        c.layer.write(k, k, bounds, past, -1)
    for args in ((q[:, :3], 1, 1, 1.0), (q.float(), 1, 1, 1.0), (q, -1, 1, 1.0), (q, 1, -1, 1.0), (q, 1, 1, 0.0),
                 (q, 1, 1, float("nan")), (q, 1, 1, 1.0, 0), (q, 1, 1, 1.0, 4, -1),
                 (q.detach().clone().requires_grad_(), 1, 1, 1.0)):
        with pytest.raises(ValueError):
            c.layer.attention(args[0], bounds, past, *args[1:])
    with torch.no_grad():
        c.layer.attention(q.detach().clone().requires_grad_(), bounds, past, 1, 64, 1.0)
    with pytest.raises(ValueError):
        c.layer.read(past, bounds, past, 1, 2, (k[0], k[0]))
    with pytest.raises(ValueError):
        c.layer.read(past[:1], bounds, past, 1, 2)
    good = torch.empty(2, 2, 64, dtype=torch.float16, device="cuda")
    for out in ((good, good[:1]), (good, None), (good.float(), good), (good, good.expand(2, 2, 64)[:, :, :32])):
        with pytest.raises(ValueError):
            c.layer.read(past, bounds, past, 1, 2, out)
    with pytest.raises(ValueError):
        c.layer.read(past, bounds, past, 1, -1)
    layer = c.layer
    for name, value in (("codes", layer.codes.view(torch.uint8)), ("scales", layer.scales[:-1]),
                        ("tail", layer.tail.float()), ("table", layer.table.long()), ("table", layer.table[:1])):
        parts = {n: getattr(layer, n) for n in ("codes", "scales", "tail", "table")}
        with pytest.raises(ValueError):
            CacheLayer(**{**parts, name: value}).attention(q, bounds, past, 1, 64, 1.0)
