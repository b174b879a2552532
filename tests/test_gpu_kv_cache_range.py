"""The 8-bit cache's attention (kv_cache.CacheLayer) at the ends of its ranges: values as large as their type
holds, and long sequences whose every part shows in the output. Tolerances are those of
test_gpu_kv_cache.py unless a test derives its own."""

import pytest
import torch

from test_gpu_kv_cache import Case

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
