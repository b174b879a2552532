"""Few-token products on a layer's NF4 codes (LayerGroup.nf4_gemv) against float64 products of the
group's own dequantized fp16 weights (which are bit-exact against the oracle, test_gpu_kernels.py).

Tolerance: the output's rounding u = 2^-11 |y|, and the fp32 sums. A result is at most cols / 32 + 64
additions deep (32 products per MFMA step, up to 16 wavefronts x 4 parts joined): (cols / 32 + 96)
2^-24 of the magnitudes summed."""

import pytest
import torch

pytestmark = pytest.mark.gpu

SHAPES = ((256, 512), (128, 512), (128, 512), (512, 256), (512, 512), (512, 512), (512, 512))


def _group(shapes=SHAPES, seed=1):
    from talm_amd.nf4_linear import Linear4bit
    from talm_amd.qgroup import LayerGroup

    g = torch.Generator("cuda").manual_seed(seed)
    modules = []
    for i, (rows, cols) in enumerate(shapes):
        w = torch.randn(rows, cols, generator=g, device="cuda") * 0.02
        bias = torch.randn(rows, generator=g, device="cuda") if i < 3 else None
        modules.append(Linear4bit.from_weight(w, bias))
    group = LayerGroup(modules)
    group.kept = modules
    return group


def _check(group, x, first, last):
    rows = sum(group.shapes[i][0] for i in range(first, last))
    out = torch.empty(x.shape[0], rows, dtype=torch.float16, device="cuda")
    group.nf4_gemv(x, first, last, out)
    w = group.dequantize(first, last).view(rows, -1).double()
    y, mag = x.double() @ w.T, x.double().abs() @ w.abs().T
    bias = group.span_bias(first, last)
    if bias is not None:
        y, mag = y + bias.double(), mag + bias.double().abs()
    tol = 2.0 ** -11 * y.abs() + (x.shape[1] / 32 + 96) * 2.0 ** -24 * mag + 2.0 ** -25
    worst = ((out.double() - y).abs() / tol).max().item()
    print(f"  {tuple(x.shape)} projections {first}..{last - 1}: {worst:.3f} of the tolerance", flush=True)
    assert worst <= 1.0


@pytest.mark.parametrize("tokens", [1, 2, 3, 4, 5, 8, 9, 16, 17, 31, 32])
def test_gemv_matches_the_dequantized_product(tokens):
    print(f"[case] gemv tokens={tokens}", flush=True)
    group = _group()
    g = torch.Generator("cuda").manual_seed(tokens)
    for first, last in ((0, 3), (0, 1), (3, 4), (4, 6), (6, 7)):
        x = torch.randn(tokens, group.shapes[first][1], generator=g, device="cuda").half()
        _check(group, x, first, last)


@pytest.mark.parametrize("cols", [64, 128, 320, 896, 1536, 4864, 8960])
def test_gemv_over_reductions(cols):
    """Reductions that are not whole units of any tile form."""
    rows = 256 if cols % 64 == 0 and (256 * cols) % 16384 == 0 else 256
    group = _group(((rows, cols),) * 7, seed=cols)
    g = torch.Generator("cuda").manual_seed(cols)
    for tokens in (1, 3, 7, 16, 20):
        _check(group, torch.randn(tokens, cols, generator=g, device="cuda").half(), 4, 5)


def test_gemv_of_the_layer_shapes():
    from talm_amd.workloads import LAYER_SHAPES

    group = _group(LAYER_SHAPES, seed=3)
    for first, last in ((0, 3), (3, 4), (4, 6), (6, 7)):
        for tokens in (1, 6, 32):
            x = torch.randn(tokens, group.shapes[first][1], device="cuda").half()
            _check(group, x, first, last)


@pytest.mark.parametrize("rows,cols", [
    (9092, 4096),    # more tiles per workgroup than the LDS joins at a time, x through LDS; a partial tile
    (20612, 4096),   # the same, x straight
    (9088, 4352),    # several units per wavefront
    (33088, 4352),
    (2044, 4096),    # two parts per tile, one unit
    (1536, 16640),   # and several
    (1536, 704),     # a table in registers
])
def test_gemv_over_tiles(rows, cols):
    print(f"[case] gemv over tiles W {rows} x {cols}", flush=True)
    group = _group(SHAPES[:6] + ((rows, cols),), seed=rows)
    g = torch.Generator("cuda").manual_seed(rows)
    for tokens in (1, 5, 6, 8, 9, 13, 16, 17, 27, 32):
        _check(group, torch.randn(tokens, cols, generator=g, device="cuda").half(), 6, 7)


def test_gemv_past_32_bit_offsets():
    """W of more than 2^31 weights: its last rows against a call on their buffers alone. Both round the same fp32
    sums, taken in another order: (cols / 32 + 96) 2^-24 of the magnitudes summed (at most 0.03 |x|) each."""
    from talm_amd import _ops  # noqa: F401 - registers torch.ops.talm.*

    rows, cols, tail = 1500000, 1536, 128
    print(f"[case] gemv W {rows} x {cols}", flush=True)
    n, at = rows * cols, (rows - tail) * cols
    assert n > 2 ** 31 and at % (64 * 256) == 0
    g = torch.Generator("cuda").manual_seed(4)
    packed = torch.randint(0, 256, (n // 2,), dtype=torch.uint8, device="cuda", generator=g)
    absmax8 = torch.randint(0, 256, (n // 64,), dtype=torch.uint8, device="cuda", generator=g)
    code = torch.linspace(-1, 1, 256, device="cuda")
    absmax2 = torch.rand(n // 16384, device="cuda", generator=g) * 0.01
    offset2 = torch.rand(n // 16384, device="cuda", generator=g) * 0.01 + 0.01
    for tokens in (1, 12, 32):
        x = torch.randn(tokens, cols, device="cuda", generator=g).half()
        out = torch.empty(tokens, rows, dtype=torch.float16, device="cuda")
        last = torch.empty(tokens, tail, dtype=torch.float16, device="cuda")
        torch.ops.talm.nf4_gemv(x, packed, absmax8, code, absmax2, offset2, rows, cols, 64, 256, None, out)
        torch.ops.talm.nf4_gemv(x, packed[at // 2:], absmax8[at // 64:], code, absmax2[at // 16384:],
                                offset2[at // 16384:], tail, cols, 64, 256, None, last)
        err = (out[:, -tail:].double() - last.double()).abs()
        mag = 0.03 * x.double().abs().sum(1, keepdim=True)
        tol = 2 * (2.0 ** -11 * last.double().abs() + (cols / 32 + 96) * 2.0 ** -24 * mag + 2.0 ** -25)
        assert last.abs().max() > 0.1 and (err <= tol).all()


def test_gemv_keeps_nan_and_infinity_to_their_token():
    """x's rows do not mix, whichever way they are loaded."""
    for cols in (512, 4096, 8960):
        group = _group(SHAPES[:6] + ((1536, cols),), seed=cols)
        for tokens in (2, 8, 12, 32):
            x = torch.randn(tokens, cols, device="cuda").half()
            out, bad = (torch.empty(tokens, 1536, dtype=torch.float16, device="cuda") for _ in range(2))
            group.nf4_gemv(x, 6, 7, out)
            x[1, cols - 1], x[tokens - 1, 3] = float("nan"), float("inf")
            group.nf4_gemv(x, 6, 7, bad)
            kept = [t for t in range(tokens) if t not in (1, tokens - 1)]
            assert torch.equal(out[kept], bad[kept])
            assert bad[1].isnan().all() and not bad[tokens - 1].isfinite().any()


def test_gemv_rows_of_a_wider_buffer_and_refusals():
    group = _group()
    wide = torch.randn(5, 1024, device="cuda").half()
    _check(group, wide[:, 256:768], 4, 6)
    _check(group, wide[:1, 256:768], 4, 6)
    out = torch.empty(5, 2048, dtype=torch.float16, device="cuda").fill_(3.0)
    group.nf4_gemv(wide[:, :512], 4, 6, out[:, 512:1536])
    assert (out[:, :512] == 3).all() and (out[:, 1536:] == 3).all()
    none = torch.empty(0, 1024, dtype=torch.float16, device="cuda")
    group.nf4_gemv(torch.empty(0, 512, dtype=torch.float16, device="cuda"), 4, 6, none)
    for x, shape in ((wide[:, :512], (5, 1000)), (wide[:, :500], (5, 1024)), (wide[:, :512].float(), (5, 1024)),
                     (torch.zeros(33, 512, dtype=torch.float16, device="cuda"), (33, 1024)),
                     (wide[:, 4:516], (5, 1024))):
        with pytest.raises(ValueError):
            group.nf4_gemv(x, 4, 6, torch.empty(shape, dtype=torch.float16, device="cuda"))
    with pytest.raises(ValueError):
        group.nf4_gemv(wide[:, :512], 2, 4, out[:, :640])  # v and o: inputs of different sizes


def test_gemv_replays_from_a_graph():
    group = _group()
    x = torch.randn(2, 512, device="cuda").half()
    out = torch.empty(2, 1024, dtype=torch.float16, device="cuda")
    group.span_bias(4, 6)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        group.nf4_gemv(x, 4, 6, out)
    for i in range(3):
        x.copy_(torch.randn(2, 512, device="cuda"))
        graph.replay()
        torch.cuda.synchronize()
        want = torch.empty_like(out)
        group.nf4_gemv(x, 4, 6, want)
        assert torch.equal(out, want)
