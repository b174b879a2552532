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


# -- buffers of any number of rows, and adapters, straight through the op ------------------------------

def _weight(rows, cols, seed):
    """The op's buffers of a W [rows, cols], and W in float64."""
    from oracle import nf4

    g = torch.Generator().manual_seed(seed)
    n = rows * cols
    blocks, groups = n // 64, (n // 64 + 255) // 256
    packed = torch.randint(0, 256, (n // 2,), generator=g, dtype=torch.uint8)
    absmax8 = torch.randint(0, 256, (blocks,), generator=g, dtype=torch.uint8)
    code = torch.linspace(-1, 1, 256)
    absmax2 = torch.rand(groups, generator=g) * 0.05
    offset2 = torch.rand(groups, generator=g) * 0.05 + 0.05
    # the oracle takes whole second-level groups
    bits = nf4.group_dequant(*(torch.nn.functional.pad(t, (0, size - t.numel())).numpy() for t, size in (
        (packed, groups * 8192), (absmax8, groups * 256), (code, 256), (absmax2, groups), (offset2, groups))))
    w = torch.from_numpy(bits.view("float16")[:n].astype("float32")).view(rows, cols)
    return [t.cuda() for t in (packed, absmax8, code, absmax2, offset2)], w.cuda().double()


def _check_op(rows, cols, tokens, segments, biased, buffers, w, pad=0):
    """segments: the adapters' (lo, hi). 16 products of an adapter are exact in fp32 and added one by one: 32
    additions more than the tolerance above counts, and the bias."""
    print(f"[case] W {rows} x {cols} tokens={tokens} adapters={segments} bias={biased}", flush=True)
    g = torch.Generator("cuda").manual_seed(rows + tokens)

    def rand(*shape):
        return torch.randn(*shape, generator=g, device="cuda").half()
    x = rand(tokens, cols + pad)[:, :cols]
    bias = rand(rows) if biased else None
    ts = rand(tokens, 16 * len(segments) + pad)[:, :16 * len(segments)] if segments else None
    ups = [rand(hi - lo, 16) for lo, hi in segments]
    wide = torch.full((tokens, rows + 16), 3.0, dtype=torch.float16, device="cuda")
    out = wide[:, 8:8 + rows]
    extra = [] if ts is None else [ts, *[v for b, (lo, hi) in zip(ups, segments) for v in (b, lo, hi)]]
    torch.ops.talm.nf4_gemv(x, *buffers, rows, cols, 64, 256, bias, out, *extra)
    y, mag = x.double() @ w.T, x.double().abs() @ w.abs().T
    if biased:
        y, mag = y + bias.double(), mag + bias.double().abs()
    for i, (b, (lo, hi)) in enumerate(zip(ups, segments)):
        t = ts[:, 16 * i:16 * i + 16].double()
        y[:, lo:hi] += t @ b.double().T
        mag[:, lo:hi] += t.abs() @ b.double().abs().T
    tol = 2.0 ** -11 * y.abs() + (cols / 32 + 96 + 33) * 2.0 ** -24 * mag + 2.0 ** -25
    worst = ((out.double() - y).abs() / tol).max().item()
    print(f"  {worst:.3f} of the tolerance", flush=True)
    assert worst <= 1.0
    assert (wide[:, :8] == 3).all() and (wide[:, 8 + rows:] == 3).all()


@pytest.mark.parametrize("cols", [64, 320, 896])
@pytest.mark.parametrize("rows", [1, 7, 13, 250])
def test_gemv_of_odd_rows_and_reductions(rows, cols):
    """Row tiles and reduction units that are both partial, down to a weight of one row."""
    buffers, w = _weight(rows, cols, rows + cols)
    for tokens in (1, 2, 3, 5, 9, 17, 32):
        _check_op(rows, cols, tokens, (), tokens % 2 == 1, buffers, w, pad=8 * (tokens % 3))


@pytest.mark.parametrize("rows,cols", [
    (250, 896), (2048, 1536),      # a table in registers
    (6203, 1600),                  # a table in LDS: one unit a wavefront
    (2051, 4672),                  # two parts per tile
    (4101, 4352), (1540, 8960),    # several units per wavefront, in one part and in two
    (20612, 4096),                 # tiles joined in several rounds
])
def test_gemv_with_adapters_matches_its_formula(rows, cols):
    """One and two adapters whose rows begin and end inside tiles, lie in the last one, or share some."""
    buffers, w = _weight(rows, cols, rows)
    third, last = rows // 3 | 1, rows - 5
    for tokens in (1, 5, 9, 17, 32):
        for segments in ([(0, rows)], [(third, last)], [(3, third), (last, rows)], [(third, rows), (1, last)],
                         [(last, last + 1), (0, 1)]):
            _check_op(rows, cols, tokens, segments, tokens != 5, buffers, w, pad=8 * (tokens & 1))
