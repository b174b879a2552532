"""Counter-based dropout (dropout.dropout) and the adapters' products with it (lora.adapter_branch,
torch.ops.talm.lora_down_drop / lora_bwd_drop), against the oracle's masks and float64 products.

The masks are exact. Tolerances of the products count roundings of at most u = 2^-11 relative (fp16),
each sum of n products in fp32 adding at most n 2^-24 of the magnitudes summed:
  t  = x A^T rounded (u), a second time as ts = s t where two products share it; y = s t B^T rounded:
       s sum |t| |B| (u + the sum of t) + u |y|
  u  = s dy B rounded; dx = u A rounded; dA = u^T x, dB = s dy^T t: of the rounded u and t, (fp16
  gradients: rounded once more)."""

import numpy as np
import pytest
import torch

from oracle import philox

pytestmark = pytest.mark.gpu

U = 2.0 ** -11


def _key(*words):
    return torch.tensor(words, dtype=torch.int64, device="cuda")


def _keep(key, rows, cols, p, site=0):
    return torch.from_numpy(philox.keep(key.tolist(), rows, cols, p, site)).cuda()


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16, torch.float32])
@pytest.mark.parametrize("rows,cols,p", [(1, 1, 0.5), (3, 13, 0.3), (131, 1536, 0.05), (7, 1001, 0.9),
                                         (64, 8, 0.0), (33, 24, 0.999999)])
def test_dropout_is_exactly_its_definition(rows, cols, p, dtype):
    from talm_amd.dropout import dropout

    print(f"[case] dropout {rows} x {cols} p={p} {dtype}", flush=True)
    g = torch.Generator("cuda").manual_seed(rows)
    key = _key(-(2 ** 63) + 12345, 2 ** 40 + 6)
    x = torch.randn(rows, cols, generator=g, device="cuda").to(dtype).requires_grad_()
    dy = torch.randn(rows, cols, generator=g, device="cuda").to(dtype)
    y = dropout(x, p, key, 9)
    (dx,) = torch.autograd.grad(y, x, dy)
    keep, f = _keep(key, rows, cols, p, 9), float(philox.factor(p))
    for got, src in ((y, x.detach()), (dx, dy)):
        want = torch.where(keep, (src.float() * f).to(dtype), torch.zeros((), dtype=dtype, device="cuda"))
        assert torch.equal(got, want)


def test_dropped_values_are_zero_whatever_they_were_and_shapes_stay():
    from talm_amd.dropout import draw_key, dropout

    torch.manual_seed(3)
    key = draw_key("cuda")
    torch.manual_seed(3)
    assert torch.equal(key, draw_key("cuda")) and not torch.equal(key, draw_key("cuda"))
    x = torch.full((2, 3, 5, 8), float("nan"), device="cuda")
    y = dropout(x, 0.5, key)
    keep = _keep(key, 30, 8, 0.5).view(2, 3, 5, 8)
    assert y.shape == x.shape and (y[~keep] == 0).all() and torch.isnan(y[keep]).all()
    for shape in ((0, 8), (4, 0), (0,)):
        assert dropout(torch.empty(shape, device="cuda"), 0.5, key).shape == shape
    one = torch.ones((), device="cuda")
    assert dropout(one, 0.0) == 1 and dropout(one, 0.0).shape == ()


@pytest.mark.parametrize("rows", [2 ** 21 + 3, 2 ** 22 + 3])
def test_dropout_of_more_blocks_than_a_launch_holds(rows):
    """Blocks past 2^30 (further launches) and past 2^31 (a 64-bit division), in place."""
    from talm_amd import _ops  # noqa: F401 - registers torch.ops.talm.*

    cols, p = 4096, 0.25
    if torch.cuda.mem_get_info()[0] < 2 * rows * cols + (4 << 30):
        pytest.skip("not enough free device memory")
    print(f"[case] dropout {rows} x {cols}", flush=True)
    key = _key(77, 88)
    x = torch.ones(rows, cols, dtype=torch.float16, device="cuda")
    torch.ops.talm.dropout(x, p, key, 3, x)
    f = torch.tensor(float(philox.factor(p))).half()
    for r in (0, 1, 2 ** 21 - 1, 2 ** 21, 2 ** 21 + 2, rows - 4, rows - 1):
        block = np.arange(cols // 8, dtype=np.uint64) + np.uint64(r * (cols // 8))
        words = philox.philox4x32((block, block >> np.uint64(32), np.full_like(block, 3), np.full_like(block, 88)),
                                  (77, 0))
        bits = np.stack(words, 1).astype("<u4").view("<u2").reshape(-1)
        keep = torch.from_numpy(bits.astype(np.int64) >= philox.threshold(p))
        assert torch.equal(x[r].cpu(), torch.where(keep, f, torch.zeros((), dtype=torch.float16)))
    del x
    torch.cuda.empty_cache()


def test_strided_rows_and_in_place():
    from talm_amd import _ops  # noqa: F401
    from talm_amd.dropout import dropout

    key = _key(1, 2)
    wide = torch.randn(40, 72, device="cuda").half()
    for view in (wide[:, 8:40], wide[:, 3:36], wide[::2, :16], wide.t(), wide[:1, :5],
                 wide[:1].expand(40, 72)):
        keep = _keep(key, *view.shape, 0.4)
        want = torch.where(keep, (view.float() * float(philox.factor(0.4))).half(), 0.0)
        assert torch.equal(dropout(view, 0.4, key), want)
    x = wide.clone()
    torch.ops.talm.dropout(x, 0.4, key, 0, x)
    assert torch.equal(x, dropout(wide, 0.4, key))


def test_dropout_refusals_on_the_gpu():
    from talm_amd.dropout import dropout

    x = torch.ones(4, 8, device="cuda")
    for args in ((x, 0.5), (x, 1.0, _key(1, 2)), (x, 0.5, torch.tensor([1, 2])), (x, 0.5, _key(1, 2, 3)),
                 (x, 0.5, _key(1, 2), -1), (x.double(), 0.5, _key(1, 2)), (x.long(), 0.5, _key(1, 2))):
        with pytest.raises(ValueError):
            dropout(*args)


def test_a_captured_dropout_follows_its_key():
    from talm_amd.dropout import draw_key, dropout

    x = torch.randn(64, 256, device="cuda").half()
    key = _key(5, 6)
    dropout(x, 0.3, key)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y = dropout(x, 0.3, key)
        drawn = draw_key("cuda")
        z = dropout(x, 0.3, drawn)
    seen = set()
    for i in range(4):
        key.copy_(_key(5, i))
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(y, dropout(x, 0.3, _key(5, i)))
        assert torch.equal(z, dropout(x, 0.3, drawn.clone()))
        seen.add(tuple(drawn.tolist()))
    assert len(seen) == 4  # a replay draws a key of its own


# -- the adapters' products ------------------------------------------------------------------------

def _branch(n, size, out, p, dtype, seed, key, site=4, scaling=2.0):
    g = torch.Generator("cuda").manual_seed(seed)
    x = torch.randn(n, size, generator=g, device="cuda").half().requires_grad_()
    a = ((torch.rand(16, size, generator=g, device="cuda") * 2 - 1) * size ** -0.5).to(dtype).requires_grad_()
    b = (torch.randn(out, 16, generator=g, device="cuda") * 0.05).to(dtype).requires_grad_()
    dy = torch.randn(n, out, generator=g, device="cuda").half()
    return x, a, b, dy


def _expect(x, a, b, dy, m, scaling, half_grads):
    """float64 values and tolerances of y, dx, dA, dB; m: the mask times its factor."""
    x, a, b, dy = (t.detach().half().double() for t in (x, a, b, dy))
    xd = x * m
    size, out, n = x.shape[1], b.shape[0], x.shape[0]
    acc = 2.0 ** -24
    t, ta = xd @ a.T, xd.abs() @ a.abs().T
    tol_t = U * t.abs() + (size + 2) * acc * ta + 2.0 ** -25
    y = scaling * t @ b.T
    tol_y = scaling * (tol_t + 2.0 ** -25) @ b.abs().T + 16 * acc * scaling * t.abs() @ b.abs().T + U * y.abs() + 2.0 ** -25
    u = scaling * dy @ b
    tol_u = U * u.abs() + out * acc * scaling * dy.abs() @ b.abs() + 2.0 ** -25
    dx = (u @ a) * m
    tol_dx = (tol_u @ a.abs() + 18 * acc * u.abs() @ a.abs()) * m + U * dx.abs() + 2.0 ** -25
    da, db = u.T @ xd, scaling * dy.T @ t
    tol_da = tol_u.T @ xd.abs() + (n + 2) * acc * u.abs().T @ xd.abs()
    tol_db = scaling * (dy.abs().T @ tol_t + (n + 2) * acc * dy.abs().T @ t.abs())
    if half_grads:
        tol_da, tol_db = tol_da + U * da.abs() + 2.0 ** -25, tol_db + U * db.abs() + 2.0 ** -25
    return (y, dx, da, db), (tol_y, tol_dx, tol_da, tol_db)


def _compare(got, want, tols):
    for name, a, b, tol in zip(("y", "dx", "dA", "dB"), got, want, tols):
        err = (a.double() - b).abs()
        worst = (err / tol.clamp_min(1e-30)).max().item() if err.numel() else 0.0
        print(f"  {name}: max err {err.max().item() if err.numel() else 0:.3e}, {worst:.3f} of its tolerance", flush=True)
        assert a.shape == b.shape and worst <= 1.0, name


@pytest.mark.parametrize("n,size,out", [(1, 32, 32), (17, 96, 160), (64, 1536, 256), (131, 896, 128),
                                        (200, 256, 1536), (70, 4864, 896)])
@pytest.mark.parametrize("p,dtype", [(0.0, torch.float32), (0.1, torch.float32), (0.5, torch.float16)])
def test_adapter_branch_matches_its_formula(n, size, out, p, dtype):
    from talm_amd.lora import adapter_branch

    print(f"[case] adapter branch {n} x {size} -> {out} p={p} {dtype}", flush=True)
    key = _key(77, n)
    x, a, b, dy = _branch(n, size, out, p, dtype, n + size, key)
    y = adapter_branch(x, a, b, 2.0, p, key if p else None, 4)
    grads = torch.autograd.grad(y, (x, a, b), dy)
    assert grads[1].dtype == grads[2].dtype == dtype
    m = _keep(key, n, size, p, 4).double() / (1 - philox.threshold(p) / 65536)
    _compare((y, *grads), *_expect(x, a, b, dy, m, 2.0, dtype == torch.float16))


def test_adapter_branch_past_32_bit_offsets():
    """x of more than 2^31 elements; only the last rows have a gradient, so that theirs are the weights' too."""
    from talm_amd.lora import adapter_branch

    n, size, out, tail, p = 300000, 8960, 32, 64, 0.25
    if torch.cuda.mem_get_info()[0] < 32 << 30:
        pytest.skip("not enough free device memory")
    print(f"[case] adapter branch {n} x {size}", flush=True)
    key = _key(41, 42)
    _, a, b, _ = _branch(1, size, out, p, torch.float32, 3, key)
    x = torch.empty(n, size, dtype=torch.float16, device="cuda").normal_().requires_grad_()
    dy = torch.zeros(n, out, dtype=torch.float16, device="cuda")
    dy[-tail:] = torch.randn(tail, out, device="cuda").half()
    y = adapter_branch(x, a, b, 2.0, p, key, 4)
    dx, da, db = torch.autograd.grad(y, (x, a, b), dy)
    block = np.arange((n - tail) * size // 8, n * size // 8, dtype=np.uint64)
    words = philox.philox4x32((block, block >> np.uint64(32), np.full_like(block, 4), np.full_like(block, 42)), (41, 0))
    bits = np.stack(words, 1).astype("<u4").view("<u2").reshape(tail, size)
    m = torch.from_numpy(bits.astype(np.int64) >= philox.threshold(p)).cuda().double() * float(philox.factor(p))
    want, tols = _expect(x[-tail:], a, b, dy[-tail:], m, 2.0, False)
    assert not dx[:-tail].any()
    _compare((y[-tail:].detach(), dx[-tail:], da, db), want, tols)
    del x, dx, y
    torch.cuda.empty_cache()


def test_adapter_branch_without_rows_and_with_batch_dimensions():
    from talm_amd.lora import adapter_branch

    key = _key(3, 4)
    x, a, b, dy = _branch(24, 64, 96, 0.2, torch.float32, 1, key)
    y = adapter_branch(x, a, b, 2.0, 0.2, key)
    y3 = adapter_branch(x.view(2, 3, 4, 64), a, b, 2.0, 0.2, key)
    assert y3.shape == (2, 3, 4, 96) and torch.equal(y3.view(24, 96), y)
    wide = torch.zeros(24, 80, dtype=torch.float16, device="cuda")
    wide[:, 4:68] = x.detach()  # rows that are not 16-byte aligned are copied
    assert torch.equal(adapter_branch(wide[:, 4:68], a, b, 2.0, 0.2, key), y)
    empty = x.detach()[:0].requires_grad_()
    out = adapter_branch(empty, a, b, 2.0, 0.2, key)
    grads = torch.autograd.grad(out.sum(), (empty, a, b))
    assert out.shape == (0, 96) and (grads[1] == 0).all() and (grads[2] == 0).all()


def test_adapter_branch_refusals():
    from talm_amd.lora import adapter_branch

    x, a, b, _ = _branch(4, 64, 32, 0.2, torch.float32, 1, None)
    key = _key(1, 2)
    for args in ((x.float(), a, b, 2.0), (x, a[:8], b[:, :8], 2.0), (x[:, :48], a[:, :48], b, 2.0),
                 (x, a, b.half(), 2.0), (x, a, b[:24], 2.0), (x, a, b, 2.0, 0.2), (x, a, b, 2.0, 1.5, key),
                 (x, a.cpu(), b.cpu(), 2.0)):
        with pytest.raises(ValueError):
            adapter_branch(*args)


def test_two_adapters_have_masks_of_their_own():
    """The products over two adapters of one x (q and v of a layer): each under its own site."""
    from talm_amd import _ops

    n, size, lo, seg = 75, 160, (0, 128), (96, 64)
    p, key, sites = 0.3, _key(8, 9), (0, 1)
    g = torch.Generator("cuda").manual_seed(2)
    def rand(*shape):
        return torch.randn(*shape, generator=g, device="cuda")
    x = rand(n, size).half()
    a = [(rand(16, size) * 0.05).half() for _ in range(2)]
    b = [(rand(s, 16) * 0.05).half() for s in seg]
    dy = rand(n, 192).half()
    half = dict(dtype=torch.float16, device="cuda")
    t, ts = torch.empty(n, 32, **half), torch.empty(n, 32, **half)
    torch.ops.talm.lora_down_drop(x, a[0], a[1], p, key, *sites, 2.0, 3.0, t, ts)
    u_raw, u = torch.empty(n, 32, **half), torch.empty(n, 32, **half)
    torch.ops.talm.lora_down(dy, b[0], b[1], seg[0], seg[1], lo[0], lo[1], 1, 2.0, 3.0, u_raw, u)
    base = rand(n, size).half()
    dx = base.clone()
    da = [torch.empty(16, size, device="cuda") for _ in range(2)]
    db = [torch.empty(s, 16, device="cuda") for s in seg]
    ws = torch.full((_ops.lora_bwd_drop_workspace_bytes(n, size, 2, *seg),), 255, dtype=torch.uint8, device="cuda")
    torch.ops.talm.lora_bwd_drop(x, dy, u, t, p, key, *sites, lo[0], seg[0], 2.0, da[0], db[0], lo[1], seg[1], 3.0,
                                 da[1], db[1], a[0], a[1], dx, dx, ws)
    alone = torch.empty_like(dx)  # dx without the weight gradients, into another tensor than its base
    torch.ops.talm.lora_bwd_drop(x, dy, u, t, p, key, *sites, lo[0], seg[0], 2.0, None, None, lo[1], seg[1], 3.0,
                                 None, None, a[0], a[1], base, alone, ws)
    assert torch.equal(alone, dx)
    total, tol = base.double(), U * base.double().abs() + 2.0 ** -24
    for i, scaling in enumerate((2.0, 3.0)):
        m = _keep(key, n, size, p, sites[i]).double() / (1 - philox.threshold(p) / 65536)
        dyi = dy[:, lo[i]:lo[i] + seg[i]]
        want, tols = _expect(x, a[i], b[i], dyi, m, scaling, False)
        _compare((ts[:, 16 * i:16 * i + 16].double() @ b[i].double().T, want[1], da[i], db[i]), want, tols)
        total, tol = total + want[1], tol + tols[1] + U * want[1].abs()
    assert ((dx.double() - total).abs() <= tol).all()


def test_a_captured_branch_replays():
    from talm_amd.lora import adapter_branch

    key = _key(1, 1)
    x, a, b, dy = _branch(96, 256, 128, 0.2, torch.float16, 5, key)

    def step():
        y = adapter_branch(x, a, b, 2.0, 0.2, key)
        return (y.detach(), *torch.autograd.grad(y, (x, a, b), dy))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        outs = step()
    for i in range(4):
        key.copy_(_key(i, 7))
        with torch.no_grad():
            x.copy_(torch.randn(96, 256, device="cuda"))
        graph.replay()
        torch.cuda.synchronize()
        for got, want in zip(outs, step()):
            assert torch.equal(got, want)


def test_the_gradients_have_no_backward():
    """Under create_graph the gradients come out, and a backward through them is an error, not zeros."""
    from talm_amd.dropout import dropout
    from talm_amd.lora import adapter_branch
    from talm_amd.unpad import window_attention

    key = _key(1, 2)
    x, a, b, _ = _branch(8, 64, 32, 0.2, torch.float32, 1, key)
    q = torch.randn(1, 2, 8, 128, device="cuda").half().requires_grad_()
    cu = torch.tensor([0, 8], dtype=torch.int32, device="cuda")
    for y, leaf in ((dropout(x, 0.2, key), x), (adapter_branch(x, a, b, 2.0, 0.2, key), a),
                    (window_attention(q, q, q, cu, 8, 0.1, 4), q)):
        (first,) = torch.autograd.grad(y.float().sum(), leaf, create_graph=True)
        assert torch.isfinite(first).all()
        with pytest.raises(RuntimeError):  # the leaf is not reached
            torch.autograd.grad(first.float().sum(), leaf, retain_graph=True)
        with pytest.raises(RuntimeError, match="differentiable once"):
            first.float().sum().backward()


@pytest.mark.parametrize("size", [96, 1536, 2048])
def test_an_infinity_reaches_its_own_token_as_the_formula_has_it(size):
    """x holds an infinity where A is positive: t and, B positive, y are infinite for that token, whatever the
    reduction's number of parts, and the others are what they are without it."""
    from talm_amd import _lib

    n, out = 40, 64
    half = dict(dtype=torch.float16, device="cuda")
    g = torch.Generator("cuda").manual_seed(size)
    x = torch.randn(n, size, generator=g, device="cuda").half()
    a = (torch.rand(16, size, generator=g, device="cuda") * 0.02 + 0.01).half()
    b = (torch.rand(out, 16, generator=g, device="cuda") + 0.5).half()
    lib = _lib.lib()

    def branch(x):
        t, y = torch.empty(n, 16, **half), torch.empty(n, out, **half)
        ws = torch.empty(lib.talm_lora_branch_fwd_workspace(n, size), dtype=torch.uint8, device="cuda")
        status = lib.talm_lora_branch_fwd(x.data_ptr(), size, n, size, out, a.data_ptr(), b.data_ptr(), 0.0, None, 0,
                                          2.0, t.data_ptr(), y.data_ptr(), ws.data_ptr(), ws.numel(),
                                          torch.cuda.current_stream().cuda_stream)
        assert status == _lib.TALM_OK
        torch.cuda.synchronize()
        return t, y
    want = branch(x)
    others = [i for i in range(n) if i != 7]
    for column in (0, size // 2, size - 1):
        for value in (float("inf"), -float("inf")):
            print(f"[case] branch of {size} columns, {value} at {column}", flush=True)
            bad = x.clone()
            bad[7, column] = value
            for got, without in zip(branch(bad), want):
                assert (got[7] == value).all() and torch.equal(got[others], without[others])


def test_adapter_gradients_of_no_tokens_are_zero_without_a():
    """dx is given for no tokens, A is not: the weight gradients are zeros."""
    from talm_amd import _lib

    lib = _lib.lib()
    da, db = torch.full((16, 64), 5.0, device="cuda"), torch.full((32, 16), 5.0, device="cuda")
    dx = torch.full((1, 64), 5.0, dtype=torch.float16, device="cuda")
    ws = torch.empty(max(lib.talm_lora_bwd_drop_workspace(0, 64, 1, 32, 0), 1), dtype=torch.uint8, device="cuda")
    status = lib.talm_lora_bwd_drop(None, 64, None, 32, None, 16, None, 16, 0, 64, 1, 0.5, _key(1, 2).data_ptr(), 0, 1,
                                    _lib.TALM_F32, 0, 32, 1.0, da.data_ptr(), db.data_ptr(), 0, 0, 0.0, None, None,
                                    None, None, None, 0, dx.data_ptr(), 64, ws.data_ptr(), ws.numel(),
                                    torch.cuda.current_stream().cuda_stream)
    torch.cuda.synchronize()
    assert status == _lib.TALM_OK and (da == 0).all() and (db == 0).all() and (dx == 5).all()
