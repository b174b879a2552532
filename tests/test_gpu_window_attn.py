"""Sliding-window attention with sinks over packed rows (unpad.window_attention) against its formula
in float64 on the CPU: output, and the gradients of q, k and v.

Tolerances count roundings, each at most half a step u of the operands' type (fp16 2^-11, bf16
2^-8), elementwise against the magnitudes summed:
  out     P is rounded (u P, and 2^-25 where fp16 turns subnormal, with a row's sum at least 1:
          relative to it at most 2^-25), the output is rounded: u (sum P |V| + |out|) + n 2^-25 max |V|
  dV      u (sum P |dO| + |dV|) + 2^-25 sum |dO| over the rows that see the key
  dS      = P (dP - D), rounded: u |dS| + 2^-25; D comes from the rounded output, off by at most
          sum |dO| tol(out)
  every result's own rounding: u, or 2^-25 where fp16 is subnormal
  dQ, dK  scale sum tol(dS) |K| (|Q|) + u |dQ|
and every P carries the fp32 error of its score: a 128-term product (128 2^-24 sum |q k| scale) and of
exp2, log2 and the scale's product (2^-19 in all for exponents up to 2^5)."""

import math

import pytest
import torch

pytestmark = pytest.mark.gpu

D = 128


def _reference(q, k, v, lengths, scale, window, sinks, dout, half, device="cpu"):
    """float64 (on the GPU for the larger cases): (values, tolerances), each (out, dq, dk, dv)."""
    u = {torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}[half]
    sub = 2.0 ** -25 if half == torch.float16 else 0.0
    q, k, v, dout = (t.detach().to(device).double().transpose(0, 1) for t in (q, k, v, dout))
    group = q.shape[0] // k.shape[0]
    vals = [torch.zeros_like(q), torch.zeros_like(q), torch.zeros_like(k), torch.zeros_like(v)]
    tols = [torch.zeros_like(t) for t in vals]
    s0 = 0
    for n in lengths:
        rows = slice(s0, s0 + n)
        s0 += n
        i = torch.arange(n, device=device)
        seen = (i[None] <= i[:, None]) & ((i[:, None] - i[None] < window) | (i[None] < sinks))
        for h in range(q.shape[0]):
            qh, kh, vh, g = q[h, rows], k[h // group, rows], v[h // group, rows], dout[h, rows]
            if n == 0:
                continue
            s = (scale * qh @ kh.T).masked_fill(~seen, -math.inf)
            p = torch.softmax(s, -1)
            rel = 128 * 2.0 ** -24 * (scale * qh.abs() @ kh.abs().T).max().item() + 2.0 ** -19
            o = p @ vh
            ds = p * (g @ vh.T - (g * o).sum(-1, keepdim=True))
            tol_o = (u + 2 * rel) * (p @ vh.abs()) + u * o.abs() + sub * n * vh.abs().max()
            tol_d = (g.abs() * tol_o).sum(-1, keepdim=True)
            tol_dp = 128 * 2.0 ** -24 * (g.abs() @ vh.abs().T)
            tol_ds = ((u + 2 * rel) * ds.abs() + p * (tol_d + tol_dp) + sub) * seen
            vals[0][h, rows] = o
            vals[1][h, rows] = scale * ds @ kh
            vals[2][h // group, rows] += scale * ds.T @ qh
            vals[3][h // group, rows] += p.T @ g
            tols[0][h, rows] = tol_o
            tols[1][h, rows] = scale * tol_ds @ kh.abs()
            tols[2][h // group, rows] += scale * tol_ds.T @ qh.abs()
            tols[3][h // group, rows] += (u + 2 * rel) * p.T @ g.abs() + sub * (seen.double().T @ g.abs())
    # the roundings of the results (out's is in already): u relative, or half of fp16's subnormal
    # spacing 2^-24 for values below 2^-14, whose rounding is not relative
    for i, (t, val) in enumerate(zip(tols, vals)):
        t += (u * val.abs() if i else 0.0) + sub
    return [t.transpose(0, 1).cpu() for t in vals], [t.transpose(0, 1).cpu() for t in tols]


def _inputs(n, hq, hkv, half, strided, seed):
    g = torch.Generator("cpu").manual_seed(seed)
    if strided:  # column views of one [N, q + k + v] buffer
        qkv = torch.randn(n, (hq + 2 * hkv) * D, generator=g).to(half).cuda()
        q, k, v = (t.view(n, -1, D) for t in qkv.split([hq * D, hkv * D, hkv * D], 1))
    else:
        q, k, v = (torch.randn(n, h, D, generator=g).to(half).cuda() for h in (hq, hkv, hkv))
    return q, k, v, torch.randn(n, hq, D, generator=g).to(half).cuda()


def _call(q, k, v, cu, longest, window, sinks, dout=None, scale=D ** -0.5):
    from talm_amd.unpad import window_attention

    leaves = [t.transpose(0, 1)[None].detach().requires_grad_() for t in (q, k, v)]
    out = window_attention(*leaves, cu, longest, scale, window, sinks)
    if dout is None:
        return out[0].detach()
    grads = torch.autograd.grad(out, leaves, dout[None])
    return [out[0].detach()] + [g[0].transpose(0, 1) for g in grads]


def _cu(lengths):
    return torch.tensor([0] + lengths).cumsum(0).to(torch.int32).cuda()


def _check(lengths, window, sinks, hq, hkv, half=torch.float16, strided=True, seed=1, device="cpu"):
    print(f"[case] window lengths={lengths if len(lengths) < 12 else len(lengths)} window={window} "
          f"sinks={sinks} heads={hq}/{hkv} {half} strided={strided} seed={seed}", flush=True)
    q, k, v, dout = _inputs(sum(lengths), hq, hkv, half, strided, seed)
    got = _call(q, k, v, _cu(lengths), max(lengths), window, sinks, dout)
    vals, tols = _reference(q, k, v, lengths, D ** -0.5, window, sinks, dout, half, device)
    for name, a, b, tol in zip(("out", "dq", "dk", "dv"), got, vals, tols):
        err = (a.double().cpu() - b).abs()
        ratio = err / tol.clamp_min(1e-30)
        worst, at = ratio.max().item(), int(ratio.argmax())
        print(f"  worst at {at}: {a.flatten()[at].item():.9g} for {b.flatten()[at].item():.9g}")
        print(f"  {name}: max err {err.max():.3e}, {worst:.3f} of its tolerance", flush=True)
        assert a.dtype == half and worst <= 1.0, name


@pytest.mark.parametrize("window,sinks", [(1, 0), (1, 1), (5, 2), (64, 0), (65, 4), (1000, 0), (2 ** 31 - 1, 7)])
def test_window_short_rows(window, sinks):
    """From a row of its own token alone to windows wider than every row, at tile borders."""
    _check([1, 17, 64, 65, 129], window, sinks, 4, 2, strided=False)


@pytest.mark.parametrize("lengths,window,sinks,hq,hkv", [
    ([300, 128, 512, 257], 100, 4, 12, 2),
    ([700], 33, 65, 4, 1),             # sinks over a tile's border and wider than the window
    ([700, 650], 20, 200, 2, 1),       # sinks in two key tiles of the backward
    ([0, 5, 0, 130, 0], 16, 3, 7, 1),  # sequences without a token
    ([1200], 900, 0, 2, 1),            # few workgroups and a long chain: the key tiles split in two
    ([1500, 64], 700, 5, 4, 4),
    ([130, 127, 128, 129], 128, 0, 7, 1),
    ([40, 64, 16, 33], 9, 1, 12, 4),   # three heads a workgroup
])
@pytest.mark.parametrize("half", [torch.float16, torch.bfloat16])
def test_window_matches_its_formula(lengths, window, sinks, hq, hkv, half):
    _check(lengths, window, sinks, hq, hkv, half)


@pytest.mark.parametrize("window,sinks", [(70, 3), (513, 130)])
def test_sinks_gradient_over_several_chunks(window, sinks):
    """Rows far past the window, whose sinks' gradients come from several chunks of rows."""
    _check([2300, 1000], window, sinks, 2, 1)


@pytest.mark.parametrize("sinks", [0, 6])
def test_window_from_the_work_queue(sinks):
    """More work items than two per CU: the backward's queue (and its items without a row)."""
    _check([150 + 7 * (i % 9) for i in range(20)] + [900], 60, sinks, 16, 16, seed=5)


@pytest.mark.parametrize("lengths,window,sinks,hq,hkv,half", [
    ([1300] * 16, 60, 6, 6, 1, torch.float16),        # all six heads an item, sinks' rows in chunks
    ([1300] * 16, 60, 0, 6, 1, torch.float16),
    ([700, 1, 65, 1500, 0, 900, 128, 2000] * 2, 300, 130, 12, 2, torch.bfloat16),   # some of the heads
    ([1111, 800] * 6, 1000, 3, 4, 2, torch.float16),
])
def test_several_heads_per_item(lengths, window, sinks, hq, hkv, half):
    """Enough work that a dK / dV item takes several heads of its KV head one after the other."""
    _check(lengths, window, sinks, hq, hkv, half, seed=7, device="cuda")


def test_rows_past_32_bit_offsets():
    """Operands of more than 2^31 elements: the last sequences' results and gradients."""
    lengths, tail, hq, hkv = [4096] * 299 + [700, 77], 777, 12, 2
    n = sum(lengths)
    if torch.cuda.mem_get_info()[0] < 64 << 30:
        pytest.skip("not enough free device memory")
    print(f"[case] window, {n} rows of {(hq + 2 * hkv) * D} columns", flush=True)
    g = torch.Generator("cuda").manual_seed(8)
    qkv = torch.empty(n, (hq + 2 * hkv) * D, dtype=torch.float16, device="cuda").normal_(generator=g)
    assert qkv.numel() > 2 ** 31
    q, k, v = (t.view(n, -1, D) for t in qkv.split([hq * D, hkv * D, hkv * D], 1))
    dout = torch.empty(n, hq, D, dtype=torch.float16, device="cuda").normal_(generator=g)
    got = [t[-tail:].clone() for t in _call(q, k, v, _cu(lengths), max(lengths), 100, 4, dout)]
    vals, tols = _reference(q[-tail:], k[-tail:], v[-tail:], [700, 77], D ** -0.5, 100, 4, dout[-tail:],
                            torch.float16, "cuda")
    for name, a, b, tol in zip(("out", "dq", "dk", "dv"), got, vals, tols):
        assert ((a.double().cpu() - b).abs() <= tol).all(), name
    del qkv, q, k, v, dout
    torch.cuda.empty_cache()


def test_many_sequences_one_workgroup_per_item():
    """More sequences than the queue takes."""
    _check([30 + i % 50 for i in range(70)], 24, 2, 2, 1, seed=6)


def test_a_window_of_the_whole_row_is_the_causal_attention():
    """Two kernels, each off the formula by at most the tolerance (the compiler contracts their products
    and sums differently, so not the same bits): apart by at most twice as much."""
    from talm_amd.unpad import VarlenAttention

    lengths = [300, 77, 513]
    q, k, v, dout = _inputs(sum(lengths), 12, 2, torch.float16, True, 9)
    got = _call(q, k, v, _cu(lengths), 513, 513, 0, dout)
    leaves = [t.transpose(0, 1)[None].detach().requires_grad_() for t in (q, k, v)]
    out = VarlenAttention.apply(*leaves, _cu(lengths), 513, D ** -0.5)
    want = [out[0]] + [g[0].transpose(0, 1) for g in torch.autograd.grad(out, leaves, dout[None])]
    _, tols = _reference(q, k, v, lengths, D ** -0.5, 513, 0, dout, torch.float16)
    for a, b, tol in zip(got, want, tols):
        assert ((a.double() - b.double()).abs().cpu() <= 2 * tol).all()


def test_gradients_against_differences():
    """The directional derivative of sum(out g) along a random direction of q, k and v, against a
    central difference of step h = 2^-4: its truncation is h^2 / 6 of the third derivative, its
    rounding error that of two fp16 outputs, sqrt(N) 2^-12 |out| |g| / (sqrt(3) h) if independent; both
    within 2% of the derivative's own scale |grad| |direction| / sqrt(count), taken five times."""
    lengths, window, sinks = [200, 90], 40, 3
    q, k, v, dout = _inputs(290, 4, 2, torch.float16, False, 13)
    cu = _cu(lengths)
    _, *grads = _call(q, k, v, cu, 200, window, sinks, dout)
    gen = torch.Generator("cpu").manual_seed(14)
    for which in range(3):
        ops = [q, k, v]
        d = torch.randn(ops[which].shape, generator=gen).cuda()
        vals, steps = [], []
        for sign in (1, -1):
            moved = list(ops)
            moved[which] = (ops[which].float() + sign * 2.0 ** -4 * d).half()
            steps.append(moved[which].double())
            vals.append((_call(*moved, cu, 200, window, sinks).double() * dout.double()).sum())
        # along the step that was taken (its ends are rounded to fp16)
        along = (grads[which].double() * (steps[0] - steps[1])).sum()
        scale = grads[which].double().norm() * (steps[0] - steps[1]).norm() / 1.0
        assert abs((vals[0] - vals[1]) - along) <= 0.02 * scale, which


def test_rows_behind_the_last_sequence():
    """They are left as they were in an output that the caller gives, and get zero gradients."""
    from talm_amd import _ops

    q, k, v, dout = _inputs(200, 4, 2, torch.float16, True, 3)
    cu = _cu([100, 60])
    out = torch.full((200, 4, D), 7.0, dtype=torch.float16, device="cuda")
    lse = torch.full((4, 200), 3.0, device="cuda")
    torch.ops.talm.attn_window_fwd(q, k, v, cu, 100, 0.1, 20, 2, out, lse)
    assert (out[160:] == 7).all() and (lse[:, 160:] == 3).all() and not (out[:160] == 7).any()
    dq, dk, dv = (torch.full_like(t, 5.0).contiguous() for t in (q, k, v))
    ws = torch.full((_ops.attn_window_bwd_workspace_bytes(200, 4, 2, 2, 100, 20, 2),), 255, dtype=torch.uint8,
                    device="cuda")  # NaN wherever it is read unwritten
    torch.ops.talm.attn_window_bwd(q, k, v, out, dout, lse, cu, 100, 0.1, 20, 2, None, None, dq, dk, dv, ws)
    for t in (dq, dk, dv):
        assert (t[160:] == 0).all() and torch.isfinite(t).all()


def test_keys_outside_every_window_tile_are_not_read():
    """Infinities in k and v where no row of another tile sees them reach no other row."""
    q, k, v, _ = _inputs(512, 2, 1, torch.float16, False, 8)
    want = _call(q, k, v, _cu([512]), 512, 32, 0)
    k, v = k.clone(), v.clone()
    k[:64], v[:64] = math.inf, math.nan
    got = _call(q, k, v, _cu([512]), 512, 32, 0)
    assert torch.equal(got[192:], want[192:])


def test_refusals_on_the_gpu():
    from talm_amd.unpad import window_attention

    q, k, v, _ = _inputs(64, 4, 2, torch.float16, False, 2)
    a = [t.transpose(0, 1)[None] for t in (q, k, v)]
    cu = _cu([64])
    for args in ((a[0], a[1].float(), a[2], cu, 64, 0.1, 4), (a[0][..., :64], a[1][..., :64], a[2][..., :64], cu, 64, 0.1, 4),
                 (a[0], a[1], a[2][:, :1], cu, 64, 0.1, 4), (*a, cu.long(), 64, 0.1, 4),
                 (*a, cu.cpu(), 64, 0.1, 4), (*a, cu, 64, 0.1, 0), (*a, cu, 64, 0.0, 4),
                 (*a, cu, 64, 0.1, 4, -1), (*a, cu, -1, 0.1, 4)):
        with pytest.raises(ValueError):
            window_attention(*args)


def test_odd_strides_and_another_stream():
    """Views that the kernels cannot read are copied; the operands' current stream is used."""
    q, k, v, dout = _inputs(150, 4, 2, torch.float16, False, 4)
    want = _call(q, k, v, _cu([150]), 150, 33, 1, dout)
    wide = [torch.empty(150, t.shape[1], D + 1, dtype=t.dtype, device="cuda") for t in (q, k, v)]
    for w, t in zip(wide, (q, k, v)):
        w[..., 1:] = t
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = _call(*[w[..., 1:] for w in wide], _cu([150]), 150, 33, 1, dout)
    side.synchronize()
    for a, b in zip(got, want):
        assert torch.equal(a, b)


def test_captured_forward_and_backward_replay():
    """Replays follow new inputs and new lengths, with eager work between them."""
    q, k, v, dout = _inputs(640, 4, 2, torch.float16, True, 21)
    cu = _cu([300, 200, 140])
    static = [t.clone() for t in (q, k, v, dout)]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        _call(*static[:3], cu, 640, 50, 3, static[3])
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        outs = _call(*static[:3], cu, 640, 50, 3, static[3])
    for seed, lengths in ((31, [640, 0, 0]), (32, [1, 400, 239]), (33, [300, 200, 140]), (34, [64, 512, 64])):
        fresh = _inputs(640, 4, 2, torch.float16, True, seed)
        for s, t in zip(static, fresh):
            s.copy_(t)
        cu.copy_(_cu(lengths))
        graph.replay()
        torch.cuda.synchronize()
        want = _call(*fresh[:3], _cu(lengths), 640, 50, 3, fresh[3])
        for a, b in zip(outs, want):
            assert torch.equal(a, b)


def test_broadcast_operands_and_gradients():
    """A KV head and gradients given as expanded views: the copies' results, a shared head's gradient the sum of
    what its copies get (two roundings of each, one of their sum: three half steps of the magnitudes)."""
    q, k, v, dout = _inputs(300, 4, 1, torch.float16, True, 9)
    cu = _cu([170, 130])
    want = _call(q, k.expand(300, 2, D).contiguous(), v.expand(300, 2, D).contiguous(), cu, 170, 40, 2, dout)
    from talm_amd.unpad import window_attention

    leaves = [t.transpose(0, 1)[None].detach().requires_grad_() for t in (q, k, v)]
    out = window_attention(leaves[0], *(t.expand(1, 2, 300, D) for t in leaves[1:]), cu, 170, D ** -0.5, 40, 2)
    grads = torch.autograd.grad(out, leaves, dout[None])
    assert torch.equal(out[0].detach(), want[0]) and torch.equal(grads[0][0].transpose(0, 1), want[1])
    for got, copies in zip(grads[1:], want[2:]):
        copies = copies.double()
        tol = 3 * 2.0 ** -11 * copies.abs().sum(1) + 2.0 ** -24
        assert ((got[0, 0].double() - copies.sum(1)).abs() <= tol).all()
    for shape in ((1, 1, 4, D), (1, 300, 1, D), (1, 300, 4, 1), (1, 1, 1, 1)):
        part = torch.randn(shape, device="cuda").half()
        dense = part.expand(1, 300, 4, D).contiguous()
        leaf = q.transpose(0, 1)[None].detach().requires_grad_()
        kv = [t.transpose(0, 1)[None] for t in (k, v)]
        for full in (part.expand(1, 300, 4, D), dense):
            out = window_attention(leaf, *kv, cu, 170, D ** -0.5, 40, 2)
            (g,) = torch.autograd.grad(out, leaf, full)
            first = g if full is not dense else first
        assert torch.equal(first, g)


def test_two_calls_at_once():
    """Calls on two streams, their workspaces their own: each one's results are those it has alone."""
    cases = [(_inputs(2000, 6, 1, torch.float16, True, s), [900, 1100], w, n) for s, w, n in ((3, 100, 5), (4, 300, 0))]
    want = [_call(*t[:3], _cu(ls), 1100, w, n, t[3]) for t, ls, w, n in cases]
    streams = [torch.cuda.Stream() for _ in cases]
    cus = [_cu(ls) for _, ls, _, _ in cases]
    torch.cuda.synchronize()
    for _ in range(3):
        got = []
        for stream, cu, (t, _, w, n) in zip(streams, cus, cases):
            with torch.cuda.stream(stream):
                got.append(_call(*t[:3], cu, 1100, w, n, t[3]))
        torch.cuda.synchronize()
        for a, b in zip(got, want):
            assert all(torch.equal(x, y) for x, y in zip(a, b))


def test_in_inference_mode():
    from talm_amd.dropout import dropout
    from talm_amd.lora import adapter_branch

    q, k, v, _ = _inputs(100, 4, 2, torch.float16, True, 2)
    key = torch.tensor([5, 6], device="cuda")
    x, a, b = torch.randn(9, 64, device="cuda").half(), torch.randn(16, 64, device="cuda"), \
        torch.randn(32, 16, device="cuda")
    want = _call(q, k, v, _cu([100]), 100, 20, 1), dropout(x, 0.3, key), adapter_branch(x, a, b, 1.0, 0.3, key)
    with torch.inference_mode():
        from talm_amd.unpad import window_attention

        out = window_attention(*(t.transpose(0, 1)[None] for t in (q, k, v)), _cu([100]), 100, D ** -0.5, 20, 1)
        got = out[0], dropout(x, 0.3, key), adapter_branch(x, a, b, 1.0, 0.3, key)
    assert all(torch.equal(x, y) for x, y in zip(got, want))


def _poison(like):
    """Leaves NaN in the memory that the next tensors of these sizes get."""
    held = [torch.full((t.numel(),), math.nan, dtype=t.dtype, device="cuda") for t in like for _ in range(4)]
    del held


@pytest.mark.parametrize("half", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("lengths", [[], [0], [0, 0, 0]])
def test_gradients_are_zero_without_a_token_in_a_sequence(lengths, half):
    """No sequence at all, or none with a token: every row lies behind the last one."""
    from talm_amd import _ops

    print(f"[case] window without tokens, lengths={lengths} {half}", flush=True)
    q, k, v, dout = _inputs(70, 4, 2, half, False, 5)
    cu = _cu(lengths) if lengths else torch.zeros(1, dtype=torch.int32, device="cuda")
    for longest in (0, 16):
        _poison((q, k, v))
        _, *grads = _call(q, k, v, cu, longest, 8, 2, dout)
        for g, t in zip(grads, (q, k, v)):
            assert g.shape == t.shape and (g == 0).all()
        out, lse = torch.zeros_like(q), torch.zeros(4, 70, device="cuda")
        angles = torch.rand(70, D, device="cuda")
        for rotated in (False, True):
            dq, dk, dv = (torch.full_like(t, 5.0) for t in (q, k, v))
            ws = torch.full((_ops.attn_window_bwd_workspace_bytes(70, 4, 2, len(lengths), longest, 8, 2),), 255,
                            dtype=torch.uint8, device="cuda")
            torch.ops.talm.attn_window_bwd(q, k, v, out, dout, lse, cu, longest, 0.1, 8, 2,
                                           angles.cos() if rotated else None, angles.sin() if rotated else None,
                                           dq, dk, dv, ws)
            assert not dq.any() and not dk.any() and not dv.any()


@pytest.mark.parametrize("window,sinks", [(40, 2 ** 31 - 1), (2 ** 31 - 1, 3), (2 ** 31 - 1, 2 ** 31 - 1), (70, 5)])
def test_the_largest_arguments_mean_the_whole_rows(window, sinks):
    """The ops with the largest 32-bit longest length, window and sinks: the results of the rows' own sizes."""
    from talm_amd import _ops

    print(f"[case] window={window} sinks={sinks} of a longest length of 2^31 - 1", flush=True)
    lengths = [500, 77, 130]
    n, cu = sum(lengths), _cu(lengths)
    q, k, v, dout = _inputs(n, 4, 2, torch.float16, True, 6)

    def call(longest, window, sinks):
        out, lse = torch.empty_like(dout), torch.empty(4, n, device="cuda")
        torch.ops.talm.attn_window_fwd(q, k, v, cu, longest, 0.1, window, sinks, out, lse)
        grads = [torch.empty(t.shape, dtype=t.dtype, device="cuda") for t in (q, k, v)]
        ws = torch.empty(_ops.attn_window_bwd_workspace_bytes(n, 4, 2, 3, longest, window, sinks), dtype=torch.uint8,
                         device="cuda")
        torch.ops.talm.attn_window_bwd(q, k, v, out, dout, lse, cu, longest, 0.1, window, sinks, None, None, *grads, ws)
        return [out, lse, *grads]
    for a, b in zip(call(2 ** 31 - 1, window, sinks), call(n, min(window, n), min(sinks, n))):
        assert torch.equal(a, b)


@pytest.mark.parametrize("which", [0, 1, 2])
@pytest.mark.parametrize("half,h", [(torch.float16, 2.0 ** -4), (torch.bfloat16, 2.0 ** -3)])
def test_gradients_against_differences_along_them(half, h, which):
    """A central difference of sum(out g) along the gradient itself of q, k or v, whose derivative is of the
    size |gradient| |step|. By the triangle inequality it is off <gradient, step> by at most the two outputs'
    tolerances against |g|, the float64 difference's own distance from the float64 derivative (its
    truncation), and the gradient's tolerance against |step|. A negated, doubled, missing or shifted gradient is
    further off (1.9 to 47 times the bound where float64 stands for the kernels)."""
    print(f"[case] difference along the gradient of {'qkv'[which]} {half}", flush=True)
    lengths, window, sinks, scale = [200, 90], 40, 3, D ** -0.5
    ops = list(_inputs(290, 4, 2, half, False, 13))
    dout, cu = ops.pop(), _cu(lengths)
    grad = _call(*ops, cu, 200, window, sinks, dout)[1 + which].double().cpu()
    vals, tols = _reference(*ops, lengths, scale, window, sinks, dout, half)
    true, tol = vals[1 + which], tols[1 + which]
    direction = h * math.sqrt(true.numel()) * true / true.norm()
    weight, ends = dout.double().cpu(), []
    for sign in (1, -1):
        moved = list(ops)
        moved[which] = (ops[which].double().cpu() + sign * direction).to(half).cuda()
        out = _call(*moved, cu, 200, window, sinks).double().cpu()
        exact, slack = (t[0] for t in _reference(*moved, lengths, scale, window, sinks, dout, half))
        ends.append((moved[which].double().cpu(), out, exact, slack))
    (at, out, exact, slack), (at_, out_, exact_, slack_) = ends
    step = at - at_
    diff = ((out - out_) * weight).sum()
    bound = ((slack + slack_) * weight.abs()).sum() + (tol * step.abs()).sum() \
        + abs(((exact - exact_) * weight).sum() - (true * step).sum())
    print(f"  difference {diff:.1f}, derivative {(grad * step).sum():.1f}, bound {bound:.1f}", flush=True)
    assert abs(diff - (grad * step).sum()) <= bound
    for wrong in (-grad, 2 * grad, 0 * grad, grad.roll(1, 0)):
        assert abs(diff - (wrong * step).sum()) > bound


@pytest.mark.parametrize("half", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("lengths,window,sinks", [
    ([1] * 9, 5, 0), ([1] * 200, 5, 3), ([1, 0, 1], 1, 1),  # rows of one token
    ([300, 65, 1], 1, 0), ([150] * 40, 1, 0),               # a window of one
    ([1300] * 16, 1, 0),                                    # several heads an item
])
def test_rows_that_see_one_key_have_no_gradient_of_their_scores(lengths, window, sinks, half):
    """A softmax over one key is 1 whatever its score: dq and dk are exactly zero, out is v, and dv the sum of
    the group's dO (four products of 1, in fp32, rounded once)."""
    print(f"[case] one key a row: {len(lengths)} sequences, window={window} {half}", flush=True)
    n, hq, hkv = sum(lengths), 8, 2
    q, k, v, dout = _inputs(n, hq, hkv, half, True, 7)
    out, dq, dk, dv = _call(q, k, v, _cu(lengths), max(lengths), window, sinks, dout)
    assert torch.equal(out, v.repeat_interleave(hq // hkv, 1))
    assert not dq.any() and not dk.any()
    want = dout.double().view(n, hkv, hq // hkv, D)
    u = {torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}[half]
    tol = u * want.sum(2).abs() + 4 * 2.0 ** -24 * want.abs().sum(2) + 2.0 ** -25
    assert ((dv.double() - want.sum(2)).abs() <= tol).all()


def test_first_rows_have_no_gradient_of_their_scores():
    """The first row of a sequence sees itself alone, whatever the window; with and without the rotation."""
    from talm_amd import _ops

    lengths, hq, hkv = [200, 1, 77, 130], 4, 2
    n, cu = sum(lengths), _cu(lengths)
    q, k, v, dout = _inputs(n, hq, hkv, torch.float16, True, 8)
    angles = torch.rand(n, D, device="cuda")
    for window, sinks, turned in ((40, 3, False), (1000, 0, True)):
        out, lse = torch.empty_like(dout), torch.empty(hq, n, device="cuda")
        torch.ops.talm.attn_window_fwd(q, k, v, cu, 200, 0.1, window, sinks, out, lse)
        dq, dk, dv = (torch.full(t.shape, 5.0, dtype=t.dtype, device="cuda") for t in (q, k, v))
        ws = torch.empty(_ops.attn_window_bwd_workspace_bytes(n, hq, hkv, 4, 200, window, sinks), dtype=torch.uint8,
                         device="cuda")
        torch.ops.talm.attn_window_bwd(q, k, v, out, dout, lse, cu, 200, 0.1, window, sinks,
                                       angles.cos() if turned else None, angles.sin() if turned else None, dq, dk, dv, ws)
        for first in (0, 200, 201, 278):
            assert not dq[first].any()
        assert not dk[200].any() and dq[1].any() and dk[0].any()


def _forward(q, k, v, lengths, window, sinks, low=True, scale=D ** -0.5):
    from talm_amd import _ops  # noqa: F401 - registers torch.ops.talm.*

    cu = _cu(lengths)
    out, lse = torch.empty_like(q, memory_format=torch.contiguous_format), torch.empty(q.shape[1], q.shape[0], device="cuda")
    lo = torch.full_like(out, 9.0) if low else None
    torch.ops.talm.attn_window_fwd(q, k, v, cu, max(lengths), scale, window, sinks, out, lse, lo)
    return cu, out, lse, lo


def _backward(q, k, v, out, lo, dout, lse, cu, lengths, window, sinks, scale=D ** -0.5):
    from talm_amd import _ops

    grads = [torch.empty(t.shape, dtype=t.dtype, device="cuda") for t in (q, k, v)]
    ws = torch.empty(_ops.attn_window_bwd_workspace_bytes(q.shape[0], q.shape[1], k.shape[1], len(lengths), max(lengths),
                                                          window, sinks), dtype=torch.uint8, device="cuda")
    torch.ops.talm.attn_window_bwd(q, k, v, out, dout, lse, cu, max(lengths), scale, window, sinks, None, None, *grads,
                                   ws, lo)
    return grads


@pytest.mark.parametrize("half", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("lengths,hq,hkv", [([300, 1, 65], 12, 2), ([700], 4, 1), ([40, 64, 16], 12, 4), ([130] * 9, 7, 7)])
def test_the_outputs_remainder(lengths, hq, hkv, half):
    """out_lo is what out's rounding to nearest left off: at most half of out's spacing (2^-8 or 2^-11 of the power
    of two at or below |out|, 2^-25 below fp16's normals), itself rounded once more; out is the same with and without
    it. Rows behind the last sequence are left as they were."""
    print(f"[case] remainder {lengths} {hq}/{hkv} {half}", flush=True)
    n = sum(lengths)
    q, k, v, _ = _inputs(n + 5, hq, hkv, half, True, 12)
    _, out, lse, lo = _forward(q, k, v, lengths, 50, 3)
    _, alone, lse2, _ = _forward(q, k, v, lengths, 50, 3, low=False)
    assert torch.equal(out[:n], alone[:n]) and torch.equal(lse[:, :n], lse2[:, :n]) and (lo[n:] == 9).all()
    out, lo = out[:n].double(), lo[:n].double()
    step = torch.exp2(torch.floor(torch.log2(out.abs().clamp_min(2.0 ** -14 if half == torch.float16 else 2.0 ** -120))))
    u = {torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}[half]
    assert (lo.abs() <= u * step).all() and (lo != 0).double().mean() > 0.9
    # the remainder fills its range: uniform over it, its mean square would be a third of the bound's
    share = (lo ** 2).sum() / ((u * step) ** 2).sum()
    assert 0.2 < share < 0.5, share


@pytest.mark.parametrize("half", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("lengths,window,sinks", [([150, 65], 40, 3), ([2] * 50, 5, 0)])
def test_the_backward_takes_out_and_its_remainder(lengths, window, sinks, half):
    """rowsum(dO (out + out_lo)) of the given tensors, whatever they hold: with an out_lo as large as out the
    gradients are P (dP - that) through K and Q. dS is rounded (u), P carries the fp32 error of its score, the sums of
    128 products 2^-17 of their magnitudes, the result is rounded (u)."""
    print(f"[case] given remainder {lengths[:3]} {half}", flush=True)
    hq, hkv, scale = 4, 2, D ** -0.5
    q, k, v, dout = _inputs(sum(lengths), hq, hkv, half, False, 15)
    cu, out, lse, _ = _forward(q, k, v, lengths, window, sinks)
    g = torch.Generator("cuda").manual_seed(1)
    lo = torch.randn(out.shape, generator=g, device="cuda").to(half)
    got = _backward(q, k, v, out, lo, dout, lse, cu, lengths, window, sinks)
    u = {torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}[half]
    s0 = 0
    want = [torch.zeros(t.shape, dtype=torch.float64) for t in (q, k)]
    tols = [torch.zeros_like(t) for t in want]
    ops = [t.cpu().double() for t in (q, k, v, dout, out, lo)]
    for n in lengths:
        i, rows = torch.arange(n), slice(s0, s0 + n)
        s0 += n
        seen = (i[None] <= i[:, None]) & ((i[:, None] - i[None] < window) | (i[None] < sinks))
        single = seen.sum(1) == 1  # a row that sees one key has no gradient of its score
        for h in range(hq):
            qh, gh, oh, lh = (ops[j][rows, h] for j in (0, 3, 4, 5))
            kh, vh = (ops[j][rows, h // 2] for j in (1, 2))
            s = (scale * qh @ kh.T).masked_fill(~seen, -math.inf)
            p = torch.softmax(s, -1)
            rel = 128 * 2.0 ** -24 * (scale * qh.abs() @ kh.abs().T).max().item() + 2.0 ** -19
            dd = (gh * (oh + lh)).sum(1, keepdim=True)
            mag = (gh.abs() * (oh.abs() + lh.abs())).sum(1, keepdim=True) + gh.abs() @ vh.abs().T
            ds = p * (gh @ vh.T - dd)
            tol = ((u + 2 * rel) * ds.abs() + p * 2.0 ** -16 * mag + 2.0 ** -25) * seen
            dq_row = torch.where(single[:, None], torch.zeros(()), ds)
            want[0][rows, h] = scale * dq_row @ kh
            tols[0][rows, h] = scale * tol @ kh.abs()
            want[1][rows, h // 2] += scale * ds.T @ qh
            tols[1][rows, h // 2] += scale * tol.T @ qh.abs()
    for name, a, b, tol in zip(("dq", "dk"), got, want, tols):
        worst = ((a.cpu().double() - b).abs() / (tol + u * b.abs() + 2.0 ** -25)).max().item()
        print(f"  {name}: {worst:.3f} of its tolerance", flush=True)
        assert worst <= 1.0, name


@pytest.mark.parametrize("half", [torch.float16, torch.bfloat16])
def test_gradients_of_rows_that_see_few_keys(half):
    """Where dO V^T and rowsum(dO O) nearly cancel, the rounding of O would be the gradients' largest error: the
    differentiable call keeps its remainder, and is nearer to 64 bits than the ops on out alone."""
    lengths = [2, 3] * 120
    q, k, v, dout = _inputs(sum(lengths), 8, 2, half, False, 16)
    vals, _ = _reference(q, k, v, lengths, D ** -0.5, 9, 0, dout, half)
    _, *near = _call(q, k, v, _cu(lengths), 3, 9, 0, dout)
    cu, out, lse, _ = _forward(q, k, v, lengths, 9, 0, low=False)
    far = _backward(q, k, v, out, None, dout, lse, cu, lengths, 9, 0)
    u = {torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}[half]
    for name, a, b, want in zip(("dq", "dk"), near, far, vals[1:]):
        e, e_out = (((t.cpu().double() - want).norm() / want.norm()).item() for t in (a, b))
        print(f"  {name}: {e / u:.3f} u, {e_out / u:.3f} u of out alone", flush=True)
        assert e <= 0.85 * e_out


def test_the_remainder_is_checked():
    q, k, v, dout = _inputs(64, 4, 2, torch.float16, False, 2)
    cu, out, lse, lo = _forward(q, k, v, [64], 9, 0)
    for bad in (lo.float(), lo[:, :2], lo.transpose(0, 1).contiguous().transpose(0, 1), lo.cpu()):
        with pytest.raises(ValueError):
            torch.ops.talm.attn_window_fwd(q, k, v, cu, 64, 0.1, 9, 0, out, lse, bad)
        with pytest.raises(ValueError):
            _backward(q, k, v, out, bad, dout, lse, cu, [64], 9, 0)
