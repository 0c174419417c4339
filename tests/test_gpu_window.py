"""Sliding-window attention with sinks against its float64 statement: forward,
gradients, caches and decode steps, over types, head layouts, windows, ragged
packed batches, padding, strides, graphs and streams."""

import pytest
import torch

import _packed_oracle as O

pytestmark = pytest.mark.gpu

DT = {"bf16": torch.bfloat16, "fp16": torch.float16, "f32": torch.float32}


def _inputs(dev, lens, Hq, Hkv, Dh, dtype, pad=0, seed=0, gscale=1.0):
    g = torch.Generator().manual_seed(seed)
    T = sum(lens) + pad
    q, gy = (torch.randn(T, Hq, Dh, generator=g) for _ in range(2))
    k, v = (torch.randn(T, Hkv, Dh, generator=g) for _ in range(2))
    return [t.to(dtype).to(dev) for t in (q, k, v, gy * gscale)] + [O.borders(lens).to(dev)]


def _step(mr, q, k, v, gy, cu, window, sinks, scale=None):
    leaves = [t.detach().clone().requires_grad_() for t in (q, k, v)]
    y = mr.window_attention_packed(*leaves, cu, window, sinks=sinks, scale=scale)
    return [y.detach(), *torch.autograd.grad(y, leaves, gy)]


def _check(mr, ins, window, sinks, scale=None):
    q, k, v, gy, cu = ins
    got = _step(mr, q, k, v, gy, cu, window, sinks, scale)
    assert all(t.dtype == q.dtype for t in got)
    W = O.Attention(q, k, v, cu, window, sinks, gy, scale)
    for name, g, w, t in (("y", got[0], W.y, W.tol_y), ("grad_q", got[1], W.gq, W.tol_gq),
                          ("grad_k", got[2], W.gk, W.tol_gk), ("grad_v", got[3], W.gv, W.tol_gv)):
        O.check(name, g, w, t)
    return got


LENS = {
    "one_token": [1],
    "ones_and_zeros": [1, 0, 1, 1, 0, 2],
    "tile_borders": [128, 127, 1, 129, 64, 0, 63],
    "ragged": [5, 290, 0, 33, 401, 1],
    "long": [1100],
    "many_short": [3, 1, 7, 2] * 30,
}


@pytest.mark.parametrize("dtype", ["bf16", "fp16", "f32"])
@pytest.mark.parametrize("window,sinks", [(1, 0), (1, 3), (64, 4), (129, 1), (200, 64), (4096, 5)])
@pytest.mark.parametrize("lens", sorted(LENS))
def test_window_attention_packed(mr, cuda_dev, lens, window, sinks, dtype):
    _check(mr, _inputs(cuda_dev, LENS[lens], 2, 1, 64, DT[dtype], seed=window), window, sinks)


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("Dh", [32, 64, 96, 128])
@pytest.mark.parametrize("Hq,Hkv", [(1, 1), (3, 1), (4, 4), (8, 2)])
def test_head_layouts(mr, cuda_dev, Hq, Hkv, Dh, dtype):
    _check(mr, _inputs(cuda_dev, [150, 260], Hq, Hkv, Dh, DT[dtype], seed=Dh), 100, 2)


@pytest.mark.parametrize("dtype", ["bf16", "fp16", "f32"])
def test_dense_batch_equals_packed(mr, cuda_dev, dtype):
    B, L = 3, 200
    q, k, v, gy, cu = _inputs(cuda_dev, [L] * B, 4, 2, 64, DT[dtype], seed=1)
    want = _check(mr, (q, k, v, gy, cu), 70, 4)
    leaves = [t.detach().unflatten(0, (B, L)).clone().requires_grad_() for t in (q, k, v)]
    y = mr.window_attention(*leaves, 70, sinks=4)
    grads = torch.autograd.grad(y, leaves, gy.unflatten(0, (B, L)))
    for got, w in zip((y, *grads), want):
        assert torch.equal(got.flatten(0, 1), w)


def test_reference_loop_agrees(mr, cuda_dev):
    q, k, v, gy, cu = _inputs(cuda_dev, [120], 4, 2, 32, torch.float32, seed=2)
    W = O.Attention(q, k, v, cu, 30, 3)
    y = mr.window_attention_reference(q[None].double(), k[None].double(), v[None].double(), 30, sinks=3)[0]
    assert (y - W.y).abs().max() < 1e-12


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
def test_large_scores(mr, cuda_dev, dtype):
    """Scores of several hundred: the running maximum has to carry them. A one-hot-like softmax."""
    q, k, v, gy, cu = _inputs(cuda_dev, [300], 2, 2, 64, DT[dtype], seed=3)
    _check(mr, (q * 8, k * 8, v, gy, cu), 150, 2)


def test_scale_argument(mr, cuda_dev):
    _check(mr, _inputs(cuda_dev, [200], 2, 1, 64, torch.bfloat16, seed=4), 90, 1, scale=0.5)


@pytest.mark.parametrize("gscale", [1e-5, 3e4])
def test_fp16_gradients_of_any_size(mr, cuda_dev, gscale):
    """Loss scaling moves grad_y over many powers of two; what lies between grad_y and the gradients must not
    overflow or vanish in fp16 (the gradients themselves here do neither, save below fp16's smallest number)."""
    q, k, v, gy, cu = _inputs(cuda_dev, [300], 2, 1, 64, torch.float16, seed=5, gscale=1.0)
    gy = (gy * 0.2 * gscale).clamp(-6e4, 6e4)
    q, v = q * 0.05, v * 0.02
    got = _step(mr, q, k, v, gy, cu, 120, 2)
    W = O.Attention(q, k, v, cu, 120, 2, gy)
    fits = W.gv.abs().max() < 6e4
    assert fits
    for name, g, w, t in (("y", got[0], W.y, W.tol_y), ("grad_q", got[1], W.gq, W.tol_gq),
                          ("grad_k", got[2], W.gk, W.tol_gk), ("grad_v", got[3], W.gv, W.tol_gv)):
        O.check(name, g, w, t)


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
def test_padding_rows(mr, cuda_dev, dtype):
    """Rows behind the last sequence: zeros come out, and what they hold changes nothing."""
    lens, pad = [100, 0, 173], 90
    q, k, v, gy, cu = _inputs(cuda_dev, lens, 4, 2, 64, DT[dtype], pad=pad, seed=6)
    n = sum(lens)
    want = None
    for junk in (0.0, float("nan"), float("inf")):
        for t in (q, k, v, gy):
            t[n:] = junk
        got = _check(mr, (q, k, v, gy, cu), 64, 4)
        assert all((t[n:] == 0).all() for t in got)
        assert want is None or all(torch.equal(a, b) for a, b in zip(got, want))
        want = got


@pytest.mark.parametrize("dtype", ["bf16", "fp16", "f32"])
@pytest.mark.parametrize("bad", [float("nan"), float("inf")])
def test_unseen_values_have_no_influence(mr, cuda_dev, dtype, bad):
    """A token's q, k, v, gy reach only the rows that see it (or that it sees), not the others of its tiles."""
    lens, window, sinks, at = [90, 200, 150], 40, 3, 90 + 100
    q, k, v, gy, cu = _inputs(cuda_dev, lens, 2, 1, 64, DT[dtype], seed=7)
    W = O.Attention(q, k, v, cu, window, sinks, gy)
    see = O.visible(sum(lens), cu, window, sinks, cuda_dev)
    k, v = k.clone(), v.clone()
    k[at], v[at] = bad, bad
    got = _step(mr, q, k, v, gy, cu, window, sinks)
    sees = see[:, at]  # queries whose row the bad key reaches
    O.check("y", got[0][~sees], W.y[~sees], W.tol_y[~sees])
    O.check("grad_q", got[1][~sees], W.gq[~sees], W.tol_gq[~sees])
    touched = see[sees].any(0)  # keys that such a query sees
    O.check("grad_k", got[2][~touched], W.gk[~touched], W.tol_gk[~touched])
    O.check("grad_v", got[3][~touched], W.gv[~touched], W.tol_gv[~touched])
    assert not torch.isfinite(got[0][sees].float()).all(-1).any()
    q, k, v, gy, cu = _inputs(cuda_dev, lens, 2, 1, 64, DT[dtype], seed=7)
    q, gy = q.clone(), gy.clone()
    q[at], gy[at] = bad, bad
    got = _step(mr, q, k, v, gy, cu, window, sinks)
    mine = see[at]  # keys that the bad query sees
    rows = torch.arange(sum(lens), device=cuda_dev) != at
    O.check("y", got[0][rows], W.y[rows], W.tol_y[rows])
    O.check("grad_q", got[1][rows], W.gq[rows], W.tol_gq[rows])
    O.check("grad_k", got[2][~mine], W.gk[~mine], W.tol_gk[~mine])
    O.check("grad_v", got[3][~mine], W.gv[~mine], W.tol_gv[~mine])
    assert not torch.isfinite(got[2][mine].float()).all(-1).any()


def test_gradients_against_differences(mr, cuda_dev):
    q, k, v, gy, cu = _inputs(cuda_dev, [90, 75], 2, 1, 32, torch.float32, seed=8)
    got = _step(mr, q, k, v, gy, cu, 33, 2)
    W = O.Attention(q, k, v, cu, 33, 2, gy)
    eps = 1e-5
    for n, (at, tol) in enumerate((((100, 1, 3), W.tol_gq), ((91, 0, 5), W.tol_gk), ((130, 0, 7), W.tol_gv))):
        loss = []
        for d in (eps, -eps):
            t = [x.double().clone() for x in (q, k, v)]
            t[n][at] += d
            loss.append((O.Attention(*t, cu, 33, 2).y * gy.double()).sum())
        diff = float((loss[0] - loss[1]) / (2 * eps))
        # central differences: eps^2 times a third derivative of at most a few hundred, and 2^-52 |loss| / eps
        assert abs(float(got[n + 1][at]) - diff) <= float(tol[at]) + 1e-7


def test_fused_projection_slices_are_read_in_place(mr, cuda_dev):
    q, k, v, gy, cu = _inputs(cuda_dev, [130, 99], 4, 2, 64, torch.bfloat16, seed=9)
    want = _step(mr, q, k, v, gy, cu, 50, 2)
    fused = torch.cat((q.flatten(1), k.flatten(1), v.flatten(1)), 1).requires_grad_()
    parts = [t.unflatten(1, (-1, 64)) for t in fused.split([256, 128, 128], 1)]
    y = mr.window_attention_packed(*parts, cu.int(), 50, sinks=2)
    grad, = torch.autograd.grad(y, fused, gy)
    assert torch.equal(y, want[0])
    assert torch.equal(grad, torch.cat([t.flatten(1) for t in want[1:]], 1))
    # head-major memory, and a start off the alignment
    kt = k.transpose(0, 1).contiguous().transpose(0, 1)
    off = torch.empty(v.numel() + 1, dtype=v.dtype, device=cuda_dev)[1:].view_as(v)
    off.copy_(v)
    assert torch.equal(mr.window_attention_packed(q, kt, off, cu, 50, sinks=2), want[0])
    # a broadcast head
    ke = k[:, :1].expand(-1, 2, -1)
    a = mr.window_attention_packed(q, ke, v, cu, 50, sinks=2)
    assert torch.equal(a, mr.window_attention_packed(q, ke.contiguous(), v, cu, 50, sinks=2))


def test_results_do_not_vary(mr, cuda_dev):
    ins = _inputs(cuda_dev, [700, 900], 8, 2, 128, torch.bfloat16, seed=10)
    want = _step(mr, *ins, 300, 4)
    for _ in range(3):
        assert all(torch.equal(a, b) for a, b in zip(_step(mr, *ins, 300, 4), want))


def test_graph_replay_and_side_stream(mr, cuda_dev):
    q, k, v, gy, cu = _inputs(cuda_dev, [200, 0, 150], 4, 2, 64, torch.bfloat16, seed=11)
    static = [t.clone() for t in (q, k, v, gy)] + [cu.int()]
    side = torch.cuda.Stream(cuda_dev)
    side.wait_stream(torch.cuda.current_stream(cuda_dev))
    with torch.cuda.stream(side):
        first = _step(mr, *static, 64, 4)
    torch.cuda.current_stream(cuda_dev).wait_stream(side)
    graphs, outs = [torch.cuda.CUDAGraph() for _ in range(2)], []
    for g in graphs:
        with torch.cuda.graph(g):
            outs.append(_step(mr, *static, 64, 4))
    assert all(torch.equal(a, b) for a, b in zip(first, _step(mr, q, k, v, gy, cu, 64, 4)))
    for s, t in zip(static, (q.flip(0), k.flip(0), v.flip(0), gy.flip(0), O.borders([0, 150, 200]).to(cuda_dev))):
        s.copy_(t)
    for _ in range(2):
        for g in graphs:
            g.replay()
    torch.cuda.synchronize()
    want = _step(mr, *static, 64, 4)
    assert all(torch.equal(a, b) for o in outs for a, b in zip(o, want))


def test_two_streams_at_once(mr, cuda_dev):
    """Forward and backward of different head sizes (TMEM and shared memory shares) at the same time."""
    ins = [_inputs(cuda_dev, [900, 700], 8, 4, Dh, torch.bfloat16, seed=20 + Dh) for Dh in (64, 128)]
    want = [_step(mr, *i, 200, 4) for i in ins]
    streams = [torch.cuda.Stream(cuda_dev) for _ in ins]
    torch.cuda.synchronize()
    got = [[], []]
    for _ in range(5):
        for n, s in enumerate(streams):
            with torch.cuda.stream(s):
                got[n].append(_step(mr, *ins[n], 200, 4))
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for n in range(2) for g in got[n] for a, b in zip(g, want[n]))


def test_padded_front(mr, cuda_dev):
    """Borders that do not start at 0: the rows before them belong to no sequence either."""
    q, k, v, gy, _ = _inputs(cuda_dev, [50, 160, 90], 2, 1, 64, torch.bfloat16, seed=23)
    for t in (q, k, v, gy):
        t[:50] = float("nan")
    cu = torch.tensor([50, 210, 300], device=cuda_dev)
    got = _check(mr, (q, k, v, gy, cu), 40, 2)
    assert all((t[:50] == 0).all() for t in got)


def test_empty_batches(mr, cuda_dev):
    z = torch.zeros(0, 2, 64, device=cuda_dev, dtype=torch.bfloat16, requires_grad=True)
    cu = torch.tensor([0, 0, 0], device=cuda_dev)
    y, ck, cv = mr.window_attention_packed_with_state(z, z, z, cu, 10, sinks=2)
    assert y.shape == z.shape and ck.shape == (2, 12, 2, 64) and (ck == 0).all() and (cv == 0).all()
    assert torch.autograd.grad(y, z, torch.zeros_like(y))[0].shape == z.shape
    q = torch.randn(7, 2, 64, device=cuda_dev)
    assert (mr.window_attention_packed(q, q, q, torch.tensor([0], device=cuda_dev), 10) == 0).all()
    assert mr.window_attention(q[:0].view(0, 5, 2, 64), q[:0].view(0, 5, 2, 64), q[:0].view(0, 5, 2, 64), 3).numel() == 0


# ---- caches and decode steps -------------------------------------------------------------------


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("window,sinks", [(1, 0), (16, 4), (50, 0), (300, 2)])
def test_caches_hold_the_newest_tokens(mr, cuda_dev, window, sinks, dtype):
    lens = [0, 1, 5, 16, 20, 21, 150, 333]
    q, k, v, gy, cu = _inputs(cuda_dev, lens, 2, 2, 32, DT[dtype], seed=12)
    y, ck, cv = mr.window_attention_packed_with_state(q, k, v, cu, window, sinks=sinks)
    assert torch.equal(y, mr.window_attention_packed(q, k, v, cu, window, sinks=sinks))
    for cache, src in ((ck, k), (cv, v)):
        want = torch.zeros_like(cache)
        for s, (lo, hi) in enumerate(zip(cu[:-1].tolist(), cu[1:].tolist())):
            for t in range(hi - lo):
                want[s, t if t < sinks else sinks + (t - sinks) % window] = src[lo + t]
        assert torch.equal(cache, want)


@pytest.mark.parametrize("dtype", ["bf16", "fp16", "f32"])
@pytest.mark.parametrize("Hq,Hkv,Dh", [(2, 2, 32), (8, 2, 64), (10, 1, 64), (3, 1, 96), (16, 4, 128)])
def test_step(mr, cuda_dev, Hq, Hkv, Dh, dtype):
    """One step at positions from the first token to far past the window, free rows among them."""
    window, sinks = 37, 3
    pos = torch.tensor([0, 1, 2, 3, 36, 39, 40, 41, -1, 77, 1 << 40, -5], device=cuda_dev)
    B, slots, dt = len(pos), window + sinks, DT[dtype]
    g = torch.Generator().manual_seed(13)
    q = torch.randn(B, Hq, Dh, generator=g).to(dt).to(cuda_dev)
    k, v = (torch.randn(B, Hkv, Dh, generator=g).to(dt).to(cuda_dev) for _ in range(2))
    ck, cv = (torch.randn(B, slots, Hkv, Dh, generator=g).to(dt).to(cuda_dev) for _ in range(2))
    for b, p in enumerate(pos.tolist()):  # slots that no token has reached hold anything
        if 0 <= p < slots:
            ck[b, p:], cv[b, p:] = float("nan"), float("inf")
    old = (ck.clone(), cv.clone())
    y = mr.window_attention_step(q, k, v, ck, cv, pos, sinks=sinks)
    assert y.dtype == dt
    for b, p in enumerate(pos.tolist()):
        if p < 0:
            assert (y[b] == 0).all()
        else:
            n, slot = min(p + 1, slots), p if p < sinks else sinks + (p - sinks) % window
            old[0][b, slot], old[1][b, slot] = k[b], v[b]
            # the visible tokens in slot order, the query as the newest of a window that sees them all
            qq = torch.zeros(n, Hq, Dh, dtype=dt, device=cuda_dev)
            qq[-1] = q[b]
            W = O.Attention(qq, old[0][b, :n], old[1][b, :n], torch.tensor([0, n]), n, 0)
            O.check(f"y at position {p}", y[b], W.y[-1], W.tol_y[-1])
    for a, b in zip((ck, cv), old):
        assert torch.equal(a.nan_to_num(7.0, 8.0), b.nan_to_num(7.0, 8.0))


@pytest.mark.parametrize("dtype,Hq,Hkv,Dh,window,sinks", [("bf16", 4, 2, 64, 48, 4), ("f32", 2, 2, 32, 20, 0),
                                                          ("fp16", 6, 1, 128, 130, 1)])
def test_decoding_continues_a_prefill(mr, cuda_dev, dtype, Hq, Hkv, Dh, window, sinks):
    """Prefill, then 30 steps: each step's row equals the row of the whole sequence."""
    lens, more = [1, 30, 300], 30
    q, k, v, gy, cu = _inputs(cuda_dev, [n + more for n in lens], Hq, Hkv, Dh, DT[dtype], seed=14)
    W = O.Attention(q, k, v, cu, window, sinks)
    part = [torch.cat([t[lo:lo + n] for lo, n in zip(cu.tolist(), lens)]) for t in (q, k, v)]
    y, ck, cv = mr.window_attention_packed_with_state(*part, O.borders(lens).to(cuda_dev), window, sinks=sinks)
    pos = torch.tensor(lens, device=cuda_dev)
    for _ in range(more):
        rows = cu[:-1] + pos
        y = mr.window_attention_step(q[rows], k[rows], v[rows], ck, cv, pos, sinks=sinks)
        O.check("step", y, W.y[rows], W.tol_y[rows])
        pos += 1


@pytest.mark.parametrize("B", [1, 5])
def test_step_long_cache(mr, cuda_dev, B):
    """A cache long enough that its slots are split over blocks; int32 positions."""
    Hq, Hkv, Dh, window, sinks, dt = 8, 2, 64, 5000, 4, torch.bfloat16
    g = torch.Generator(device=cuda_dev).manual_seed(15)
    r = dict(device=cuda_dev, generator=g)
    q, k, v = (torch.randn(B, h, Dh, **r).to(dt) for h in (Hq, Hkv, Hkv))
    ck, cv = (torch.randn(B, window + sinks, Hkv, Dh, **r).to(dt) for _ in range(2))
    pos = torch.tensor([7000, 4000, 100, 5003, 5004][:B], device=cuda_dev)
    y = mr.window_attention_step(q, k, v, ck, cv, pos.int(), sinks=sinks)
    for b, p in enumerate(pos.tolist()):
        n = min(p + 1, window + sinks)
        s = torch.einsum("gd,nd->gn", q[b, 0:4].double(), ck[b, :n, 0].double()) / 8
        w = torch.softmax(s, -1)
        vv = cv[b, :n, 0].double()
        size = (q[b, 0:4].double().abs() @ ck[b, :n, 0].double().abs().T).amax(-1, keepdim=True) / 8
        relp = 2 * (Dh + 4) * O.U32 * size + n * O.U32
        tol = (O.half_step(dt) + relp) * (w @ vv.abs())
        O.check("y", y[b, 0:4], w @ vv, tol * (1 + 2.0 ** -8) + O.half_step(dt) * (w @ vv).abs())


def test_step_replays_from_a_graph(mr, cuda_dev):
    """A captured decode step, its position advanced inside the graph, equals eager steps."""
    B, Hq, Hkv, Dh, window, sinks, dt = 3, 4, 2, 64, 12, 2, torch.bfloat16
    g = torch.Generator().manual_seed(16)
    toks = [[torch.randn(B, h, Dh, generator=g).to(dt).to(cuda_dev) for h in (Hq, Hkv, Hkv)] for _ in range(20)]
    eager = [torch.zeros(B, window + sinks, Hkv, Dh, dtype=dt, device=cuda_dev) for _ in range(2)]
    pos = torch.tensor([0, 5, -1], device=cuda_dev)
    want = []
    for t in toks:
        want.append(mr.window_attention_step(*t, *eager, pos, sinks=sinks))
        pos += (pos >= 0).long()
    static, caches = [t.clone() for t in toks[0]], [torch.zeros_like(t) for t in eager]
    pos = torch.tensor([0, 5, -1], device=cuda_dev)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y = mr.window_attention_step(*static, *caches, pos, sinks=sinks)
        pos += (pos >= 0).long()
    for t, w in zip(toks, want):
        for s, x in zip(static, t):
            s.copy_(x)
        graph.replay()
        assert torch.equal(y, w)
    assert all(torch.equal(a, b) for a, b in zip(caches, eager))


def test_hybrid_layer_trains_and_decodes(mr, cuda_dev):
    """The operators together, as a hybrid model runs them: a packed RG-LRU layer feeding a packed window-attention
    layer, the gradients of both, and decoding both from their states."""
    lens, D, H, Dh, window, sinks = [60, 1, 145], 64, 2, 32, 24, 2
    g = torch.Generator().manual_seed(17)
    T = sum(lens) + 3 * 10
    full = [n + 10 for n in lens]
    a = (torch.rand(T, D, generator=g) * 0.5 + 0.45).to(cuda_dev)
    x = torch.randn(T, D, generator=g).to(cuda_dev)
    k, v = (torch.randn(T, H, Dh, generator=g).to(cuda_dev) for _ in range(2))
    gy = torch.randn(T, H, Dh, generator=g).to(cuda_dev)
    cu = O.borders(full).to(cuda_dev)

    la, lx, lk, lv = (t.clone().requires_grad_() for t in (a, x, k, v))
    h = mr.rglru_scan_packed(la, lx, cu)
    y = mr.window_attention_packed(h.view(T, H, Dh), lk, lv, cu, window, sinks=sinks)
    got = torch.autograd.grad(y, (la, lx, lk, lv), gy)
    h64, _, _ = O.scan_forward(a, x, cu)
    W = O.Attention(h64.view(T, H, Dh), k.double(), v.double(), cu, window, sinks, gy.double())
    ga, gx, _ = O.scan_backward(a, x, cu, W.gq.reshape(T, D))
    # float32 throughout: the scan's rounding reaches the scores (|h| up to tens), the softmax's the gradients; each of
    # some 200 steps and keys contributes half a step: 1e-4 of the largest value is above 200 * 2^-24 * 8 = 1e-4
    for p, w in ((y, W.y), (got[0], ga), (got[1], gx), (got[2], W.gk), (got[3], W.gv)):
        assert (p.double() - w).abs().max() <= 1e-4 * w.abs().max()

    pre = torch.cat([torch.arange(lo, lo + n) for lo, n in zip(cu.tolist(), lens)]).to(cuda_dev)
    cp = O.borders(lens).to(cuda_dev)
    hp, state = mr.rglru_scan_packed_with_state(a[pre], x[pre], cp)
    _, ck, cv = mr.window_attention_packed_with_state(hp.view(-1, H, Dh), k[pre], v[pre], cp, window, sinks=sinks)
    pos = torch.tensor(lens, device=cuda_dev)
    for _ in range(10):
        rows = cu[:-1] + pos
        ht = mr.rglru_step(a[rows], x[rows], state)
        yt = mr.window_attention_step(ht.view(-1, H, Dh), k[rows], v[rows], ck, cv, pos, sinks=sinks)
        assert (yt.double() - W.y[rows]).abs().max() <= 1e-4 * W.y.abs().max()
        pos += 1


def test_offsets_past_32_bits(mr, cuda_dev):
    """More than 2^31 elements in q, k, v. A window of one token returns v, and passes grad_y to v alone."""
    T, H, Dh = 1 << 20, 17, 128
    r = dict(device=cuda_dev, dtype=torch.bfloat16)
    v = torch.arange(T, device=cuda_dev).remainder(253).to(torch.bfloat16)[:, None, None].expand(T, H, Dh).contiguous()
    q, k, gy = torch.ones(T, H, Dh, **r), torch.ones(T, H, Dh, **r), torch.full((T, H, Dh), 3.0, **r)
    for t in (q, k, v):
        t.requires_grad_()
    y = mr.window_attention(q[None], k[None], v[None], 1)[0]
    gq, gk, gv = torch.autograd.grad(y, (q, k, v), gy)
    assert torch.equal(y, v) and bool((gv == 3).all())
    # dS = p (gy.v - delta) with delta from the same v: a rounding of sums of 128 terms of up to 3 * 252
    assert gq.abs().max() <= 128 * 756 * 256 * O.U32 and gk.abs().max() <= 128 * 756 * 256 * O.U32


def test_step_offsets_past_32_bits(mr, cuda_dev):
    B, Hkv, Dh, window, dt = 3, 8, 128, 1 << 20, torch.bfloat16
    ck, cv = (torch.empty(B, window, Hkv, Dh, dtype=dt, device=cuda_dev) for _ in range(2))
    assert ck[:2].numel() >= 1 << 31
    g = torch.Generator(device=cuda_dev).manual_seed(18)
    q, k, v = (torch.randn(B, Hkv, Dh, device=cuda_dev, generator=g).to(dt) for _ in range(3))
    n = 100
    ck[2, :n], cv[2, :n] = (torch.randn(n, Hkv, Dh, device=cuda_dev, generator=g).to(dt) for _ in range(2))
    y = mr.window_attention_step(q, k, v, ck, cv, torch.tensor([-1, 0, n], device=cuda_dev))
    assert (y[0] == 0).all() and torch.equal(y[1], v[1]) and torch.equal(ck[2, n], k[2]) and torch.equal(cv[2, n], v[2])
    qq = torch.zeros(n + 1, Hkv, Dh, dtype=dt, device=cuda_dev)
    qq[-1] = q[2]
    W = O.Attention(qq, ck[2, :n + 1], cv[2, :n + 1], torch.tensor([0, n + 1]), n + 1, 0)
    O.check("y", y[2], W.y[-1], W.tol_y[-1])


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
def test_many_query_heads_per_key_head(mr, cuda_dev, dtype):
    """40 query heads on one key head: the step takes them 16 at a time, the gradient sums them all."""
    window, sinks, dt = 20, 1, DT[dtype]
    ins = _inputs(cuda_dev, [70, 33], 40, 1, 32, dt, seed=19)
    _check(mr, ins, window, sinks)
    q, k, v, _, cu = ins
    W = O.Attention(q, k, v, cu, window, sinks)
    _, ck, cv = mr.window_attention_packed_with_state(q[:69], k[:69], v[:69], cu[:1].new_tensor([0, 69]), window, sinks=sinks)
    y = mr.window_attention_step(q[69:70], k[69:70], v[69:70], ck, cv, cu.new_tensor([69]), sinks=sinks)
    O.check("step", y, W.y[69:70], W.tol_y[69:70])
