"""rglru_scan_packed against its step-by-step float64 statement: ragged lengths
(zero, one, chunk borders), any width, every type, states, padding, strides,
streams, graphs."""

import pytest
import torch

import _packed_oracle as O

pytestmark = pytest.mark.gpu

DT = {"bf16": torch.bfloat16, "fp16": torch.float16, "f32": torch.float32}


def _inputs(dev, lens, D, dtype, pad=0, seed=0, wild=False):
    g = torch.Generator().manual_seed(seed)
    T, S = sum(lens) + pad, len(lens)
    a = torch.rand(T, D, generator=g) * 0.6 + 0.4 if not wild else torch.randn(T, D, generator=g)
    x, gy = torch.randn(T, D, generator=g), torch.randn(T, D, generator=g)
    h0, gf = torch.randn(S, D, generator=g), torch.randn(S, D, generator=g)
    return [t.to(dev) for t in (a.to(dtype), x.to(dtype), gy, h0, gf)] + [O.borders(lens).to(dev)]


def _check(mr, a, x, gy, h0, gf, cu, state):
    h, f = (h0, gf) if state else (None, None)
    leaves = [t.detach().clone().requires_grad_() for t in ((a, x, h0) if state else (a, x))]
    if state:
        y, final = mr.rglru_scan_packed_with_state(leaves[0], leaves[1], cu, h0=leaves[2])
        grads = torch.autograd.grad((y, final), leaves, (gy, gf))
    else:
        y = mr.rglru_scan_packed(leaves[0], leaves[1], cu)
        grads = torch.autograd.grad(y, leaves, gy)
    assert y.dtype == torch.float32 and grads[0].dtype == a.dtype
    wy, _, wf = O.scan_forward(a, x, cu, h)
    wa, wx, wh = O.scan_backward(a, x, cu, gy, f, h)
    ty, tf, ta, tx, th = O.scan_bounds(a, x, cu, gy, f, h)
    r = 0.0 if a.dtype == torch.float32 else O.half_step(a.dtype)
    tiny = 2.0 ** -25 if a.dtype == torch.float16 else 0.0
    O.check("y", y, wy, ty)
    O.check("grad_a", grads[0], wa, ta + r * (wa.abs() + ta) + tiny)
    O.check("grad_x", grads[1], wx, tx + r * (wx.abs() + tx) + tiny)
    if state:
        O.check("final", final, wf, tf)
        O.check("grad_h0", grads[2], wh, th)


LENS = {
    "one_token": [1],
    "ones_and_zeros": [0, 1, 0, 0, 1, 1, 0],
    "chunk_borders": [128, 127, 1, 129, 256, 0, 64],
    "ragged": [3, 300, 17, 0, 41, 530, 1],
    "long": [2100],
    "many_short": [2, 1, 3] * 60,
}


@pytest.mark.parametrize("dtype", ["bf16", "fp16", "f32"])
@pytest.mark.parametrize("D", [1, 33, 64, 130])
@pytest.mark.parametrize("lens", sorted(LENS))
def test_packed_scan(mr, cuda_dev, lens, D, dtype):
    _check(mr, *_inputs(cuda_dev, LENS[lens], D, DT[dtype]), state=D != 64)


@pytest.mark.parametrize("state", [False, True])
def test_gates_of_any_value(mr, cuda_dev, state):
    """Negative gates, gates above one and exact zeros (short sequences: products stay finite)."""
    a, *rest = _inputs(cuda_dev, [20, 150, 9], 40, torch.float32, wild=True, seed=3)
    a[5] = 0.0
    a.clamp_(-1.05, 1.05)
    _check(mr, a, *rest, state=state)


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
def test_padding_rows_come_out_as_zeros(mr, cuda_dev, dtype):
    lens, pad, D = [70, 200, 0], 77, 96
    a, x, gy, h0, gf, cu = _inputs(cuda_dev, lens, D, DT[dtype], pad=pad, seed=4)
    n = sum(lens)
    want = None
    for junk in (0.0, float("nan"), float("inf")):
        for t in (a, x, gy):
            t[n:] = junk
        la, lx, lh = (t.detach().clone().requires_grad_() for t in (a, x, h0))
        y, final = mr.rglru_scan_packed_with_state(la, lx, cu, h0=lh)
        got = [y.detach(), final.detach(), *torch.autograd.grad((y, final), (la, lx, lh), (gy, gf))]
        for t in (got[0], got[2], got[3]):
            assert (t[n:] == 0).all()
        if want is not None:
            assert all(torch.equal(p, q) for p, q in zip(got, want))
        want = got


def test_padded_front(mr, cuda_dev):
    """Borders that do not start at 0: the rows before them belong to no sequence either."""
    a, x, gy, _, _, _ = _inputs(cuda_dev, [140, 200], 32, torch.float32, seed=13)
    a[:140], x[:140], gy[:140] = float("nan"), float("inf"), float("nan")
    cu = torch.tensor([140, 150, 340], device=cuda_dev)
    la, lx = (t.clone().requires_grad_() for t in (a, x))
    y = mr.rglru_scan_packed(la, lx, cu)
    got = [y.detach(), *torch.autograd.grad(y, (la, lx), gy)]
    want = mr.rglru_scan_packed(a[140:], x[140:], cu - 140)
    assert all((t[:140] == 0).all() for t in got)
    tol, *_ = O.scan_bounds(a[140:], x[140:], cu - 140, gy[140:])
    assert ((got[0][140:] - want).double().abs() <= 2 * tol).all() and all(torch.isfinite(t).all() for t in got)


def test_nan_stays_in_its_sequence(mr, cuda_dev):
    lens = [130, 60, 140]
    a, x, gy, h0, gf, cu = _inputs(cuda_dev, lens, 64, torch.bfloat16, seed=5)
    x[150] = float("nan")  # in the second sequence
    a[170] = float("inf")
    la, lx = (t.detach().clone().requires_grad_() for t in (a, x))
    y = mr.rglru_scan_packed(la, lx, cu)
    ga, gx = torch.autograd.grad(y, (la, lx), gy)
    for t in (y, ga, gx):
        assert torch.isfinite(t[:130].float()).all() and torch.isfinite(t[190:].float()).all()
    assert torch.isnan(y[150:190]).all()


def test_split_scan_property(mr, cuda_dev):
    """A scan continued from the returned state equals the whole scan (exactly the same sums up to rounding)."""
    a, x, gy, h0, gf, cu = _inputs(cuda_dev, [700], 48, torch.float32, seed=6)
    whole = mr.rglru_scan_packed(a, x, cu)
    y1, s1 = mr.rglru_scan_packed_with_state(a[:300], x[:300], torch.tensor([0, 300], device=cuda_dev))
    y2 = mr.rglru_scan_packed(a[300:], x[300:], torch.tensor([0, 400], device=cuda_dev), h0=s1)
    tol, *_ = O.scan_bounds(a, x, cu, gy)
    assert ((torch.cat((y1, y2)) - whole).double().abs() <= 2 * tol).all()


def test_matches_the_dense_scan(mr, cuda_dev):
    B, L, D = 3, 256, 64
    a, x, gy, _, _, cu = _inputs(cuda_dev, [L] * B, D, torch.bfloat16, seed=7)
    dense = mr.rglru_scan(a.view(B, L, D), x.view(B, L, D))
    tol, *_ = O.scan_bounds(a, x, cu, gy)
    assert ((mr.rglru_scan_packed(a, x, cu) - dense.view(-1, D)).double().abs() <= 2 * tol).all()


def test_gradients_against_differences(mr, cuda_dev):
    a, x, gy, h0, gf, cu = _inputs(cuda_dev, [5, 0, 131], 4, torch.float32, seed=8)
    la, lx, lh = (t.clone().requires_grad_() for t in (a, x, h0))

    def loss64(a, x, h0):
        y, _, f = O.scan_forward(a, x, cu, h0)
        return (y * gy.double()).sum() + (f * gf.double()).sum()

    y, final = mr.rglru_scan_packed_with_state(la, lx, cu, h0=lh)
    grads = torch.autograd.grad((y, final), (la, lx, lh), (gy, gf))
    base = [t.double() for t in (a, x, h0)]
    _, _, ta, tx, th = O.scan_bounds(a, x, cu, gy, gf, h0)
    eps = 1e-5
    for n, (row, tol) in enumerate(((3, ta), (100, tx), (1, th))):
        d = [t.clone() for t in base]
        d[n][row, 2] += eps
        up = loss64(*d)
        d[n][row, 2] -= 2 * eps
        diff = float((up - loss64(*d)) / (2 * eps))
        # central differences of a function whose third derivative is of the size of the value itself: eps^2 relative,
        # and 2^-52 |loss| / eps from the subtraction
        slack = 1e-9 * (1 + abs(diff)) + 2.0 ** -52 * 1e4 / eps
        assert abs(float(grads[n][row, 2]) - diff) <= float(tol[row, 2]) + slack


def test_strided_views_unaligned_starts_and_int32_borders(mr, cuda_dev):
    a, x, gy, h0, gf, cu = _inputs(cuda_dev, [90, 45], 66, torch.bfloat16, seed=9)
    want = mr.rglru_scan_packed(a, x, cu)
    wide = torch.stack((a, x), dim=1)  # [T, 2, D]: each half is strided
    assert torch.equal(mr.rglru_scan_packed(wide[:, 0], wide[:, 1], cu.int()), want)
    flat = torch.empty(a.numel() + 1, dtype=a.dtype, device=cuda_dev)
    off = flat[1:].view_as(a)  # contiguous, 2 bytes past the alignment
    off.copy_(a)
    got = mr.rglru_scan_packed(off, x, cu)
    tol, *_ = O.scan_bounds(a, x, cu, gy)
    assert ((got - want).double().abs() <= 2 * tol).all()


def test_empty_batches(mr, cuda_dev):
    z = torch.zeros(0, 8, device=cuda_dev)
    y, final = mr.rglru_scan_packed_with_state(z, z, torch.tensor([0, 0, 0], device=cuda_dev),
                                               h0=torch.ones(2, 8, device=cuda_dev))
    assert y.shape == (0, 8) and (final == 1).all()
    a = torch.rand(5, 8, device=cuda_dev)
    y, final = mr.rglru_scan_packed_with_state(a, a, torch.tensor([0], device=cuda_dev))
    assert (y == 0).all() and final.shape == (0, 8)
    h = torch.ones(2, 8, device=cuda_dev, requires_grad=True)
    za = torch.zeros(0, 8, device=cuda_dev, requires_grad=True)
    y, final = mr.rglru_scan_packed_with_state(za, za, torch.tensor([0, 0, 0], device=cuda_dev), h0=h)
    assert (torch.autograd.grad(final, h, torch.full((2, 8), 3.0, device=cuda_dev))[0] == 3).all()


def test_side_stream_and_graph_replay(mr, cuda_dev):
    a, x, gy, h0, gf, cu = _inputs(cuda_dev, [300, 0, 500, 77], 160, torch.bfloat16, seed=10)

    def step(a, x, h0, cu):
        leaves = [t.detach().requires_grad_() for t in (a, x, h0)]
        y, f = mr.rglru_scan_packed_with_state(leaves[0], leaves[1], cu, h0=leaves[2])
        return [y.detach(), f.detach(), *torch.autograd.grad((y, f), leaves, (gy, gf))]

    static = [t.clone() for t in (a, x, h0)] + [cu.int()]
    side = torch.cuda.Stream(cuda_dev)
    side.wait_stream(torch.cuda.current_stream(cuda_dev))
    with torch.cuda.stream(side):
        first = step(*static)
    torch.cuda.current_stream(cuda_dev).wait_stream(side)
    graphs = [torch.cuda.CUDAGraph() for _ in range(2)]
    outs = []
    for g in graphs:  # two captured steps, replayed one after the other
        with torch.cuda.graph(g):
            outs.append(step(*static))
    want = step(a, x, h0, cu)
    for p, q in zip(first, want):
        assert torch.equal(p, q)
    for s, t in zip(static, (a.flip(0), x.flip(0), h0.flip(0), O.borders([77, 500, 0, 300]).to(cuda_dev))):
        s.copy_(t)
    for _ in range(2):
        for g in graphs:
            g.replay()
    torch.cuda.synchronize()
    want = step(*static)
    for o in outs:
        for p, q in zip(o, want):
            assert torch.equal(p, q)


def test_two_streams_at_once(mr, cuda_dev):
    ins = [_inputs(cuda_dev, [3000, 1000], 256, torch.bfloat16, seed=20 + i) for i in range(2)]
    want = [mr.rglru_scan_packed(i[0], i[1], i[5]) for i in ins]
    streams = [torch.cuda.Stream(cuda_dev) for _ in range(2)]
    torch.cuda.synchronize()
    got = [[], []]
    for _ in range(10):
        for n, s in enumerate(streams):
            with torch.cuda.stream(s):
                got[n].append(mr.rglru_scan_packed(ins[n][0], ins[n][1], ins[n][5]))
    torch.cuda.synchronize()
    assert all(torch.equal(g, want[n]) for n in range(2) for g in got[n])


def test_decode_continues_a_packed_prefill(mr, cuda_dev):
    lens = [33, 200, 1]
    a, x, _, _, _, cu = _inputs(cuda_dev, lens, 64, torch.float32, seed=11)
    _, state = mr.rglru_scan_packed_with_state(a, x, cu)
    an, xn = torch.rand(3, 64, device=cuda_dev), torch.randn(3, 64, device=cuda_dev)
    want = an * state + xn
    y = mr.rglru_step(an, xn, state)
    assert torch.allclose(y, want, rtol=2 ** -22, atol=2 ** -22) and torch.equal(y, state)


def test_offsets_past_32_bits(mr, cuda_dev):
    """More than 2^31 elements. With gates of zero y = x, grad_x = grad_y and grad_a = grad_y h_{t-1}, exactly (but
    for the rounding of grad_a)."""
    T, D = 1 << 20, 2112
    a = torch.zeros(T, D, dtype=torch.bfloat16, device=cuda_dev)
    x = torch.arange(T, device=cuda_dev).remainder(251).to(torch.bfloat16)[:, None].expand(T, D).contiguous()
    gy = torch.full((T, D), 2.0, device=cuda_dev)
    cu = torch.tensor([0, T // 3, T], device=cuda_dev)
    y = mr.rglru_scan_packed(a.requires_grad_(), x.requires_grad_(), cu)
    ga, gx = torch.autograd.grad(y, (a, x), gy)
    for rows in (slice(0, 3), slice(T // 3 - 2, T // 3 + 3), slice(T - 3, T)):
        assert torch.equal(y[rows], x[rows].float()) and (gx[rows] == 2).all()
    assert torch.equal(ga[T - 3:], (2 * x[T - 4:T - 1])) and torch.equal(ga[T // 3 + 1], 2 * x[T // 3])
    assert (ga[T // 3] == 0).all() and (ga[0] == 0).all()
    assert bool((gx == 2).all())
