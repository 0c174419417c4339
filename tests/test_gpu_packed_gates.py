"""The packed RG-LRU scan where what one chunk hands to the next matters: gates
near one (bits must not depend on how far the other blocks have come) and
gates whose products leave float32's range though the recurrence does not."""

import pytest
import torch

import _packed_oracle as O

pytestmark = pytest.mark.gpu


def _grads(mr, a, x, cu, h0, gy, gf):
    leaves = [t.detach().clone().requires_grad_() for t in (a, x, h0)]
    y, final = mr.rglru_scan_packed_with_state(leaves[0], leaves[1], cu, h0=leaves[2])
    return [y.detach(), final.detach(), *torch.autograd.grad((y, final), leaves, (gy, gf))]


def _check(mr, a, x, cu, h0, gy, gf):
    got = _grads(mr, a, x, cu, h0, gy, gf)
    y, _, final = O.scan_forward(a, x, cu, h0)
    ga, gx, gh = O.scan_backward(a, x, cu, gy, gf, h0)
    ty, tf, ta, tx, th = O.scan_bounds(a, x, cu, gy, gf, h0)
    for name, g, w, t in (("y", got[0], y, ty), ("final", got[1], final, tf), ("grad_a", got[2], ga, ta),
                          ("grad_x", got[3], gx, tx), ("grad_h0", got[4], gh, th)):
        O.check(name, g, w, t)
    return got


# ---- the same bits every time ------------------------------------------------------------------


@pytest.mark.parametrize("dtype,D,lens", [(torch.bfloat16, 128, [40000]), (torch.float32, 33, [9000, 3, 12000]),
                                          (torch.float16, 512, [30000, 20000])])
def test_results_do_not_vary(mr, cuda_dev, dtype, D, lens):
    """Gates of 0.985 to 1: a chunk's product is far from zero, so every chunk depends on those before it. Alone, and
    beside another stream's work, which delays some blocks."""
    g = torch.Generator(device=cuda_dev).manual_seed(41)
    r = dict(device=cuda_dev, generator=g)
    T, S, cu = sum(lens), len(lens), O.borders(lens).to(cuda_dev)
    a = (1 - 0.015 * torch.rand(T, D, **r)).to(dtype)
    x, gy = torch.randn(T, D, **r).to(dtype), torch.randn(T, D, **r)
    h0, gf = torch.randn(S, D, **r), torch.randn(S, D, **r)
    want = _grads(mr, a, x, cu, h0, gy, gf)
    side, busy = torch.cuda.Stream(cuda_dev), torch.randn(2048, 2048, device=cuda_dev)
    torch.cuda.synchronize()
    for n in range(12):
        if n >= 4:
            with torch.cuda.stream(side):
                for _ in range(n):
                    busy @ busy
        for name, p, q in zip(("y", "final", "grad_a", "grad_x", "grad_h0"), _grads(mr, a, x, cu, h0, gy, gf), want):
            assert torch.equal(p, q), (name, n, int((p != q).sum()))
    torch.cuda.synchronize()


def test_gates_near_one_against_float64(mr, cuda_dev):
    g = torch.Generator().manual_seed(42)
    lens, D = [1500, 0, 700], 36
    T = sum(lens)
    a = 1 - 0.01 * torch.rand(T, D, generator=g)
    x, gy, h0, gf = (torch.randn(n, D, generator=g) for n in (T, T, 3, 3))
    _check(mr, *(t.to(cuda_dev) for t in (a, x, O.borders(lens), h0, gy, gf)))


# ---- gates above one ---------------------------------------------------------------------------


@pytest.mark.parametrize("D", [64, 33])  # (33: rows that no 16-byte copy takes)
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("gate", [1.25, 3.0, -40.0, 1e4])
def test_zero_state_under_growing_gates(mr, cuda_dev, gate, dtype, D):
    """x, h0 and gf are zero and gy too but for the first tokens: everything the gates' products would multiply is
    zero, so y is, and what little is not zero has the plain bounds."""
    lens = [700, 130, 0, 900]
    T, S, cu = sum(lens), len(lens), O.borders(lens).to(cuda_dev)
    a = torch.full((T, D), gate, device=cuda_dev).to(dtype)
    x, gy = torch.zeros(T, D, device=cuda_dev).to(dtype), torch.zeros(T, D, device=cuda_dev)
    for lo in (0, 700, 830):
        gy[lo:lo + 5] = torch.arange(1.0, 6.0, device=cuda_dev)[:, None]
    z = torch.zeros(S, D, device=cuda_dev)
    got = _grads(mr, a, x, cu, z, gy, z)
    assert (got[0] == 0).all() and (got[1] == 0).all() and (got[2] == 0).all()
    ga, gx, gh = O.scan_backward(a, x, cu, gy, z, z)
    _, _, _, tx, th = O.scan_bounds(a, x, cu, gy, z, z)
    r = 0.0 if dtype == torch.float32 else O.half_step(dtype)
    O.check("grad_x", got[3], gx, tx + r * (gx.abs() + tx))
    O.check("grad_h0", got[4], gh, th)


@pytest.mark.parametrize("D", [64, 33])
@pytest.mark.parametrize("start", [0, 60, 128, 200])
def test_products_out_of_range_and_back(mr, cuda_dev, start, D):
    """Gates of 2 for 150 tokens, then of 1/2 for 120: their product passes 2^128, the states stay between 2^-100 and
    2^50, the adjoints between 2^-40 and 2^110. Powers of two: exact in every order. A sequence before it and one
    behind it are ordinary."""
    g = torch.Generator().manual_seed(43)
    lens = [start, 270, 90]
    T, cu = sum(lens), O.borders(lens)
    a, x, gy = torch.rand(T, D, generator=g), torch.randn(T, D, generator=g), torch.randn(T, D, generator=g)
    h0, gf = torch.randn(3, D, generator=g), torch.randn(3, D, generator=g)
    mid = slice(start, start + 270)
    a[mid], x[mid], gy[mid] = 0.5, 0.0, 0.0
    a[start:start + 150] = 2.0
    h0[1], gf[1] = 2.0 ** -100, 2.0 ** 80
    # a channel of ordinary gates beside it, and one whose gates are all one
    a[mid, 3], x[mid, 3], gy[mid, 3], h0[1, 3], gf[1, 3] = 0.9, 1.0, 1.0, 1.0, 1.0
    a[mid, 5] = 1.0
    got = _check(mr, *(t.to(cuda_dev) for t in (a, x, cu, h0, gy, gf)))
    assert (got[1][1, 6:] == 2.0 ** -70).all() and (got[4][1, 6:] == 2.0 ** 110).all()
    # adj_t h_t is the same for all t where gy and x are zero (2^80 2^-70), and grad_a_t = adj_t h_t / a_t
    assert (got[2][mid, 6:].cpu() * a[mid, 6:] == 2.0 ** 10).all()


def test_late_input_under_growing_gates(mr, cuda_dev):
    """Zeros for 2800 tokens under gates of 1.05, then input for 200: the gates' product over the zeros, some 1e59,
    multiplies nothing. The other way round for the adjoint."""
    g = torch.Generator().manual_seed(44)
    T, D = 3000, 40
    a = torch.full((T, D), 1.05)
    x, gy = torch.randn(T, D, generator=g), torch.randn(T, D, generator=g)
    x[:2800], gy[200:] = 0.0, 0.0
    z = torch.zeros(1, D)
    _check(mr, *(t.to(cuda_dev) for t in (a, x, O.borders([T]), z, gy, z)))


def test_states_that_overflow_are_infinite(mr, cuda_dev):
    """y itself leaves float32's range: infinite from there on, finite and right before."""
    T, D = 1000, 40
    a, x = torch.full((T, D), 2.0, device=cuda_dev), torch.zeros(T, D, device=cuda_dev)
    x[300] = 1.0  # 2^(t - 300) from here on
    y = mr.rglru_scan_packed(a, x, torch.tensor([0, T], device=cuda_dev))
    want = torch.zeros(T, dtype=torch.float64)
    want[300:] = 2.0 ** torch.arange(700, dtype=torch.float64).clamp(max=1000)
    want = want.float().to(cuda_dev)
    assert torch.equal(y, want[:, None].expand(T, D))


# ---- many borders at one place -----------------------------------------------------------------


@pytest.mark.parametrize("many", [1000, 70000])
def test_many_empty_sequences(mr, cuda_dev, many):
    """Borders padded to a fixed count (a captured graph's): whole runs of empty sequences in front, at a chunk's
    border, inside a chunk and behind the last token change nothing, and each hands on its own state."""
    g = torch.Generator().manual_seed(45)
    T, D, at = 700, 48, [0, 128, 300, 700]
    a, x, gy = torch.rand(T, D, generator=g), torch.randn(T, D, generator=g), torch.randn(T, D, generator=g)
    a, x, gy = a.to(cuda_dev), x.to(cuda_dev), gy.to(cuda_dev)
    cu = torch.tensor([b for b in at for _ in range(many)], device=cuda_dev)
    S = cu.numel() - 1
    h0, gf = torch.randn(S, D, generator=g).to(cuda_dev), torch.randn(S, D, generator=g).to(cuda_dev)
    real = torch.tensor([many - 1, 2 * many - 1, 3 * many - 1], device=cuda_dev)  # the sequences that hold tokens
    got = _grads(mr, a, x, cu, h0, gy, gf)
    want = _grads(mr, a, x, torch.tensor(at, device=cuda_dev), h0[real], gy, gf[real])
    for i in (0, 2, 3):
        assert torch.equal(got[i], want[i])
    for i, own in ((1, h0), (4, gf)):
        own[real] = want[i]
        assert torch.equal(got[i], own)
