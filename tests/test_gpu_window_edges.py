"""Sliding-window attention at its edges: rows that belong to no sequence beside
values that are not finite, rows whose every score is minus infinity, gradients
of very different sizes in one fp16 batch, mixed types, empty rows, derivatives
that it does not have."""

import importlib

import pytest
import torch
import torch.autograd.forward_ad as fwd_ad

import _packed_oracle as O
from _window_oracle import Window

pytestmark = pytest.mark.gpu

DT = {"bf16": torch.bfloat16, "fp16": torch.float16, "f32": torch.float32}


def _inputs(dev, lens, Hq, Hkv, Dh, dtype, pad=0, seed=0):
    g = torch.Generator().manual_seed(seed)
    T = sum(lens) + pad
    q, gy = (torch.randn(T, Hq, Dh, generator=g) for _ in range(2))
    k, v = (torch.randn(T, Hkv, Dh, generator=g) for _ in range(2))
    return [t.to(dtype).to(dev) for t in (q, k, v, gy)] + [O.borders(lens).to(dev)]


def _step(mr, q, k, v, gy, cu, window, sinks):
    leaves = [t.detach().clone().requires_grad_() for t in (q, k, v)]
    y = mr.window_attention_packed(*leaves, cu, window, sinks=sinks)
    return [y.detach(), *torch.autograd.grad(y, leaves, gy)]


def _check(got, W, names=("y", "gq", "gk", "gv")):
    for n in names:
        O.check(n, got[("y", "gq", "gk", "gv").index(n)], getattr(W, n), getattr(W, "tol_" + n))


# ---- rows outside every sequence ---------------------------------------------------------------


@pytest.mark.parametrize("dtype", sorted(DT))
@pytest.mark.parametrize("bad", [float("nan"), float("inf")])
@pytest.mark.parametrize("what", ["k", "v", "q", "gy"])
def test_rows_outside_are_zero_beside_values_that_are_not_finite(mr, cuda_dev, what, bad, dtype):
    """Padding before and behind the sequences, in the tiles of tokens that hold infinities or NaN."""
    q, k, v, gy, _ = _inputs(cuda_dev, [200], 2, 1, 64, DT[dtype], seed=51)
    cu = torch.tensor([30, 90, 170], device=cuda_dev)
    t = dict(q=q, k=k, v=v, gy=gy)[what]
    t[31], t[169] = bad, bad
    for name, g in zip(("y", "grad_q", "grad_k", "grad_v"), _step(mr, q, k, v, gy, cu, 40, 2)):
        assert (g[:30] == 0).all() and (g[170:] == 0).all(), name


# ---- rows that every visible key gives minus infinity ------------------------------------------


@pytest.mark.parametrize("dtype", sorted(DT))
def test_scores_of_minus_infinity_alone_give_nan(mr, cuda_dev, dtype):
    """softmax of nothing but -inf is NaN: in y, in lse's row of the gradients, and nowhere else."""
    lens, at = [50, 200], 140
    q, k, v, gy, cu = _inputs(cuda_dev, lens, 2, 1, 64, DT[dtype], seed=52)
    W = Window(q, k, v, cu, 1, 0, gy)
    q[at], k[at] = 1.0, -float("inf")
    got = _step(mr, q, k, v, gy, cu, 1, 0)
    rest = torch.arange(250, device=cuda_dev) != at
    for t in got:
        assert torch.isnan(t[at]).all() and torch.isfinite(t[rest]).all()
    O.check("y", got[0][rest], W.y[rest], W.tol_y[rest])
    # a first token that sees only itself, and rows behind it that give it no weight
    q, k, v, gy, cu = _inputs(cuda_dev, lens, 2, 1, 64, DT[dtype], seed=53)
    q.abs_()
    k[50] = -float("inf")
    y = mr.window_attention_packed(q, k, v, cu, 3)
    assert torch.isnan(y[50]).all() and torch.isfinite(y[:50]).all() and torch.isfinite(y[51:]).all()
    # the decode step says the same
    pos = torch.zeros(1, dtype=torch.long, device=cuda_dev)
    ck, cv = (torch.zeros(1, 4, 1, 64, dtype=DT[dtype], device=cuda_dev) for _ in range(2))
    y = mr.window_attention_step(q[50:51], k[50:51], v[50:51], ck, cv, pos)
    assert torch.isnan(y).all()


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
def test_finite_inputs_whose_scores_overflow(mr, cuda_dev, dtype):
    q, k, v, gy, cu = _inputs(cuda_dev, [3], 1, 1, 32, DT[dtype], seed=54)
    q[0], k[0] = 1e25, -1e25
    y = mr.window_attention_packed(q, k, v, cu, 1)
    assert torch.isnan(y[0]).all() and torch.equal(y[1:], v[1:])


# ---- fp16 gradients of very different sizes in one batch ---------------------------------------


@pytest.mark.parametrize("Dh", [64, 128])
@pytest.mark.parametrize("sinks", [0, 4])
def test_fp16_gradients_of_one_sequence_beside_anothers(mr, cuda_dev, sinks, Dh):
    """grad_y of one sequence 10^5 times the other's: each keeps the precision of its own size."""
    lens = [100, 300, 190]
    q, k, v, gy, cu = _inputs(cuda_dev, lens, 2, 1, Dh, torch.float16, seed=55)
    gy *= 0.05
    gy[100:400] = (gy[100:400].double() * 1e5).to(torch.float16)
    got = _step(mr, q, k, v, gy, cu, 120, sinks)
    _check(got, Window(q, k, v, cu, 120, sinks, gy))


@pytest.mark.parametrize("Dh", [32, 96])
def test_fp16_gradients_of_one_head_and_token_beside_others(mr, cuda_dev, Dh):
    q, k, v, gy, cu = _inputs(cuda_dev, [150, 333], 4, 2, Dh, torch.float16, seed=56)
    gy *= 0.02
    gy[:, 2:] = (gy[:, 2:].double() * 1e5).to(torch.float16)  # the second key head's
    gy[300, 0] = (gy[300, 0].double() * 1e6).to(torch.float16)
    got = _step(mr, q, k, v, gy, cu, 100, 3)
    _check(got, Window(q, k, v, cu, 100, 3, gy))


@pytest.mark.parametrize("vscale", [1e-3, 30.0, 2000.0])
def test_fp16_gradients_with_values_of_any_size(mr, cuda_dev, vscale):
    """|dS| itself may pass fp16's range where neither gy, v nor the gradients do."""
    q, k, v, gy, cu = _inputs(cuda_dev, [260, 40], 2, 1, 64, torch.float16, seed=57)
    v = (v * vscale).to(torch.float16)
    q, k = q * 0.05, k * 0.05
    got = _step(mr, q, k, v, gy, cu, 90, 2)
    _check(got, Window(q, k, v, cu, 90, 2, gy))


# ---- layouts ---------------------------------------------------------------------------------------


@pytest.mark.parametrize("dtype", ["bf16", "fp16", "f32"])
@pytest.mark.parametrize("Dh,sinks", [(32, 64), (96, 5), (96, 64), (128, 0), (128, 4), (128, 64)])
def test_head_sizes_and_sinks(mr, cuda_dev, Dh, sinks, dtype):
    q, k, v, gy, cu = _inputs(cuda_dev, [333, 1, 210], 4, 2, Dh, DT[dtype], seed=58)
    _check(_step(mr, q, k, v, gy, cu, 100, sinks), Window(q, k, v, cu, 100, sinks, gy))


# ---- what the backward gets beside y -----------------------------------------------------------


@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
@pytest.mark.parametrize("Dh", [64, 128])
def test_y_low_is_what_rounding_dropped(mr, cuda_dev, Dh, dtype):
    """Through the C entry point: y + y_low is y before it was rounded, in ragged tiles, in padding and in rows that
    are computed again because of a value that they do not see. With q = 0 every probability is one over the count of
    the row's keys, which the kernels hold without rounding (1, and the sum that divides): y's rounding is all there is."""
    lib = importlib.import_module("mlx-recurrence_b200._lib")
    lens, pad, H, window, sinks = [140, 0, 203], 27, 2, 60, 2
    q, k, v, _, cu = _inputs(cuda_dev, lens, H, 1, Dh, DT[dtype], pad=pad, seed=59)
    q.zero_()
    W = Window(q, k, v, cu, window, sinks, r=0.0)
    at, T = 200, sum(lens) + pad
    v = v.clone()
    v[at] = float("nan")
    clean = ~O.visible(T, cu, window, sinks, cuda_dev)[:, at]
    y, low = torch.empty_like(q), torch.empty_like(q)
    lse, cu32 = torch.empty(H, T, device=cuda_dev), cu.int()
    lib.call_on(cuda_dev, "mr_window_attn_fwd", q.data_ptr(), k.data_ptr(), v.data_ptr(), H * Dh, Dh, Dh, Dh, Dh, Dh,
                cu32.data_ptr(), len(lens), 0, lib.DTYPE_CODE[DT[dtype]], T, H, 1, Dh, window, sinks, Dh ** -0.5,
                y.data_ptr(), low.data_ptr(), lse.data_ptr())
    O.check("y", y[clean], W.y[clean], W.tol_y[clean])
    O.check("y + y_low", (y.double() + low.double())[clean], W.y[clean], W.tol_sum[clean])
    assert ((y.double() - W.y).abs() > W.tol_sum)[clean].double().mean() > 0.5  # (y alone is not within that bound)
    assert (y[sum(lens):] == 0).all() and (low[sum(lens):] == 0).all()


# ---- the decode step's own precision -----------------------------------------------------------


@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
@pytest.mark.parametrize("Hq,Hkv,Dh", [(4, 2, 64), (5, 1, 128), (2, 2, 96)])
def test_step_does_not_round_the_probabilities(mr, cuda_dev, Hq, Hkv, Dh, dtype):
    """The probabilities' rounding is carried along: what is left is its square and the rounding of y."""
    B, n, dt = 3, 300, DT[dtype]
    g = torch.Generator().manual_seed(60)
    q, k, v = (torch.randn(B, h, Dh, generator=g).to(dt).to(cuda_dev) for h in (Hq, Hkv, Hkv))
    ck, cv = (torch.randn(B, n, Hkv, Dh, generator=g).to(dt).to(cuda_dev) for _ in range(2))
    pos = torch.tensor([n - 1, 200, 5 * n], device=cuda_dev)
    y = mr.window_attention_step(q, k, v, ck, cv, pos)
    for b, p in enumerate(pos.tolist()):
        m = min(p + 1, n)
        qq = torch.zeros(m, Hq, Dh, dtype=dt, device=cuda_dev)
        qq[-1] = q[b]
        W = Window(qq, ck[b, :m], cv[b, :m], torch.tensor([0, m]), m, 0, r=O.half_step(dt) ** 2)
        O.check(f"y at position {p}", y[b], W.y[-1], W.tol_y[-1])


# ---- mixed types -------------------------------------------------------------------------------


@pytest.mark.parametrize("qd,kd", [("f32", "bf16"), ("bf16", "f32"), ("fp16", "bf16")])
def test_caches_of_mixed_types_serve_the_step(mr, cuda_dev, qd, kd):
    """Caches come in the common dtype of q, k and v, which is what the step asks for."""
    q, k, v, _, cu = _inputs(cuda_dev, [9, 30], 4, 2, 32, torch.float32, seed=61)
    q, k, v = q.to(DT[qd]), k.to(DT[kd]), v.to(DT[kd])
    y, ck, cv = mr.window_attention_packed_with_state(q, k, v, cu, 12, sinks=2)
    assert ck.dtype == cv.dtype == y.dtype == torch.promote_types(DT[qd], DT[kd])
    pos = torch.tensor([9, 30], device=cuda_dev)
    assert mr.window_attention_step(q[:2], k[:2], v[:2], ck, cv, pos, sinks=2).dtype == y.dtype


# ---- empty rows --------------------------------------------------------------------------------


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
def test_dense_batch_of_empty_rows(mr, cuda_dev, dtype):
    z = torch.zeros(3, 0, 2, 64, dtype=DT[dtype], device=cuda_dev)
    y, ck, cv = mr.window_attention_with_state(z, z, z, 7, sinks=2)
    assert y.shape == z.shape and ck.shape == cv.shape == (3, 9, 2, 64) and (ck == 0).all() and (cv == 0).all()
    none = torch.zeros(0, 5, 2, 64, dtype=DT[dtype], device=cuda_dev)
    assert mr.window_attention_with_state(none, none, none, 7)[1].shape == (0, 7, 2, 64)


# ---- derivatives that there are none of --------------------------------------------------------


def test_forward_mode_derivatives_are_refused(mr, cuda_dev):
    """A tangent would be dropped without a word; the other scans refuse it too."""
    q, k, v, gy, cu = _inputs(cuda_dev, [40], 2, 1, 32, torch.float32, seed=62)
    a, x, h0 = torch.rand(40, 8, device=cuda_dev), torch.rand(40, 8, device=cuda_dev), torch.rand(1, 8, device=cuda_dev)

    def dual(t):
        return fwd_ad.make_dual(t, torch.ones_like(t))

    with fwd_ad.dual_level():
        for call in (lambda: mr.window_attention_packed(dual(q), k, v, cu, 8),
                     lambda: mr.window_attention_packed(q, k, dual(v), cu, 8),
                     lambda: mr.window_attention(q[None], dual(k[None]), v[None], 8),
                     lambda: mr.rglru_scan_packed(dual(a), x, cu), lambda: mr.rglru_scan_packed(a, dual(x), cu),
                     lambda: mr.rglru_scan_packed_with_state(a, x, cu, h0=dual(h0)),
                     lambda: mr.rglru_scan(dual(a[None, :32].repeat(1, 1, 4)), x[None, :32].repeat(1, 1, 4))):
            with pytest.raises(NotImplementedError):
                call()
            with torch.no_grad(), pytest.raises(NotImplementedError):
                call()
        assert mr.rglru_scan_packed(a, x, cu).shape == a.shape  # no tangent, no refusal
