"""Arguments of window attention that must not reach a kernel."""

import ctypes
import importlib

import pytest
import torch


def test_scales_that_overflow_in_the_kernels_are_refused(mr):
    """The exponent's factor is scale * log2(e): a scale that takes it to infinity would turn scores of zero into NaN."""
    q = torch.randn(1, 4, 2, 64)
    for scale in (2.4e38, 2.9e38, 3.4e38, float("inf")):
        with pytest.raises(ValueError, match="scale"):
            mr.window_attention(q, q, q, 2, scale=scale)
    with pytest.raises(RuntimeError, match="CUDA"):  # past the checks of values
        mr.window_attention(q, q, q, 2, scale=1e38)
    m = importlib.import_module("mlx-recurrence_b200._lib")
    lib, p, n = m.load(), ctypes.c_void_p(256), None
    args = (p, p, p, 64, 64, 64, 64, 64, 64, p, 1, 0, 1, 8, 2, 1, 64, 4, 0)
    assert lib.mr_window_attn_fwd(*args, 2.4e38, p, n, n, n) == m.MR_E_SHAPE
    assert lib.mr_window_step(p, p, p, p, p, p, 1, 1, 2, 2, 2, 64, 5, 4, 2.4e38, p, n) == m.MR_E_SHAPE
