"""Gradients of attention under caps far below 1: scores of the order of the cap, and scores that it holds at its limits, where
the derivative 1 - tanh^2 is next to 0."""
import os
import sys

import pytest
import torch

sys.path.insert(0, os.path.dirname(os.path.abspath(__file__)))
from test_gpu_attn import inputs, slopes_of
from test_gpu_attn_large_caps import check, loud_rows

gpu = pytest.mark.gpu
F16, BF16 = torch.float16, torch.bfloat16


@gpu
@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("causal,slopes", [(False, False), (True, True)])
@pytest.mark.parametrize("cap,scale", [
    (1.0, 0.125), (1e-2, 0.125), (1e-3, 0.125), (1e-5, 0.125), (1e-8, 0.125), (1e-30, 0.125),  # held at the limits
    (1e-2, 1e-3), (1e-3, 1e-4), (1e-3, -1e-4), (1e-5, 1e-6), (1e-5, 2e-7)])  # of the order of the cap, and below it
def test_gradients(cap, scale, causal, slopes, dtype):
    q, k, v, dout = inputs(1, 150, 290, 4, 2, 64, dtype, seed=5)
    check(q, k, v, dout, scale, cap, causal=causal, slopes=slopes_of(4) if slopes else None)


@gpu
@pytest.mark.parametrize("d", [40, 128])
def test_bent_and_straight_rows_together(d):
    q, k, v, dout = inputs(2, 140, 260, 2, 2, d, BF16, seed=6)
    check(loud_rows(q, slice(30, 90), 1000.0), k, v, dout, 1e-4, 0.01, causal=True)
