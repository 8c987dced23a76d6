"""Attention under caps far above the scores, where a capped score is the score itself: every form of every operator, and rows of
very different sizes next to one another."""
import math
import os
import sys

import pytest
import torch

sys.path.insert(0, os.path.dirname(os.path.abspath(__file__)))
import attn_cap_oracle as O
import attn_oracle as A
from test_gpu_attn import inputs, run, slopes_of
from test_gpu_attn_tree import Case

gpu = pytest.mark.gpu
F16, BF16 = torch.float16, torch.bfloat16


def loud_rows(q, at, by):
    """Some queries much larger than the others: under a cap between the two, one is bent and its neighbours are not."""
    q = q.clone()
    q[:, at] = (q[:, at].float() * by).to(q.dtype)
    return q


@gpu
@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("cap", [1e3, 1e4, 1e6, 1e8, 1e30])
@pytest.mark.parametrize("t,hq,slopes", [(1, 4, False), (3, 8, True), (8, 8, False), (20, 8, True)])
def test_tree(t, hq, slopes, cap, dtype):
    """Up to 32 rows to a key head and more: 2, 12, 32 and 80."""
    hk, d = 2, 64
    c = Case([600, 77], t, hq, hk, d, 16, dtype, seed=t)
    check_tree(c, 1 / math.sqrt(d), cap, slopes_of(hq) if slopes else None)


@gpu
@pytest.mark.parametrize("t,hq", [(4, 8), (20, 8)])
@pytest.mark.parametrize("cap", [1e4, 1e6])
def test_tree_next_to_a_loud_row(t, hq, cap):
    c = Case([600, 77], t, hq, 2, 64, 16, BF16, seed=t)
    c.q = loud_rows(c.q, 2, cap)
    check_tree(c, 0.125, cap, None)


def check_tree(c, scale, cap, slopes):
    o = c.run(scale, cap, slopes).cpu()
    for i in range(c.b):
        n = int(c.lens[i])
        see = torch.cat([torch.ones(c.t, n, dtype=torch.bool), c.see[i]], 1)
        where = torch.cat([torch.arange(n), n + c.depths[i]])
        dist = (where[n:, None] - where[None, :]).abs().to(torch.float64)
        for h in range(c.hq):
            g = h // (c.hq // c.hk)
            r = O.one_head(*(x.to(torch.float64) for x in (c.q[i, :, h], c.keys[i][:, g], c.values[i][:, g])), see, dist, scale, cap,
                           0.0 if slopes is None else float(slopes[h]), None, c.q.dtype)
            A.assert_close(o[i, :, h], r["o"], r["o_tol"], f"sequence {i} head {h}")


def check(q, k, v, dout, scale, cap, **kw):
    got, ref = run(q, k, v, dout, scale, cap=cap, **kw), O.attention(q, k, v, dout, scale, cap, **kw)
    for name in got:
        A.assert_close(got[name], ref[name], ref[name + "_tol"], name)


@gpu
@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("cap", [1e3, 1e4, 1e6, 1e8, 1e30])
@pytest.mark.parametrize("causal,slopes", [(False, False), (True, True)])
def test_forward_and_backward(causal, slopes, cap, dtype):
    q, k, v, dout = inputs(1, 150, 290, 4, 2, 64, dtype, seed=3)
    check(q, k, v, dout, 0.125, cap, causal=causal, slopes=slopes_of(4) if slopes else None)


@gpu
@pytest.mark.parametrize("lq,lk,h", [(150, 290, 2), (150, 290, 160)])
@pytest.mark.parametrize("cap", [1e4, 1e6])
def test_next_to_a_loud_row(cap, lq, lk, h):
    """In blocks of one and of two tiles of queries."""
    q, k, v, dout = inputs(1, lq, lk, h, 1, 64, BF16, seed=4)
    check(loud_rows(q, 37, cap), k, v, dout, 0.125, cap)
