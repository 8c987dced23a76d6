"""The operators together, as a program uses them: a prompt through attn_fwd, its keys and values into a paged cache, then a step
that verifies drafted tokens: 4-bit projections to q, k, v, the cache, attn_tree, the 4-bit projection back.  Every stage is held
to 64 bits on the inputs that it got; and the step's attention to attn_fwd over the same tokens."""
import math
import os
import sys

import pytest
import torch

sys.path.insert(0, os.path.dirname(os.path.abspath(__file__)))
import attn_oracle as A
from gpu_util import assert_status_ok
from rocwmma_b200 import api

pytestmark = pytest.mark.gpu
F64 = torch.float64


class W4:
    """A packed weight with group scales and zero points, and the same in 64 bits."""

    def __init__(self, m, n, group, dtype, g):
        self.m, self.n, self.group = m, n, group
        self.a = torch.randint(0, 256, (m, n // 2), generator=g, dtype=torch.uint8)
        self.s = ((torch.rand(m, n // group, generator=g) + 0.5) / (4.6 * math.sqrt(n))).to(dtype)
        self.z = torch.randint(6, 10, (m, n // group), generator=g, dtype=torch.uint8)
        q = torch.stack((self.a & 15, self.a >> 4), 2).reshape(m, n).to(F64)
        of = torch.arange(n) // group
        self.exact = (q - self.z.to(F64)[:, of]) * self.s.to(F64)[:, of]
        self.gpu = (self.a.cuda(), self.s.cuda(), self.z.cuda())

    def __call__(self, x, out=None):
        rows = x.shape[0]
        y = torch.empty(rows, self.m, dtype=out or x.dtype, device="cuda")
        a, s, z = self.gpu
        api.gemv_w4(self.m, self.n, rows, a, self.n // 2, s, s.shape[1], self.group, x, self.n, y, self.m, 1.0, 0.0, zeros=z, ld_zeros=s.shape[1])
        xx = x.cpu().to(F64)
        ref, size = xx @ self.exact.T, xx.abs() @ self.exact.abs().T
        tol = torch.finfo(y.dtype).eps / 2 * ref.abs() + (self.n + 8) * 2.0 ** -24 * size + 2.0 ** -25
        assert bool(((y.cpu().to(F64) - ref).abs() <= tol).all())
        return y


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("drafts", [1, 6, 33])
def test_prompt_then_a_verified_step(dtype, drafts):
    g = torch.Generator().manual_seed(drafts)
    hidden, hq, hk, d, page, prompt, cap = 256, 8, 2, 64, 16, 150, 20.0
    wq, wk, wv, wo = (W4(m, n, 64, dtype, g) for m, n in ((hq * d, hidden), (hk * d, hidden), (hk * d, hidden), (hidden, hq * d)))
    scale, slopes = 1 / math.sqrt(d), torch.exp2(-torch.arange(1.0, hq + 1)).cuda()
    split = lambda y, h: y.view(1, -1, h, d)
    x = torch.randn(prompt, hidden, generator=g).to(dtype).cuda()
    q, k, v = split(wq(x), hq), split(wk(x), hk), split(wv(x), hk)
    o, lse = torch.empty_like(q), torch.empty(1, hq, prompt, device="cuda")
    api.attn_fwd(q, k, v, o, lse, scale, causal=True, cap=cap, slopes=slopes)
    ref = A.attention(q.cpu(), k.cpu(), v.cpu(), scale, causal=True, cap=cap, slopes=slopes.cpu())
    A.assert_close(o, ref["o"], ref["o_tol"], "prompt")

    # pages in any order; rows that no token has hold NaN
    need = -(-(prompt + drafts) // page)
    table = torch.randperm(need + 2, generator=g)[:need].to(torch.int32)[None].cuda()
    kc, vc = (torch.full((need + 2, page, hk, d), math.nan, dtype=dtype, device="cuda") for _ in range(2))
    def put(cache, rows, start):
        at = torch.arange(start, start + rows.shape[0], device="cuda")
        cache[table[0, at // page].long(), at % page] = rows
    put(kc, k[0], 0), put(vc, v[0], 0)

    xd = torch.randn(drafts, hidden, generator=g).to(dtype).cuda()
    qd, kd, vd = split(wq(xd), hq), split(wk(xd), hk), split(wv(xd), hk)
    put(kc, kd[0], prompt), put(vc, vd[0], prompt)
    od = torch.empty_like(qd)
    ws = torch.empty(api.attn_tree_workspace_bytes(1, drafts, hq, hk, d, need * page), dtype=torch.uint8, device="cuda")
    lens = torch.tensor([prompt], dtype=torch.int32, device="cuda")
    api.attn_tree(qd, kc, vc, table, lens, od, scale, cap=cap, slopes=slopes, workspace=ws)
    y = wo(od.reshape(drafts, hq * d), out=torch.float32)
    assert y.shape == (drafts, hidden) and bool(torch.isfinite(y).all())
    # a chain of drafts is causal attention of the last queries over all tokens
    ref = A.attention(qd.cpu(), torch.cat([k, kd], 1).cpu(), torch.cat([v, vd], 1).cpu(), scale, causal=True, cap=cap, slopes=slopes.cpu())
    A.assert_close(od, ref["o"], ref["o_tol"], "drafts")
    full = torch.empty_like(qd)
    api.attn_fwd(qd, torch.cat([k, kd], 1), torch.cat([v, vd], 1), full, None, scale, causal=True, cap=cap, slopes=slopes)
    A.assert_close(full, ref["o"], ref["o_tol"], "drafts by attn_fwd")

    # the same step captured once and replayed for other tokens
    graph = torch.cuda.CUDAGraph()
    def step():
        api.attn_tree(qd, kc, vc, table, lens, od, scale, cap=cap, slopes=slopes, workspace=ws)
    torch.cuda.synchronize()
    with torch.cuda.graph(graph):
        step()
    qd.copy_(torch.randn(qd.shape, generator=g).to(dtype))
    graph.replay()
    replayed = od.clone()
    step()
    torch.cuda.synchronize()
    assert torch.equal(replayed, od)
    assert_status_ok()
