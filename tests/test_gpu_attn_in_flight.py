"""Attention calls that overlap on the GPU, each with a workspace of its own: everything is prepared first, then calls go to two
streams without a synchronisation between them, and the bits are compared at the end."""
import os
import sys

import pytest
import torch

sys.path.insert(0, os.path.dirname(os.path.abspath(__file__)))
from gpu_util import assert_status_ok
from rocwmma_b200 import api
from test_gpu_attn import documents, inputs, on_gpu, workspace
from test_gpu_attn_tree import Case

pytestmark = pytest.mark.gpu
F16, BF16 = torch.float16, torch.bfloat16


class Step:
    """attn_fwd and attn_bwd on tensors of their own."""

    def __init__(self, b, lq, lk, hq, hk, d, dtype, seed, scale, **kw):
        q, k, v, dout = (t.cuda() for t in inputs(b, lq, lk, hq, hk, d, dtype, seed=seed))
        self.kw = on_gpu(kw)
        self.out = {"o": torch.empty_like(q), "lse": torch.empty(b, hq, lq, device="cuda"), "dq": torch.empty_like(q),
                    "dk": torch.empty_like(k), "dv": torch.empty_like(v)}
        ws = workspace(b, hq, lq, lk, True)
        o = self.out
        def call():
            api.attn_fwd(q, k, v, o["o"], o["lse"], scale, workspace=ws, **self.kw)
            api.attn_bwd(q, k, v, o["o"], dout, o["lse"], o["dq"], o["dk"], o["dv"], scale, workspace=ws, **self.kw)
        self.call = call

    def results(self):
        return {n: t.clone() for n, t in self.out.items()}

    def clear(self):
        for t in self.out.values():
            t.fill_(float("nan"))


STEPS = {
    "documents": lambda seed: Step(1, 900, 900, 4, 4, 128, BF16, seed, 0.1, causal=True, doc_q=documents("sorted", 900, 1)[None],
                                   doc_kv=documents("sorted", 900, 2)[None]),
    "cap": lambda seed: Step(1, 900, 900, 4, 4, 128, BF16, seed, 0.2, cap=3.0),
    "few key heads": lambda seed: Step(1, 1200, 500, 8, 1, 64, F16, seed, 0.125, causal=True),
    "one block": lambda seed: Step(1, 100, 100, 1, 1, 64, F16, seed, 0.125, causal=True),
}


@pytest.mark.parametrize("one,other", [("documents", "cap"), ("few key heads", "few key heads"), ("few key heads", "one block"),
                                       ("documents", "documents")])
def test_forward_and_backward_on_two_streams(one, other):
    steps = [STEPS[one](43), STEPS[other](44)]
    want = []
    for s in steps:
        s.call()
        torch.cuda.synchronize()
        want.append(s.results())
        s.clear()
    streams = [torch.cuda.Stream() for _ in steps]
    torch.cuda.synchronize()
    for _ in range(8):
        for s, stream in zip(steps, streams):
            with torch.cuda.stream(stream):
                s.call()
    torch.cuda.synchronize()
    assert_status_ok()
    for s, w in zip(steps, want):
        for name, t in s.out.items():
            assert torch.equal(t, w[name]), name


@pytest.mark.parametrize("lens,t,hq,hk,d", [([900, 77], 5, 8, 2, 128), ([9000], 1, 8, 2, 64), ([2000, 2100, 5], 16, 4, 2, 128)])
def test_tree_graphs_on_two_streams(lens, t, hq, hk, d):
    """Up to 32 rows to a key head, tokens split over blocks and joined by a kernel that starts early: two graphs in flight."""
    cases = [Case(lens, t, hq, hk, d, 16, BF16, seed=s) for s in (81, 82)]
    want = [c.check(0.1) for c in cases]
    assert all(c.state["ws"].numel() > 0 for c in cases)
    graphs, streams = [torch.cuda.CUDAGraph() for _ in cases], [torch.cuda.Stream() for _ in cases]
    torch.cuda.synchronize()
    for c, graph in zip(cases, graphs):
        with torch.cuda.graph(graph):
            c.call()
        c.state["o"].zero_()
    torch.cuda.synchronize()
    for _ in range(8):
        for graph, stream in zip(graphs, streams):
            with torch.cuda.stream(stream):
                graph.replay()
    torch.cuda.synchronize()
    assert_status_ok()
    for c, w in zip(cases, want):
        assert torch.equal(c.state["o"].cpu(), w)
