"""b200wmma_attn_fwd / b200wmma_attn_bwd against the definition in 64 bits (attn_oracle.py, which also derives the bounds)."""
import ctypes as C
import math
import os
import subprocess
import sys

import pytest
import torch

sys.path.insert(0, os.path.dirname(os.path.abspath(__file__)))
import attn_oracle as A
from gpu_util import assert_status_ok
from rocwmma_b200 import _lib, api

gpu = pytest.mark.gpu
F16, BF16 = torch.float16, torch.bfloat16


def inputs(b, lq, lk, hq, hk, d, dtype, seed=0, loud=2.0):
    g = torch.Generator().manual_seed(seed)
    r = lambda *s: torch.randn(*s, generator=g)
    return ((r(b, lq, hq, d) * loud).to(dtype), r(b, lk, hk, d).to(dtype), r(b, lk, hk, d).to(dtype), r(b, lq, hq, d).to(dtype))


def slopes_of(h):
    return torch.exp2(-8.0 * (torch.arange(h, dtype=torch.float32) + 1) / h)


def workspace(b, hq, lq, lk, backward):
    return torch.full((api.attn_workspace_bytes(b, hq, lq, lk, backward),), 0xEE, dtype=torch.uint8, device="cuda")


def on_gpu(kw):
    return {n: x.cuda() if isinstance(x, torch.Tensor) else x for n, x in kw.items()}


def run(q, k, v, dout, scale, layout=lambda t: t.cuda(), backward=True, **kw):
    """o, lse (and gradients) of the kernels; every output starts as NaN."""
    b, lq, hq, _ = q.shape
    kw = on_gpu(kw)
    ws = workspace(b, hq, lq, k.shape[1], backward)
    gq, gk, gv, gd = (layout(t) for t in (q, k, v, dout))
    o = layout(torch.full_like(q, math.nan))
    lse = torch.full((b, hq, lq), math.nan, device="cuda")
    api.attn_fwd(gq, gk, gv, o, lse, scale, workspace=ws, **kw)
    out = {"o": o, "lse": lse}
    if backward:
        out |= {"dq": layout(torch.full_like(q, math.nan)), "dk": layout(torch.full_like(k, math.nan)), "dv": layout(torch.full_like(v, math.nan))}
        api.attn_bwd(gq, gk, gv, o, gd, lse, out["dq"], out["dk"], out["dv"], scale, workspace=ws, **kw)
    assert_status_ok()
    return out


def check(q, k, v, dout, scale, **kw):
    layout = kw.pop("layout", lambda t: t.cuda())
    got = run(q, k, v, dout, scale, layout=layout, **kw)
    ref = A.attention(q, k, v, scale, dout=dout, **kw)
    for name in got:
        A.assert_close(got[name], ref[name], ref[name + "_tol"], name)
    return got


SIZES = [  # b, lq, lk, hq, hk, d
    (1, 1, 1, 1, 1, 64), (2, 1, 130, 4, 2, 128), (1, 130, 1, 2, 1, 64), (2, 64, 64, 2, 2, 32), (1, 127, 129, 2, 1, 128),
    (1, 128, 128, 1, 1, 128), (1, 129, 127, 1, 1, 64), (1, 257, 300, 2, 2, 80), (2, 300, 257, 3, 1, 8), (1, 385, 640, 4, 2, 120),
    (3, 33, 517, 2, 2, 72)]


@gpu
@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize("b,lq,lk,hq,hk,d", SIZES)
def test_sizes(b, lq, lk, hq, hk, d, causal, dtype):
    q, k, v, dout = inputs(b, lq, lk, hq, hk, d, dtype, seed=lq + lk)
    check(q, k, v, dout, 1 / math.sqrt(d), causal=causal)


@gpu
@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("lq,lk,d", [(150, 290, 64), (290, 290, 128)])
@pytest.mark.parametrize("causal", [False, True])
def test_cap_and_bias(lq, lk, d, causal, dtype):
    q, k, v, dout = inputs(2, lq, lk, 4, 2, d, dtype, seed=3, loud=6.0)
    check(q, k, v, dout, 1 / math.sqrt(d), causal=causal, cap=5.0)
    check(q, k, v, dout, 1 / math.sqrt(d), causal=causal, slopes=slopes_of(4))
    check(q, k, v, dout, -0.05, causal=causal, cap=30.0, slopes=slopes_of(4))


@gpu
@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("prefix", [(0, 1), (-5, 200), (128, 129), (1000, 77)])
def test_prefix(prefix, dtype):
    q, k, v, dout = inputs(2, 270, 290, 2, 1, 64, dtype, seed=5)
    p = torch.tensor(prefix, dtype=torch.int32)
    check(q, k, v, dout, 0.125, causal=True, prefix=p)
    check(q, k, v, dout, 0.125, causal=True, prefix=p, slopes=slopes_of(2), cap=20.0)
    check(q, k, v, dout, 0.125, causal=False, prefix=p)  # everything is visible already


def documents(kind, n, seed):
    g = torch.Generator().manual_seed(seed)
    if kind == "sorted":
        return torch.sort(torch.randint(0, 5, (n,), generator=g)).values.to(torch.int32)
    if kind == "mixed":  # any order, padding in between
        return torch.randint(-1, 3, (n,), generator=g).to(torch.int32)
    if kind == "padded":  # documents and a padded end, large ids
        d = torch.sort(torch.randint(0, 3, (n,), generator=g)).values.to(torch.int32) + 2000000000
        d[n - n // 3:] = -7
        return d
    if kind == "one":
        return torch.zeros(n, dtype=torch.int32)
    return torch.full((n,), -1, dtype=torch.int32)  # "none"


@gpu
@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize("kind", ["sorted", "mixed", "padded", "one", "none"])
@pytest.mark.parametrize("n,d", [(400, 128), (190, 40)])
def test_documents(kind, n, d, causal, dtype):
    q, k, v, dout = inputs(2, n, n, 2, 1, d, dtype, seed=7)
    docs = torch.stack([documents(kind, n, 1), documents(kind, n, 2)])
    check(q, k, v, dout, 1 / math.sqrt(d), causal=causal, doc_q=docs, doc_kv=docs)


@gpu
@pytest.mark.parametrize("dtype", [F16, BF16])
def test_documents_of_other_queries(dtype):
    """Queries and keys with documents of their own; one query document has no key at all; prefix, cap and bias on top."""
    q, k, v, dout = inputs(2, 200, 333, 2, 2, 64, dtype, seed=9)
    dq = torch.stack([torch.arange(200) // 30, torch.arange(200) // 90 + 3]).to(torch.int32)
    dk = torch.stack([torch.arange(333) // 60, torch.arange(333) % 5]).to(torch.int32)
    check(q, k, v, dout, 0.125, doc_q=dq, doc_kv=dk)
    check(q, k, v, dout, 0.125, causal=True, prefix=torch.tensor([40, 140], dtype=torch.int32), doc_q=dq, doc_kv=dk, cap=15.0, slopes=slopes_of(2))


@gpu
@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("d", [64, 128])
def test_padding_may_hold_anything(d, dtype):
    n = 300
    q, k, v, dout = inputs(1, n, n, 2, 1, d, dtype, seed=11)
    docs = documents("padded", n, 4)[None].clone()
    docs[0, 17], docs[0, 130:133] = -1, -2
    clean = check(q, k, v, dout, 0.1, causal=True, doc_q=docs, doc_kv=docs)
    bad = (docs[0] < 0).nonzero().flatten()
    for t, fill in ((q, math.nan), (k, math.inf), (v, math.nan), (dout, -math.inf)):
        t[:, bad] = fill
    dirty = run(q, k, v, dout, 0.1, causal=True, doc_q=docs, doc_kv=docs)
    for name in clean:
        assert torch.equal(clean[name], dirty[name]), name


def strided(order, gap=0):
    """Puts a [batch, tokens, heads, dim] tensor into memory in another order of its axes, with unused elements between rows."""
    def put(t):
        shape = [t.shape[i] for i in order] + [t.shape[3] + gap]
        back = [order.index(i) for i in range(3)] + [3]
        out = torch.full(shape, math.nan, dtype=t.dtype, device="cuda").permute(back)[..., :t.shape[3]]
        out.copy_(t)
        return out
    return put


@gpu
@pytest.mark.parametrize("order,gap", [((0, 2, 1), 0), ((1, 0, 2), 8), ((2, 1, 0), 16), ((2, 0, 1), 0)])
def test_strides(order, gap):
    q, k, v, dout = inputs(2, 140, 205, 4, 2, 72, F16, seed=13)
    a = check(q, k, v, dout, 0.1, causal=True)
    b = run(q, k, v, dout, 0.1, causal=True, layout=strided(order, gap))
    for name in a:
        assert torch.equal(a[name], b[name]), name


@gpu
def test_shared_rows_of_inputs_and_untouched_surroundings():
    """One packed tensor holds q, k and v; the output is a slice of a larger one."""
    b, n, h, d = 2, 150, 3, 64
    g = torch.Generator().manual_seed(1)
    packed = torch.randn(b, n, 3 * h, d, generator=g).to(BF16).cuda()
    q, k, v = packed[:, :, :h], packed[:, :, h:2 * h], packed[:, :, 2 * h:]
    big = torch.full((b, n + 2, h + 1, d), 7.0, dtype=BF16, device="cuda")
    lse = torch.empty(b, h, n, device="cuda")
    api.attn_fwd(q, k, v, big[:, 1:n + 1, :h], lse, 0.125, causal=True)
    ref = A.attention(q.cpu(), k.cpu(), v.cpu(), 0.125, causal=True)
    A.assert_close(big[:, 1:n + 1, :h], ref["o"], ref["o_tol"], "o")
    assert bool((big[:, 0] == 7).all()) and bool((big[:, n + 1] == 7).all()) and bool((big[:, :, h] == 7).all())
    api.attn_fwd(q, k, v, big[:, 1:n + 1, :h], None, 0.125, causal=True)  # without lse


@gpu
@pytest.mark.parametrize("dtype", [F16, BF16])
def test_growing_and_large_scores(dtype):
    """Scores that grow along the keys, so that the running maximum moves at every step, and very large ones."""
    q, k, v, dout = inputs(1, 260, 700, 1, 1, 64, dtype, seed=17, loud=0.5)
    k = (k.float() * (torch.arange(700) / 100.0 + 0.1)[None, :, None, None]).to(dtype)
    check(q, k, v, dout, 0.5)
    q, k, v, dout = inputs(1, 140, 300, 1, 1, 64, dtype, seed=18, loud=30.0)
    check(q, k, v, dout, 1.0, causal=True)
    check(torch.zeros_like(q), k, v, dout, 1.0)  # all scores equal
    falling = torch.tensor([50.0])
    check(q, k, v, dout, 0.01, slopes=falling)


@gpu
def test_steep_slopes_far_away():
    """Only far keys are visible: every score is far below zero, the weights still add up to one."""
    q, k, v, dout = inputs(1, 8, 900, 1, 1, 64, F16, seed=19)
    dk = (torch.arange(900) >= 100).to(torch.int32)[None]
    check(q, k, v, dout, 0.125, slopes=torch.tensor([2.0]), doc_q=torch.zeros(1, 8, dtype=torch.int32), doc_kv=dk)


@gpu
@pytest.mark.parametrize("dtype", [F16, BF16])
def test_a_longer_sequence(dtype):
    q, k, v, dout = inputs(1, 1500, 1500, 2, 1, 128, dtype, seed=23)
    docs = (torch.arange(1500) // 611).to(torch.int32)[None]
    check(q, k, v, dout, 1 / math.sqrt(128), causal=True, doc_q=docs, doc_kv=docs)
    check(q, k, v, dout, 1 / math.sqrt(128), causal=True)


@gpu
@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("lq,lk,d", [(300, 300, 128), (257, 390, 64), (384, 150, 80)])
def test_more_blocks_than_run_at_once(lq, lk, d, dtype):
    """Grids large enough that a block takes two tiles of queries, with each kind of mask and score."""
    q, k, v, dout = inputs(4, lq, lk, 20, 5, d, dtype, seed=29, loud=3.0)
    docs = lambda n: torch.stack([documents(kind, n, 1) for kind in ("sorted", "mixed", "padded", "none")])
    check(q, k, v, dout, 1 / math.sqrt(d), causal=True)
    check(q, k, v, dout, 1 / math.sqrt(d), causal=True, cap=20.0, prefix=torch.tensor([0, 30, 140, 600], dtype=torch.int32))
    check(q, k, v, dout, 1 / math.sqrt(d), slopes=slopes_of(20))
    check(q, k, v, dout, 1 / math.sqrt(d), causal=lq == lk, doc_q=docs(lq), doc_kv=docs(lk) if lq != lk else docs(lq))


@gpu
@pytest.mark.parametrize("batch", [1, 40])
@pytest.mark.parametrize("how", ["rising", "falling", "some"])
@pytest.mark.parametrize("cap", [0.0, 15.0])
def test_scores_of_very_different_sizes(cap, how, batch):
    """Key tiles that outgrow one another by more than the maximum may lag behind, in either order and now and then; under a cap
    some of them bent hard and others hardly."""
    lq, lk = 200, 1100
    q, k, v, dout = inputs(batch, lq, lk, 2, 2, 64, BF16, seed=31)
    at = torch.arange(lk) // 128
    size = {"rising": 0.02 * 3.0 ** at, "falling": 0.02 * 3.0 ** (8 - at), "some": torch.where(at % 3 == 1, 30.0, 0.1)}[how]
    k = (k.float() * size[None, :, None, None]).to(BF16)
    check(q, k, v, dout, 0.125, cap=cap)


@gpu
@pytest.mark.parametrize("lq,lk", [(3, 66000), (66000, 3), (260, 66100)])
@pytest.mark.parametrize("docs", [False, True])
def test_more_tiles_than_one_list_holds(lq, lk, docs):
    """Key (and query) tiles are listed 512 at a time: 66000 tokens are more."""
    q, k, v, dout = inputs(1, lq, lk, 1, 1, 64, BF16, seed=37)
    kw = {}
    if docs:
        kw = {"doc_q": (torch.arange(lq) * 3 // lq).to(torch.int32)[None], "doc_kv": (torch.arange(lk) * 3 // lk).to(torch.int32)[None]}
    check(q, k, v, dout, 0.125, **kw)


@gpu
@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("b,lq,lk,hq,hk,d", [(1, 1500, 900, 8, 1, 128), (2, 700, 700, 12, 2, 72), (1, 40, 130, 16, 1, 64), (1, 5000, 100, 1, 1, 128)])
def test_few_key_heads(b, lq, lk, hq, hk, d, dtype):
    """Few blocks for dk and dv, whose steps are split; bits do not depend on the call."""
    q, k, v, dout = inputs(b, lq, lk, hq, hk, d, dtype, seed=53)
    got = check(q, k, v, dout, 1 / math.sqrt(d), causal=True)
    again = run(q, k, v, dout, 1 / math.sqrt(d), causal=True)
    for name in got:
        assert torch.equal(got[name], again[name]), name
    docs = lambda n: torch.stack([documents(("sorted", "mixed")[i], n, 3) for i in range(b)])
    check(q, k, v, dout, 1 / math.sqrt(d), cap=9.0, slopes=slopes_of(hq), doc_q=docs(lq), doc_kv=docs(lk))


@gpu
@pytest.mark.parametrize("causal", [False, True])
def test_long_keys_and_many_blocks(causal):
    """More key tiles than one list holds, for blocks of two tiles of queries; three of the heads are compared."""
    lq, lk, hq, d = 129, 66000, 75, 64
    q, k, v, dout = inputs(1, lq, lk, hq, 1, d, BF16, seed=47)
    got = run(q, k, v, dout, 0.125, causal=causal, backward=False)
    few = [0, 37, 74]
    ref = A.attention(q[:, :, few], k, v, 0.125, causal=causal)
    A.assert_close(got["o"][:, :, few], ref["o"], ref["o_tol"], "o")
    A.assert_close(got["lse"][:, few], ref["lse"], ref["lse_tol"], "lse")


@gpu
def test_rows_far_apart():
    """Offsets that pass 2^31 elements."""
    n, h, d, stride = 300, 2, 64, 8 << 20
    big = torch.zeros(n * stride, dtype=BF16, device="cuda")
    g = torch.Generator().manual_seed(41)
    q, k, v, dout = inputs(1, n, n, h, h, d, BF16, seed=41)
    at = iter(range(0, 8 * h * d, h * d))
    def far(t):
        x = big.as_strided((1, n, h, d), (n * stride, stride, d, 1), next(at))
        x.copy_(t)
        return x
    assert n * stride > 1 << 31
    check(q, k, v, dout, 0.125, causal=True, layout=far)


@gpu
def test_two_streams_at_once():
    """Two calls in flight, each with a workspace of its own."""
    q, k, v, dout = inputs(1, 900, 900, 4, 4, 128, BF16, seed=43)
    docs = documents("sorted", 900, 1)[None]
    alone = run(q, k, v, dout, 0.1, causal=True, doc_q=docs, doc_kv=docs)
    other = run(q, k, v, dout, 0.2, cap=3.0)
    streams = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    both = []
    for _ in range(3):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                both.append(run(q, k, v, dout, 0.2, cap=3.0) if i else run(q, k, v, dout, 0.1, causal=True, doc_q=docs, doc_kv=docs))
    torch.cuda.synchronize()
    for i, got in enumerate(both):
        for name in got:
            assert torch.equal(got[name], (other if i % 2 else alone)[name]), name


@gpu
def test_first_call_of_a_process_may_be_captured():
    code = """
import torch
from rocwmma_b200 import api
q = torch.randn(1, 200, 2, 64, device="cuda").half()
o, o2, lse = torch.empty_like(q), torch.empty_like(q), torch.empty(1, 2, 200, device="cuda")
dq, dk, dv = (torch.empty_like(q) for _ in range(3))
ws = torch.empty(api.attn_workspace_bytes(1, 2, 200, 200, True), dtype=torch.uint8, device="cuda")
g = torch.cuda.CUDAGraph()
with torch.cuda.graph(g):
    api.attn_fwd(q, q, q, o, lse, 0.125, causal=True)
    api.attn_bwd(q, q, q, o, q, lse, dq, dk, dv, 0.125, causal=True, workspace=ws)
g.replay()
api.attn_fwd(q, q, q, o2, lse, 0.125, causal=True)
torch.cuda.synchronize()
assert torch.equal(o, o2) and bool(torch.isfinite(dq).all()) and api.device_status()[0] == 0
print("captured")
"""
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    done = subprocess.run([sys.executable, "-c", code], cwd=root, capture_output=True, text=True, timeout=300)
    assert done.returncode == 0 and "captured" in done.stdout, done.stderr[-2000:]


@gpu
def test_tensors_of_another_device_are_refused():
    if torch.cuda.device_count() < 2:
        pytest.skip("needs two GPUs")
    t = torch.zeros(1, 4, 2, 64, dtype=F16, device="cuda:1")
    with pytest.raises(ValueError):
        api.attn_fwd(t, t, t, t.clone(), None, 1.0)


@gpu
def test_repeat_stream_and_graph():
    """The same bits again, on another stream, and from a captured graph with new inputs."""
    q, k, v, dout = inputs(2, 300, 300, 4, 2, 64, BF16, seed=29)
    docs = torch.stack([documents("sorted", 300, 1), documents("padded", 300, 2)])
    a = run(q, k, v, dout, 0.125, causal=True, doc_q=docs, doc_kv=docs)
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        b = run(q, k, v, dout, 0.125, causal=True, doc_q=docs, doc_kv=docs)
    side.synchronize()
    for name in a:
        assert torch.equal(a[name], b[name]), name
    gq, gk, gv, gd, gdoc = (t.cuda() for t in (q, k, v, dout, docs))
    ws, lse = workspace(2, 4, 300, 300, True), torch.empty(2, 4, 300, device="cuda")
    o, dq, dk, dv = torch.empty_like(gq), torch.empty_like(gq), torch.empty_like(gk), torch.empty_like(gv)
    graph = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph):
        api.attn_fwd(gq, gk, gv, o, lse, 0.125, causal=True, doc_q=gdoc, doc_kv=gdoc, workspace=ws)
        api.attn_bwd(gq, gk, gv, o, gd, lse, dq, dk, dv, 0.125, causal=True, doc_q=gdoc, doc_kv=gdoc, workspace=ws)
    for seed in (30, 31):
        new = inputs(2, 300, 300, 4, 2, 64, BF16, seed=seed)
        ids = torch.stack([documents("mixed", 300, seed), documents("sorted", 300, seed)])
        for t, x in zip((gq, gk, gv, gd, gdoc), (*new, ids)):
            t.copy_(x)
        graph.replay()
        torch.cuda.synchronize()
        c = run(*new, 0.125, causal=True, doc_q=ids, doc_kv=ids)
        for name, t in (("o", o), ("lse", lse), ("dq", dq), ("dk", dk), ("dv", dv)):
            assert torch.equal(t, c[name]), name


def test_definition_against_differences():
    """The gradients that the kernels are held to, against central differences of the definition (64 bits, no GPU)."""
    g = torch.Generator().manual_seed(2)
    lq, lk, d = 7, 9, 8
    q, k, v, dout = (torch.randn(n, d, generator=g, dtype=torch.float64) for n in (lq, lk, lk, lq))
    docs_q, docs_k = torch.tensor([0, 0, 1, 1, 1, -1, 2]), torch.tensor([0, 0, 0, 1, 1, 1, 1, -1, 1])
    see = A.visible(lq, lk, True, 3, docs_q, docs_k)
    assert not see[5].any() and not see[6].any()
    how = dict(see=see, dist=A.distance(lq, lk), scale=0.4, cap=2.0, slope=0.3)
    ref = A.one_head(q, k, v, dout=dout, **how)
    h = 1e-5
    for name, x in (("dq", q), ("dk", k), ("dv", v)):
        num = torch.zeros_like(x)
        for at in range(x.numel()):
            for sign in (1, -1):
                y = x.clone()
                y.view(-1)[at] += sign * h
                o = A.one_head(*[y if t is x else t for t in (q, k, v)], **how)["o"]
                num.view(-1)[at] += sign * (o * dout).sum() / (2 * h)
        assert (num - ref[name]).abs().max() < 1e-8, name
    assert (ref["o"][5:] == 0).all() and (ref["dq"][5:] == 0).all() and (ref["dk"][7] == 0).all()


# ---- refusals (no GPU) --------------------------------------------------------------------------------------------
def args(**kw):
    a = _lib.AttnArgs()
    a.batch, a.heads_q, a.heads_kv, a.len_q, a.len_kv, a.head_dim, a.scale = 2, 4, 2, 16, 24, 64, 0.125
    for name in ("q", "o", "dout", "dq"):
        s = getattr(a, name)
        s.batch, s.token, s.head = 16 * 4 * 64, 4 * 64, 64
    for name in ("k", "v", "dk", "dv"):
        s = getattr(a, name)
        s.batch, s.token, s.head = 24 * 2 * 64, 2 * 64, 64
    for name, x in kw.items():
        at, last = a, name
        if "_" in name and name.split("_")[0] in ("q", "k", "v", "o", "dout", "dq", "dk", "dv"):
            first, last = name.split("_")
            at = getattr(a, first)
        setattr(at, last, x)
    return a


@pytest.mark.parametrize("how,code", [
    (dict(batch=0), 1), (dict(heads_q=0), 1), (dict(heads_kv=0), 1), (dict(len_q=0), 1), (dict(len_kv=0), 1), (dict(head_dim=0), 1),
    (dict(heads_q=3), 1), (dict(head_dim=60), 2), (dict(head_dim=136), 2), (dict(data_type=1), 1), (dict(cap=-1.0), 1),
    (dict(cap=math.inf), 1), (dict(cap=math.nan), 1), (dict(scale=math.nan), 1), (dict(scale=math.inf), 1), (dict(doc_q=16), 1),
    (dict(doc_kv=16), 1), (dict(len_q=1 << 30), 2), (dict(batch=1 << 24), 2), (dict(q_token=4 * 64 + 4), 3), (dict(k_batch=0), 1), (dict(v_head=-64), 1),
    (dict(o_head=32), 1), (dict(o_token=64), 1), (dict(q_batch=1 << 38), 2)])
@pytest.mark.parametrize("backward", [False, True])
def test_refusals(how, code, backward):
    L = _lib.lib()
    a = args(**how)
    if backward:
        rc = L.b200wmma_attn_bwd(C.byref(a), 16, 16, 16, 16, 16, 16, 16, 16, 16, 16, 1 << 30, None)
        if "o_head" in how or "o_token" in how:
            return  # o is only read there
    else:
        rc = L.b200wmma_attn_fwd(C.byref(a), 16, 16, 16, 16, 16, 16, 1 << 30, None)
    assert rc == code, L.b200wmma_last_error_string()
    assert (b"attn_bwd" if backward else b"attn_fwd") in L.b200wmma_last_error_string()


@pytest.mark.parametrize("at,bad,code", [(i, None, 1) for i in range(9)] + [(i, 24, 3) for i in (0, 1, 2, 3, 4, 6, 7, 8)])
def test_refused_pointers(at, bad, code):
    L = _lib.lib()
    ptr = [16] * 9  # q, k, v, o, dout, lse, dq, dk, dv
    ptr[at] = bad
    assert L.b200wmma_attn_bwd(C.byref(args()), *ptr, 16, 1 << 30, None) == code
    if at < 4:
        assert L.b200wmma_attn_fwd(C.byref(args()), *ptr[:4], 16, 16, 1 << 30, None) == code


def test_refused_workspaces_and_gradients():
    L = _lib.lib()
    a = args()
    need = L.b200wmma_attn_workspace_bytes(2, 4, 16, 24, 1)
    assert need > 0
    bwd = lambda a, ws, size: L.b200wmma_attn_bwd(C.byref(a), 16, 16, 16, 16, 16, 16, 16, 16, 16, ws, size, None)
    assert bwd(a, None, need) == 1 and bwd(a, 16, need - 1) == 1 and bwd(a, 24, need) == 3
    assert L.b200wmma_attn_fwd(None, 16, 16, 16, 16, 16, 16, 1 << 30, None) == 1
    for how in (dict(dq_token=64), dict(dk_batch=8), dict(dv_head=0)):
        assert bwd(args(**how), 16, need) == 1, how


def test_wrapper_refuses_wrong_tensors():
    t = torch.zeros(1, 4, 2, 64, dtype=F16)
    with pytest.raises(TypeError):
        api.attn_fwd(t, t, t, t, None, 1.0)  # not on a GPU
    with pytest.raises(TypeError):
        api.attn_fwd(t.float(), t, t, t, None, 1.0)


@gpu
def test_wrapper_refuses_wrong_shapes():
    t = torch.zeros(1, 4, 2, 64, dtype=F16, device="cuda")
    for bad in (t[0], torch.zeros(1, 4, 2, 128, dtype=F16, device="cuda")[..., ::2], t.to(BF16)):
        with pytest.raises((TypeError, ValueError)):
            api.attn_fwd(t, bad, t, t.clone(), None, 1.0)
    with pytest.raises(ValueError):
        api.attn_fwd(t, t, t, t.clone(), None, 1.0, slopes=torch.zeros(3, device="cuda"))
    with pytest.raises(ValueError):
        api.attn_fwd(t, t, t, t.clone(), torch.zeros(1, 2, 5, device="cuda"), 1.0)
    with pytest.raises(ValueError):
        api.attn_fwd(t, t, t, t.clone(), None, 1.0, prefix=torch.zeros(2, dtype=torch.int32, device="cuda"))
