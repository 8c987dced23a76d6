"""b200wmma_attn_tree against the definition in 64 bits (attn_oracle.py derives the bounds): pages in any order, trees of
drafted tokens, ragged batches, broken page tables."""
import ctypes as C
import math
import os
import sys

import pytest
import torch

sys.path.insert(0, os.path.dirname(os.path.abspath(__file__)))
import attn_oracle as A
from gpu_util import assert_status_ok
from rocwmma_b200 import _lib, api

gpu = pytest.mark.gpu
F16, BF16 = torch.float16, torch.bfloat16
F64 = torch.float64


def random_tree(t, seed):
    """(words, depths, truth matrix) of a tree of t drafted tokens."""
    g = torch.Generator().manual_seed(seed)
    see, depth = torch.zeros(t, t, dtype=torch.bool), torch.zeros(t, dtype=torch.int32)
    for i in range(t):
        see[i, i] = True
        p = int(torch.randint(-1, i, (1,), generator=g)) if i else -1
        if p >= 0:
            see[i] |= see[p]
            depth[i] = depth[p] + 1
    return (see.to(torch.int64) << torch.arange(t)).sum(1), depth, see


class Case:
    def __init__(self, lens, t, hq, hk, d, page, dtype, seed=0, spare=3, loud=2.0, kind="tree", n_drafts=None):
        g = torch.Generator().manual_seed(seed)
        r = lambda *s: torch.randn(*s, generator=g)
        b = len(lens)
        self.b, self.t, self.hq, self.hk, self.d, self.page, self.kind, self.n_drafts = b, t, hq, hk, d, page, kind, n_drafts
        need = [max(1, -(-(max(n, 0) + t) // page)) for n in lens]
        width = max(need) + 1
        pages = sum(need) + spare
        order = torch.randperm(pages, generator=g)
        self.table = torch.full((b, width), 1 << 30, dtype=torch.int32)  # places that no token needs hold nonsense
        self.k = torch.full((pages, page, hk, d), math.nan).to(dtype)
        self.v = torch.full((pages, page, hk, d), math.nan).to(dtype)
        at = 0
        self.keys, self.values = [], []
        for i, n in enumerate(lens):
            mine = order[at:at + need[i]]
            at += need[i]
            self.table[i, :need[i]] = mine.to(torch.int32)
            live = max(n, 0) + (t if n_drafts is None else max(0, min(n_drafts[i], t)))
            kk, vv = r(live, hk, d).to(dtype), r(live, hk, d).to(dtype)
            self.keys.append(kk), self.values.append(vv)
            if live:
                p, row = mine[torch.arange(live) // page], torch.arange(live) % page
                self.k[p, row], self.v[p, row] = kk, vv
        self.lens = torch.tensor(lens, dtype=torch.int32)
        self.q = (r(b, t, hq, d) * loud).to(dtype)
        trees = [random_tree(t, seed * 100 + i) for i in range(b)]
        self.words, self.depths = torch.stack([x[0] for x in trees]), torch.stack([x[1] for x in trees])
        self.see = [x[2] for x in trees]
        if kind == "chain":
            self.see, self.depths = [torch.tril(torch.ones(t, t, dtype=torch.bool))] * b, torch.arange(t, dtype=torch.int32).repeat(b, 1)

    def run(self, scale, cap=0.0, slopes=None, change=lambda s: None, layout=lambda x: x.cuda()):
        s = {"q": layout(self.q), "k": layout(self.k), "v": layout(self.v), "table": self.table.cuda(), "lens": self.lens.cuda(),
             "o": layout(torch.full_like(self.q, 77.0))}
        s["tree"] = None if self.kind == "chain" else self.words.cuda()
        s["depths"] = None if self.kind == "chain" else self.depths.cuda()
        s["n_drafts"] = None if self.n_drafts is None else torch.tensor(self.n_drafts, dtype=torch.int32, device="cuda")
        change(s)
        need = api.attn_tree_workspace_bytes(self.b, self.t, self.hq, self.hk, self.d, self.table.shape[1] * self.page)
        s["ws"] = torch.full((need,), 0xEE, dtype=torch.uint8, device="cuda")
        self.call = lambda: api.attn_tree(s["q"], s["k"], s["v"], s["table"], s["lens"], s["o"], scale, tree=s["tree"], depths=s["depths"],
                                          n_drafts=s["n_drafts"], cap=cap, slopes=None if slopes is None else slopes.cuda(), workspace=s["ws"])
        self.call()
        assert_status_ok()
        self.state = s
        return s["o"]

    def check(self, scale, cap=0.0, slopes=None, hide=None, **kw):
        """hide(b, token) -> True where a token's page is broken."""
        o = self.run(scale, cap, slopes, **kw).cpu()
        eps = torch.finfo(self.q.dtype).eps / 2
        for i in range(self.b):
            n = max(int(self.lens[i]), 0)
            live = self.keys[i].shape[0] - n
            see = torch.cat([torch.ones(live, n, dtype=torch.bool), self.see[i][:live, :live]], 1)
            if hide is not None:
                see = see & ~torch.tensor([hide(i, p) for p in range(n + live)], dtype=torch.bool)[None]
            where = torch.cat([torch.arange(n), n + self.depths[i, :live]])
            dist = (where[n:, None] - where[None, :]).abs().to(F64)
            for h in range(self.hq if live else 0):
                g = h // (self.hq // self.hk)
                r = A.one_head(self.q[i, :live, h].to(F64), self.keys[i][:, g].to(F64), self.values[i][:, g].to(F64), see, dist, scale, cap,
                               0.0 if slopes is None else float(slopes[h]), None, eps)
                A.assert_close(o[i, :live, h], r["o"], r["o_tol"], f"sequence {i} head {h}")
            assert bool((o[i, live:] == 77.0).all())  # rows of tokens that do not exist stay as they were
        return o


def slopes_of(h):
    return torch.exp2(-8.0 * (torch.arange(h, dtype=torch.float32) + 1) / h)


@gpu
@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("lens,t,hq,hk,d,page", [
    ([0], 1, 1, 1, 64, 16), ([1, 0, 5], 1, 4, 1, 128, 16), ([127, 128, 129], 1, 8, 2, 64, 64), ([700], 1, 32, 4, 128, 128),
    ([63, 300], 5, 4, 4, 80, 16), ([1000, 2, 64], 17, 6, 2, 128, 1), ([250], 64, 8, 1, 64, 48), ([33, 4097], 64, 2, 2, 8, 100),
    ([15, 16, 17, 31], 16, 16, 16, 128, 16), ([2500], 3, 40, 8, 72, 256), ([511], 33, 6, 2, 120, 8)])
def test_trees(lens, t, hq, hk, d, page, dtype):
    Case(lens, t, hq, hk, d, page, dtype, seed=sum(lens) + t).check(1 / math.sqrt(d))


@gpu
@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("lens,t,hq,hk,d,page", [([90, 1300], 1, 4, 2, 128, 32), ([5, 800], 12, 8, 2, 64, 16)])
def test_cap_and_bias(lens, t, hq, hk, d, page, dtype):
    c = Case(lens, t, hq, hk, d, page, dtype, seed=5, loud=6.0)
    c.check(1 / math.sqrt(d), cap=5.0)
    c.check(1 / math.sqrt(d), slopes=slopes_of(hq))
    c.check(-0.2, cap=30.0, slopes=slopes_of(hq))


@gpu
@pytest.mark.parametrize("t", [1, 7, 64])
def test_chain(t):
    Case([100, 0, 333], t, 4, 2, 64, 16, BF16, seed=t, kind="chain").check(0.125, slopes=slopes_of(4))


@gpu
@pytest.mark.parametrize("n_drafts", [(0, 3, 9), (9, -2, 50)])
def test_ragged_drafts(n_drafts):
    Case([40, 0, 260], 9, 4, 1, 128, 16, F16, seed=3, n_drafts=n_drafts).check(0.1, slopes=slopes_of(4))


@gpu
def test_negative_lengths_and_empty_rows():
    c = Case([-3, 20], 4, 2, 1, 64, 16, F16, seed=8)
    c.check(0.125)
    c = Case([0, 20], 4, 2, 1, 64, 16, F16, seed=9)
    def blind(s):
        s["tree"][:, 2] = 0
    c.see = [x.clone() for x in c.see]
    for x in c.see:
        x[2] = False
    o = c.check(0.125, change=blind)
    assert bool((o[0, 2] == 0).all()) and bool(torch.isfinite(o[1, 2]).all())


@gpu
@pytest.mark.parametrize("t", [1, 20])
def test_broken_pages_and_short_tables(t):
    """Page numbers outside the cache and a table that ends before the tokens do: those tokens are not there."""
    c = Case([200, 75], t, 4, 2, 64, 16, BF16, seed=21)
    def damage(s):
        s["table"][0, 1], s["table"][0, 4], s["table"][1, 0] = -1, s["k"].shape[0], 2147483647
    c.check(0.125, change=damage, hide=lambda i, p: p // 16 in ((1, 4) if i == 0 else (0,)))
    def cut(s):
        s["table"] = s["table"][:, :6].contiguous()
    c.check(0.125, change=cut, hide=lambda i, p: p >= 6 * 16)
    def nothing(s):
        s["table"].fill_(-1)
    c.check(0.125, change=nothing, hide=lambda i, p: True)


@gpu
def test_strides_of_heads_first_caches():
    c = Case([150, 31], 6, 4, 2, 72, 16, F16, seed=31)
    a = c.check(0.1)
    def put(x):  # heads before tokens, unused elements between rows
        out = torch.full((x.shape[0], x.shape[2], x.shape[1], x.shape[3] + 8), 77.0, dtype=x.dtype, device="cuda").transpose(1, 2)[..., :x.shape[3]]
        out.copy_(x)
        return out
    assert torch.equal(a, c.check(0.1, layout=put))


@gpu
def test_long_cache_and_one_new_token():
    """A cache whose offsets pass 2^31 bytes, most of it unused; results of many splits are joined."""
    d, page, n = 64, 128, 40000
    pages = 140000  # x 128 x 64 x 2 bytes = 2.3 GB
    k = torch.zeros(pages, page, 1, d, dtype=F16, device="cuda")
    g = torch.Generator().manual_seed(3)
    need = -(-(n + 2) // page)
    table = (pages - 1 - torch.randperm(need, generator=g)).to(torch.int32)[None].cuda()
    kk, vv, q = (torch.randn(s, generator=g).to(F16) for s in ((n + 2, d), (n + 2, d), (1, 2, 3, d)))
    at = torch.arange(n + 2)
    k[table[0, at // page].long(), at % page, 0] = kk.cuda()
    v = torch.zeros_like(k)
    v[table[0, at // page].long(), at % page, 0] = vv.cuda()
    o = torch.empty(1, 2, 3, d, dtype=F16, device="cuda")
    ws = torch.empty(api.attn_tree_workspace_bytes(1, 2, 3, 1, d, need * page), dtype=torch.uint8, device="cuda")
    api.attn_tree(q.cuda(), k, v, table, torch.tensor([n], dtype=torch.int32, device="cuda"), o, 0.125, workspace=ws)
    assert_status_ok()
    see = torch.ones(2, n + 2, dtype=torch.bool)
    see[0, n + 1] = False
    dist = torch.zeros(2, n + 2, dtype=F64)
    for h in range(3):
        r = A.one_head(q[0, :, h].to(F64), kk.to(F64), vv.to(F64), see, dist, 0.125, out_eps=2.0 ** -11)
        A.assert_close(o[0, :, h], r["o"], r["o_tol"], f"head {h}")


@gpu
def test_repeat_stream_and_graphs():
    """The same bits again, on another stream, and from two captured graphs with a workspace each."""
    c = Case([900, 77], 5, 8, 2, 128, 16, BF16, seed=41)
    a = c.check(0.1)
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        b = c.run(0.1)
    side.synchronize()
    assert torch.equal(a, b.cpu())
    graph = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph):
        c.call()
    c.state["o"].zero_()
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(a, c.state["o"].cpu())
    c.state["lens"][0] = 411  # lengths are read on the device: a replay sees new ones
    graph.replay()
    torch.cuda.synchronize()
    other = c.state["o"].clone()
    c.call()
    assert torch.equal(other, c.state["o"]) and not torch.equal(other.cpu(), a)


@gpu
@pytest.mark.parametrize("batch,hk,d", [(1, 1, 64), (1, 2, 128), (6, 2, 128), (30, 2, 64), (40, 1, 128)])
def test_many_splits_and_few(batch, hk, d):
    """A long table makes many splits, of which short sequences fill a few: 148 blocks' worth to 4."""
    g = torch.Generator().manual_seed(batch)
    lens = [int(x) for x in torch.randint(0, 400, (batch,), generator=g)]
    lens[0] = 24000 // batch
    Case(lens, 2, 2 * hk, hk, d, 32, F16, seed=batch).check(0.1)


@gpu
@pytest.mark.parametrize("t,hq", [(1, 2), (12, 4), (20, 8)])
@pytest.mark.parametrize("n", [30, 3000])
def test_a_query_that_is_nan_shows(t, hq, n):
    """Its row is NaN, also where nothing else is to be seen; the others are what they were."""
    c = Case([n, n // 2], t, hq, 2, 64, 16, F16, seed=61, kind="chain")
    a = c.check(0.1)
    c.q[1, t - 1, 1] = math.nan
    b = c.run(0.1).cpu()
    assert bool(torch.isnan(b[1, t - 1, 1]).all())
    b[1, t - 1, 1] = a[1, t - 1, 1]
    assert torch.equal(a, b)


@gpu
@pytest.mark.parametrize("t,hq", [(4, 2), (40, 4)])
def test_no_drafted_token_at_all_then_some(t, hq):
    """A replayed graph of a batch without work writes nothing, and sees the counts that the next replay finds."""
    c = Case([5000, 70], t, hq, 2, 128, 16, BF16, seed=63, n_drafts=[0, 0])
    o = c.run(0.1)
    assert bool((o == 77.0).all())
    graph = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph):
        c.call()
    full = Case([5000, 70], t, hq, 2, 128, 16, BF16, seed=63, n_drafts=[t, t - 1])
    want = full.check(0.1)
    for name in ("q", "k", "v", "table", "lens", "tree", "depths"):
        assert c.state[name].shape == full.state[name].shape
        c.state[name].copy_(full.state[name])
    graph.replay()
    torch.cuda.synchronize()
    assert bool((c.state["o"] == 77.0).all())
    c.state["n_drafts"].copy_(torch.tensor([t, t - 1], dtype=torch.int32))
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(c.state["o"].cpu(), want)


@gpu
def test_many_rows_repeat_stream_and_two_graphs():
    """More than 32 rows to a key head: the same bits again, on another stream, and from two graphs in flight at once."""
    cases = [Case([2100, 900], 16, 8, 2, 128, 16, BF16, seed=s) for s in (71, 72)]
    want = [c.check(0.1) for c in cases]
    graphs, streams = [torch.cuda.CUDAGraph() for _ in cases], [torch.cuda.Stream() for _ in cases]
    torch.cuda.synchronize()
    for c, graph in zip(cases, graphs):
        with torch.cuda.graph(graph):
            c.call()
        c.state["o"].zero_()
    torch.cuda.synchronize()
    for _ in range(3):
        for graph, s in zip(graphs, streams):
            with torch.cuda.stream(s):
                graph.replay()
    torch.cuda.synchronize()
    for c, w in zip(cases, want):
        assert torch.equal(c.state["o"].cpu(), w)


@gpu
def test_agrees_with_attention_over_the_same_tokens():
    """A chain of drafted tokens behind a cache is causal attention of the last queries: both kernels, one definition."""
    n, t, hq, hk, d = 301, 11, 4, 2, 128
    c = Case([n], t, hq, hk, d, 16, BF16, seed=51, kind="chain")
    o = c.check(0.1, cap=20.0, slopes=slopes_of(hq))
    k, v = c.keys[0][None].cuda(), c.values[0][None].cuda()
    full = torch.empty(1, t, hq, d, dtype=BF16, device="cuda")
    api.attn_fwd(c.q.cuda(), k, v, full, None, 0.1, causal=True, cap=20.0, slopes=slopes_of(hq).cuda())
    # each is within its own bound of the definition; o is near 1, both bounds together are below 2 half steps and the two roundings of p
    assert (full.cpu().float() - o.float()).abs().max() <= 4 * 2.0 ** -9 * 4


def targs(**kw):
    a = _lib.AttnArgs()
    a.batch, a.heads_q, a.heads_kv, a.head_dim, a.scale = 2, 4, 2, 64, 0.125
    for name in ("q", "o"):
        s = getattr(a, name)
        s.batch, s.token, s.head = 5 * 4 * 64, 4 * 64, 64
    for name in ("k", "v"):
        s = getattr(a, name)
        s.batch, s.token, s.head = 16 * 2 * 64, 2 * 64, 64
    for name, x in kw.items():
        first, _, last = name.partition("_")
        if first in ("q", "k", "v", "o"):
            setattr(getattr(a, first), last, x)
        else:
            setattr(a, name, x)
    return a


def call(a, drafts=5, q=16, k=16, v=16, pages=10, page=16, table=16, ld=4, lens=16, o=16, ws=16, size=1 << 30):
    return _lib.lib().b200wmma_attn_tree(C.byref(a) if a else None, drafts, q, k, v, pages, page, table, ld, lens, None, None, None, o, ws, size, None)


@pytest.mark.parametrize("how,code", [
    (dict(batch=0), 1), (dict(heads_q=3), 1), (dict(head_dim=36), 2), (dict(head_dim=256), 2), (dict(data_type=1), 1), (dict(cap=-2.0), 1),
    (dict(len_q=5), 1), (dict(len_kv=5), 1), (dict(causal=1), 1), (dict(prefix=16), 1), (dict(doc_q=16), 1), (dict(doc_kv=16), 1),
    (dict(k_token=68), 3), (dict(v_batch=-8), 1), (dict(o_head=8), 1)])
def test_refused_arguments(how, code):
    assert call(targs(**how)) == code and b"attn_tree" in _lib.lib().b200wmma_last_error_string()


@pytest.mark.parametrize("how,code", [
    (dict(drafts=0), 2), (dict(drafts=65), 2), (dict(q=None), 1), (dict(k=None), 1), (dict(v=None), 1), (dict(o=None), 1), (dict(table=None), 1),
    (dict(lens=None), 1), (dict(pages=0), 1), (dict(page=0), 1), (dict(ld=0), 1), (dict(q=8), 3), (dict(v=24), 3), (dict(o=4), 3),
    (dict(page=1 << 16, ld=1 << 16), 2)])
def test_refused_calls(how, code):
    assert call(targs(), **how) == code and b"attn_tree" in _lib.lib().b200wmma_last_error_string()


def test_refused_null_args():
    assert call(None) == 1


def test_refused_workspaces():
    need = _lib.lib().b200wmma_attn_tree_workspace_bytes(2, 5, 4, 2, 64, 64 * 16)
    assert need > 0
    assert call(targs(), ld=64, ws=None, size=need) == 1 and call(targs(), ld=64, size=need - 1) == 1 and call(targs(), ld=64, ws=24, size=need) == 3
    assert _lib.lib().b200wmma_attn_tree_workspace_bytes(2, 5, 4, 2, 64, 16) == 0  # too short to be split


@pytest.mark.parametrize("shape", [
    (0, 5, 4, 2), (2, 0, 4, 2), (2, 65, 4, 2), (2, 5, 0, 2), (2, 5, 4, 0), (2, 5, 4, 3), (2, 5, 1, 2), (1, 64, 1 << 31, 1 << 5),
    (1 << 31, 4, 1 << 31, 1), (1, 2, 1 << 31, 1)])
def test_shapes_that_are_refused_need_no_workspace(shape):
    batch, drafts, hq, hk = shape
    assert _lib.lib().b200wmma_attn_tree_workspace_bytes(batch, drafts, hq, hk, 64, 1 << 16) == 0
    assert call(targs(batch=batch, heads_q=hq, heads_kv=hk), drafts=drafts) in (1, 2)


@pytest.mark.parametrize("how", [dict(scale=1e31), dict(cap=1e-40), dict(cap=1e-10, scale=1e25), dict(cap=1e31)])
def test_refused_scales(how):
    assert call(targs(**how)) == 2


def test_wrapper_refuses_wrong_tensors():
    t = torch.zeros(1, 4, 2, 64, dtype=F16)
    with pytest.raises(TypeError):
        api.attn_tree(t, t, t, torch.zeros(1, 1, dtype=torch.int32), torch.zeros(1, dtype=torch.int32), t, 1.0)
