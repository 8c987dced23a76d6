"""b200wmma_gemv_w4 against the definition in 64 bits.

The products x * (q - z) are exact in fp32 (11 + 5 significant bits), so what is off is the fp32 summation, scaling and the
final rounding.  Tolerance per output: half a step of the output type relative to the value, plus 2^-24 for each of at most
n + 8 additions and scalings (n of them in the worst order) relative to the sum of magnitudes."""
import numpy as np
import pytest
import torch

from gpu_util import assert_status_ok
from rocwmma_b200 import _lib, api

gpu = pytest.mark.gpu
F16, BF16, F32 = torch.float16, torch.bfloat16, torch.float32


def make(m, n, rows, group, dtype, zeros, pad=0, seed=0):
    rng = np.random.default_rng(seed)
    groups = -(-n // group)
    a = rng.integers(0, 256, (m, n // 2 + 16 * pad), dtype=np.uint8)
    s = torch.from_numpy(rng.uniform(0.01, 0.03, (m, groups + pad)).astype(np.float32)).to(dtype)
    z = rng.integers(0, 256, (m, groups + 2 * pad), dtype=np.uint8) if zeros else None  # the upper bits are ignored
    x = torch.from_numpy(rng.standard_normal((rows, n + 8 * pad)).astype(np.float32)).to(dtype)
    return a, s, z, x


def dense(a, s, z, n, group):
    """(q - z, scale) of each weight in 64 bits."""
    q = np.empty((a.shape[0], n), np.float64)
    q[:, 0::2], q[:, 1::2] = a[:, :n // 2] & 15, a[:, :n // 2] >> 4
    of = np.arange(n) // group
    if z is None:
        q = np.where(q > 7, q - 16, q)
    else:
        q = q - (z & 15)[:, of]
    return q * s.double().numpy()[:, of]


def check(m, n, rows, group, dtype, zeros=False, out=None, alpha=1.0, beta=0.0, pad=0, seed=0):
    a, s, z, x = make(m, n, rows, group, dtype, zeros, pad, seed)
    out = out or dtype
    ldy = m + 3 * pad
    y0 = torch.from_numpy(np.random.default_rng(seed + 1).standard_normal((rows, ldy)).astype(np.float32)).to(out)
    if beta == 0.0:
        y0[:, :m] = float("nan")  # not read
    y = y0.cuda()
    api.gemv_w4(m, n, rows, torch.from_numpy(a).cuda(), a.shape[1], s.cuda(), s.shape[1], group, x.cuda(), x.shape[1], y, ldy, alpha, beta,
                zeros=None if z is None else torch.from_numpy(z).cuda(), ld_zeros=0 if z is None else z.shape[1])
    assert_status_ok()
    got = y.cpu()
    assert torch.equal(got[:, m:], y0[:, m:])  # behind the rows nothing is written
    w, xx = dense(a, s, z, n, group), x.double().numpy()[:, :n]
    ref, size = alpha * (xx @ w.T), abs(alpha) * (np.abs(xx) @ np.abs(w).T)
    if beta != 0.0:
        ref, size = ref + beta * y0.double().numpy()[:, :m], size + np.abs(beta * y0.double().numpy()[:, :m])
    tol = torch.finfo(out).eps / 2 * np.abs(ref) + (n + 8) * 2.0 ** -24 * size + 2.0 ** -25
    err = np.abs(got[:, :m].double().numpy() - ref)
    assert (err <= tol).all(), (err / tol).max()
    return y


@gpu
@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("zeros", [False, True])
@pytest.mark.parametrize("m,n,rows,group", [
    (1, 32, 1, 32), (16, 256, 1, 128), (17, 96, 2, 64), (100, 4128, 1, 128), (33, 2048, 8, 32), (250, 1056, 3, 96), (64, 8192, 9, 128),
    (129, 544, 16, 64), (70, 320, 17, 1024), (40, 1280, 33, 256), (19, 2080, 64, 32), (24, 64, 65, 32), (13, 288, 130, 160),
    (2051, 224, 5, 64), (16, 40000, 4, 4000), (5, 200000, 1, 128), (5, 200000, 2, 96), (130, 96, 12, 32), (260, 1600, 40, 320)])
def test_matches_the_definition(m, n, rows, group, dtype, zeros):
    check(m, n, rows, group, dtype, zeros, seed=m + n)


@gpu
@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("rows", [1, 4, 20])
def test_strides_types_alpha_beta(dtype, rows):
    check(45, 480, rows, 64, dtype, True, pad=1, alpha=0.5, beta=-1.5)
    check(45, 480, rows, 64, dtype, False, out=F32, pad=3, alpha=-2.0, beta=1.0)
    check(45, 480, rows, 64, dtype, False, out=F32, pad=2)


@gpu
def test_large_sizes_and_repeat():
    """A wide matrix and a tall one; the same call twice gives the same bits."""
    a, b = check(4100, 8192, 1, 128, BF16, True), check(4100, 8192, 1, 128, BF16, True)
    assert torch.equal(a, b)
    a, b = check(300, 28672, 7, 128, F16), check(300, 28672, 7, 128, F16)
    assert torch.equal(a, b)


@gpu
def test_infinite_and_nan_inputs_stay_in_their_row():
    m, n, rows = 37, 512, 5
    a, s, _, x = make(m, n, rows, 128, F16, False)
    x[2, 7], x[3, 100] = float("nan"), float("inf")
    y = torch.zeros(rows, m, dtype=F16, device="cuda")
    api.gemv_w4(m, n, rows, torch.from_numpy(a).cuda(), n // 2, s.cuda(), 4, 128, x.cuda(), n, y, m, 1.0, 0.0)
    got = y.cpu()
    assert torch.isfinite(got[[0, 1, 4]]).all() and torch.isnan(got[2]).all() and not torch.isfinite(got[3]).any()


@gpu
def test_other_stream_and_graph_replay():
    m, n, rows = 300, 1024, 2
    a, s, _, x = make(m, n, rows, 64, BF16, False)
    a, s, x = torch.from_numpy(a).cuda(), s.cuda(), x.cuda()
    want, y = torch.empty(rows, m, dtype=BF16, device="cuda"), torch.zeros(rows, m, dtype=BF16, device="cuda")
    call = lambda out: api.gemv_w4(m, n, rows, a, n // 2, s, n // 64, 64, x, n, out, m, 1.0, 0.0)
    call(want)
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        call(y)
    side.synchronize()
    assert torch.equal(y, want)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        call(y)
    for seed in (1, 2):
        x.copy_(make(m, n, rows, 64, BF16, False, seed=seed)[3])
        graph.replay()
        call(want)
        torch.cuda.synchronize()
        assert torch.equal(y, want)


@gpu
@pytest.mark.parametrize("group", [32, 64, 128])
@pytest.mark.parametrize("rows", [12, 20, 50])
def test_many_vectors_repeat_and_graph(rows, group):
    """More than 8 vectors: the same bits again, and from two graphs in flight at once."""
    m, n = 520, 2400
    a, s, z, x = make(m, n, rows, group, F16, True)
    a, s, z, x = torch.from_numpy(a).cuda(), s.cuda(), torch.from_numpy(z).cuda(), x.cuda()
    groups = -(-n // group)
    y = [torch.zeros(rows, m, dtype=F16, device="cuda") for _ in range(3)]
    call = lambda out: api.gemv_w4(m, n, rows, a, n // 2, s, groups, group, x, n, out, m, 1.0, 0.0, zeros=z, ld_zeros=groups)
    call(y[0])
    graphs, streams = [torch.cuda.CUDAGraph() for _ in range(2)], [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    for graph, out in zip(graphs, y[1:]):
        with torch.cuda.graph(graph):
            call(out)
    for _ in range(3):
        for graph, side in zip(graphs, streams):
            with torch.cuda.stream(side):
                graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(y[0], y[1]) and torch.equal(y[0], y[2])
    assert_status_ok()


@gpu
@pytest.mark.parametrize("group", [32, 64, 128])
def test_many_vectors_nan_stays_in_its_row(group):
    m, n, rows = 150, 544, 18
    a, s, _, x = make(m, n, rows, group, F16, False)
    x[2, 7], x[17, 543] = float("nan"), float("inf")
    groups = -(-n // group)
    y = torch.zeros(rows, m, dtype=F16, device="cuda")
    api.gemv_w4(m, n, rows, torch.from_numpy(a).cuda(), n // 2, s.cuda(), groups, group, x.cuda(), n, y, m, 1.0, 0.0)
    got = torch.isfinite(y.cpu())
    keep = [r for r in range(rows) if r not in (2, 17)]
    assert got[keep].all() and not got[2].any() and not got[17].any()


def w4(L, m=64, n=128, rows=1, a=16, lda=64, s=16, lds=1, z=None, ldz=0, group=128, x=16, ldx=128, y=16, ldy=64, dt=0, out=0):
    return L.b200wmma_gemv_w4(m, n, rows, a, lda, s, lds, z, ldz, group, x, ldx, y, ldy, 1.0, 0.0, dt, out, None)


@pytest.mark.parametrize("how,code", [
    (dict(m=0), 1), (dict(n=0), 1), (dict(rows=0), 1), (dict(group=0), 1), (dict(a=None), 1), (dict(s=None), 1), (dict(x=None), 1),
    (dict(y=None), 1), (dict(dt=1), 1), (dict(dt=7), 1), (dict(out=2), 1), (dict(dt=2, out=0), 1), (dict(n=48, lda=32), 2), (dict(group=48), 2),
    (dict(rows=1 << 16, ldx=128), 2), (dict(lda=48), 1), (dict(ldx=120), 1), (dict(ldy=63), 1), (dict(group=64), 1), (dict(z=16, ldz=0), 1),
    (dict(a=8), 3), (dict(lda=72), 3), (dict(x=8), 3), (dict(ldx=132), 3)])
def test_refusals(how, code):
    L = _lib.lib()
    assert w4(L, **how) == code
    assert b"gemv_w4" in L.b200wmma_last_error_string()


def test_wrapper_refuses_wrong_tensors():
    x = torch.zeros(1, 64, dtype=F16)
    with pytest.raises(TypeError):
        api.gemv_w4(8, 64, 1, torch.zeros(8, 32, dtype=torch.uint8), 32, x, 1, 64, x, 64, x, 8, 1.0, 0.0)  # not on a GPU
    with pytest.raises(TypeError):
        api.gemv_w4(8, 64, 1, None, 32, None, 1, 64, x.float(), 64, x, 8, 1.0, 0.0)
