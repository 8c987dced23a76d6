"""Attention, forward and backward, from its definition in 64 bits on the CPU, with bounds on what a kernel that keeps scores
and sums in fp32 and rounds the softmax weights (and the gradients of the scores) to 16 bits may be off by."""
import math

import torch

F64 = torch.float64
U32 = 2.0 ** -24  # half a step of fp32, relative


def visible(len_q, len_kv, causal=False, prefix=None, doc_q=None, doc_kv=None):
    """[len_q, len_kv] truth values of one batch entry; prefix an int, documents [len] tensors."""
    i, j = torch.arange(len_q)[:, None] + (len_kv - len_q), torch.arange(len_kv)[None, :]
    see = torch.ones(len_q, len_kv, dtype=torch.bool)
    if causal:
        see = (j <= i) | (j < (prefix if prefix is not None else 0))
    if doc_q is not None:
        see = see & (doc_q[:, None] == doc_kv[None, :]) & (doc_q >= 0)[:, None]
    return see


def distance(len_q, len_kv):
    return (torch.arange(len_q)[:, None] + (len_kv - len_q) - torch.arange(len_kv)[None, :]).abs().to(F64)


def one_head(q, k, v, see, dist, scale, cap=0.0, slope=0.0, dout=None, out_eps=0.0):
    """Results and bounds for one head of one batch entry: 2-D fp64 tensors.  out_eps is half a step of the 16-bit type.
    Values of keys that no query sees are not looked at."""
    used = see.any(0)
    k, v = torch.where(used[:, None], k, 0.0), torch.where(used[:, None], v, 0.0)
    live = see.any(1)
    q = torch.where(live[:, None], q, 0.0)
    n, d = see.shape[1], q.shape[1]
    raw = scale * (q @ k.T)
    tanh = torch.tanh(raw / cap) if cap else torch.zeros_like(raw)
    s = (cap * tanh if cap else raw) - slope * dist
    masked = s.masked_fill(~see, -math.inf)
    lse = torch.logsumexp(masked, 1)
    p = torch.where(see, torch.exp(s - torch.where(live, lse, 0.0)[:, None]), 0.0)
    o = p @ v
    # a score: d products and sums, the scaling; the cap's tanh is off by some ulp of 1; the bias and the sum are rounded
    size = abs(scale) * (q.abs() @ k.abs().T)
    ds_ = (d + 8) * U32 * size + 16 * U32 * cap + 4 * U32 * (slope * dist + s.abs())
    e_s = torch.where(see, ds_, 0.0).amax(1, keepdim=True) + 8 * U32  # and of its exponential
    r = {"o": o, "lse": torch.where(live, lse, -math.inf)}
    r["lse_tol"] = (e_s[:, 0] + (n + 8) * U32 + 4 * U32 * torch.where(live, lse, 0.0).abs())
    pv = p @ v.abs()
    small = 2.0 ** -25 * v.abs().sum(0) if out_eps > 0 else 0.0  # softmax weights below fp16's normal numbers
    e_p = out_eps + 2 * e_s + (n + 8) * U32
    r["o_tol"] = out_eps * o.abs() + e_p * (pv + o.abs()) + small + 2.0 ** -25
    if dout is None:
        return r
    dout = torch.where(live[:, None], dout, 0.0)
    dp = dout @ v.T
    delta = (dout * o).sum(1, keepdim=True)
    slip = 1 - tanh * tanh
    ds = torch.where(see, p * (dp - delta) * slip, 0.0)
    r["dq"], r["dk"], r["dv"] = scale * (ds @ k), scale * (ds.T @ q), p.T @ dout
    e_lse = e_s + r["lse_tol"][:, None]
    e_delta = (dout.abs() * r["o_tol"]).sum(1, keepdim=True) + (d + 8) * U32 * (dout * o).abs().sum(1, keepdim=True)
    e_dp = (d + 8) * U32 * (dout.abs() @ v.abs().T)
    e_ds = p * ((dp - delta).abs() * (2 * e_lse * slip + 32 * U32 if cap else 2 * e_lse) + (e_dp + e_delta) * slip) + out_eps * ds.abs() + 2.0 ** -24
    e_ds = torch.where(see, e_ds, 0.0)
    e_pt = torch.where(see, p * (out_eps + 2 * e_lse) + 2.0 ** -24, 0.0)
    m = see.shape[0]
    acc = lambda count, terms: (count + 8) * U32 * terms
    r["dq_tol"] = out_eps * r["dq"].abs() + abs(scale) * (e_ds @ k.abs()) + acc(n, abs(scale) * (ds.abs() @ k.abs())) + 2.0 ** -25
    # of dk and dv the rounding of the output is added by the caller, after the heads of a group are added up
    r["dk_tol"] = abs(scale) * (e_ds.T @ q.abs()) + acc(m, abs(scale) * (ds.abs().T @ q.abs())) + 2.0 ** -25
    r["dv_tol"] = e_pt.T @ dout.abs() + acc(m, p.T @ dout.abs()) + 2.0 ** -25
    return r


def attention(q, k, v, scale, causal=False, cap=0.0, slopes=None, prefix=None, doc_q=None, doc_kv=None, dout=None):
    """Results and bounds ("<name>_tol") of a whole call; q, k, v, dout [batch, tokens, heads, dim] of one 16-bit type."""
    eps = torch.finfo(q.dtype).eps / 2
    b, lq, hq, _ = q.shape
    lk, hk = k.shape[1:3]
    names = ["o"] + (["dq", "dk", "dv"] if dout is not None else [])
    r = {}
    for name in names:
        for suffix in ("", "_tol"):
            r[name + suffix] = torch.zeros((k if name in ("dk", "dv") else q).shape, dtype=F64)
    r["lse"], r["lse_tol"] = torch.zeros(b, hq, lq, dtype=F64), torch.zeros(b, hq, lq, dtype=F64)
    dist = distance(lq, lk)
    for i in range(b):
        see = visible(lq, lk, causal, None if prefix is None else int(prefix[i]), None if doc_q is None else doc_q[i],
                      None if doc_kv is None else doc_kv[i])
        for h in range(hq):
            g = h // (hq // hk)
            one = one_head(q[i, :, h].to(F64), k[i, :, g].to(F64), v[i, :, g].to(F64), see, dist, scale, cap,
                           0.0 if slopes is None else float(slopes[h]), None if dout is None else dout[i, :, h].to(F64), eps)
            for name in one:
                at = r[name]
                if name.startswith("lse"):
                    at[i, h] = one[name]
                elif name.startswith(("dk", "dv")):
                    at[i, :, g] += one[name]
                else:
                    at[i, :, h] = one[name]
    for name in ("dk", "dv"):
        if name in r:
            r[name + "_tol"] += eps * r[name].abs()
    return r


def assert_close(got, ref, tol, what):
    got = got.detach().cpu().to(F64)
    same = torch.isinf(ref) & (got == ref)
    assert torch.isfinite(got[~same]).all(), f"{what}: not finite"
    err = torch.where(same, 0.0, (got - ref).abs())
    assert bool((torch.where(same, 0.0, err) <= torch.where(same, 1.0, tol)).all()), f"{what}: {float((err / tol)[~same].max()):.3g} of the bound"
