"""Bounds for attention under a cap of any size.  attn_oracle.py gives the values, and bounds in which the cap's tanh is off by
some ulp of 1: enough for caps near the scores, but a bound that grows with the cap allows anything under a large one, and under a
small one it leaves out what the error of a raw score does to the cap's derivative.  Here the tanh is off by some ulp of itself.

With u = raw / cap, t = tanh u, E = 2^-24:
  raw    is off by e_raw = (d + 8) E |scale| sum |q k|  (d products and sums, the scaling), u by e_u = e_raw / cap + 2 E |u|
  t      by e_t = m e_u + 16 E |t|, m the largest 1 - tanh^2 between u - e_u and u + e_u: that of |u| - e_u, or 1 where 0 is between
  score  by cap e_t + 4 E (|slope distance| + |score|)  (scaling, bias, subtraction of the maximum)
  1-t^2  by 2 |t| e_t + 4 E  (formed from t in fp32)
What follows from these for o, lse and the gradients is attn_oracle.py's derivation.  The absolute terms stand for what lies
below fp16's normal numbers; bf16 has none."""
import math

import torch

import attn_oracle as A

F64, U32 = torch.float64, A.U32


def one_head(q, k, v, see, dist, scale, cap, slope, dout, dtype):
    """Results and bounds of one head (2-D tensors in 64 bits); dtype: the 16-bit type of a call's matrices."""
    eps, fp16 = torch.finfo(dtype).eps / 2, dtype == torch.float16
    r = A.one_head(q, k, v, see, dist, scale, cap, slope, dout, eps)
    (m, n), d = see.shape, q.shape[1]
    raw = scale * (q @ k.T)
    u = raw / cap
    t = torch.tanh(u)
    sech2 = lambda x: 1 / torch.cosh(x.clamp(-300, 300)) ** 2
    slip = sech2(u)
    e_raw = (d + 8) * U32 * abs(scale) * (q.abs() @ k.abs().T)
    e_u = e_raw / cap + 2 * U32 * u.abs()
    e_t = torch.clamp(sech2(torch.clamp(u.abs() - e_u, min=0.0)) * e_u + 16 * U32 * t.abs(), max=2.0)
    s = cap * t - slope * dist
    e_s = torch.where(see, cap * e_t + 4 * U32 * (slope * dist + s.abs()), 0.0).amax(1, keepdim=True) + 8 * U32
    live = see.any(1)
    lse = torch.where(live, r["lse"], 0.0)
    p = torch.where(see, torch.exp(s - lse[:, None]), 0.0)
    r["lse_tol"] = e_s[:, 0] + (n + 8) * U32 + 4 * U32 * lse.abs()
    small = 2.0 ** -25 if fp16 else 0.0
    # an error of a score is in its weight's exponent: for rows of large scores more than its first order
    grow = torch.exp(torch.clamp(2 * e_s, max=700.0)) - 1
    r["o_tol"] = eps * r["o"].abs() + (eps + grow + (n + 8) * U32) * (p @ v.abs() + r["o"].abs()) + small * (v.abs().sum(0) + 1)
    if dout is None:
        return r
    dp, delta = dout @ v.T, (dout * r["o"]).sum(1, keepdim=True)
    ds = torch.where(see, p * (dp - delta) * slip, 0.0)
    e_p = torch.exp(torch.clamp(2 * (e_s + r["lse_tol"][:, None]), max=700.0)) - 1
    e_delta = (dout.abs() * r["o_tol"]).sum(1, keepdim=True) + (d + 8) * U32 * (dout * r["o"]).abs().sum(1, keepdim=True)
    e_dp = (d + 8) * U32 * (dout.abs() @ v.abs().T)
    e_slip = 2 * t.abs() * e_t + 4 * U32
    e_ds = p * ((dp - delta).abs() * (e_p * slip + e_slip) + (e_dp + e_delta) * (slip + e_slip)) + eps * ds.abs() + 2 * small
    e_ds = torch.where(see, e_ds, 0.0)
    acc = lambda count, terms: (count + 8) * U32 * terms
    r["dq_tol"] = eps * r["dq"].abs() + abs(scale) * (e_ds @ k.abs()) + acc(n, abs(scale) * (ds.abs() @ k.abs())) + small
    # of dk and dv the rounding of the output is added by the caller, after the heads of a group are added up
    r["dk_tol"] = abs(scale) * (e_ds.T @ q.abs()) + acc(m, abs(scale) * (ds.abs().T @ q.abs())) + small
    r["dv_tol"] = torch.where(see, p * (eps + e_p) + 2 * small, 0.0).T @ dout.abs() + acc(m, p.T @ dout.abs()) + small
    return r


def attention(q, k, v, dout, scale, cap, causal=False, slopes=None):
    """Results and bounds ("<name>_tol") of attn_fwd and attn_bwd; q, k, v, dout [batch, tokens, heads, dim] of one 16-bit type."""
    (b, lq, hq, _), (lk, hk) = q.shape, k.shape[1:3]
    r = {name + suffix: torch.zeros((k if name in ("dk", "dv") else q).shape, dtype=F64)
         for name in ("o", "dq", "dk", "dv") for suffix in ("", "_tol")}
    r["lse"], r["lse_tol"] = torch.zeros(b, hq, lq, dtype=F64), torch.zeros(b, hq, lq, dtype=F64)
    see, dist = A.visible(lq, lk, causal), A.distance(lq, lk)
    for i in range(b):
        for h in range(hq):
            g = h // (hq // hk)
            one = one_head(*(x.to(F64) for x in (q[i, :, h], k[i, :, g], v[i, :, g])), see, dist, scale, cap,
                           0.0 if slopes is None else float(slopes[h]), dout[i, :, h].to(F64), q.dtype)
            for name in r:
                if name.startswith("lse"):
                    r[name][i, h] = one[name]
                elif name.startswith(("dk", "dv")):
                    r[name][i, :, g] += one[name]
                else:
                    r[name][i, :, h] = one[name]
    for name in ("dk", "dv"):
        r[name + "_tol"] += torch.finfo(q.dtype).eps / 2 * r[name].abs()
    return r
