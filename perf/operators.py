"""Measured cases of the decoding and attention operators: products with 4-bit group-scaled weights, masked attention
with its gradients, and attention of drafted tokens over a paged cache.

`run` computes each in a plain form (elementary torch operations in fp32) or, where `own` is true, through the
package's entry points.  `exact` gives the same results from the definitions in fp64."""
import math

import numpy as np
import torch

own = False

_TYPES = {"f16": torch.float16, "bf16": torch.bfloat16}


def listed():
    """Sizes are generic: powers of two where programs use them, odd ones where a batch leaves them."""
    return [
        # one token through a small projection: launch latency counts
        {"name": "w4_1x2048x2048", "op": "w4", "type": "bf16", "rows": 1, "m": 2048, "n": 2048, "group": 128, "zeros": False},
        # one token through a large projection: a stream of the weights
        {"name": "w4_1x16384x8192", "op": "w4", "type": "f16", "rows": 1, "m": 16384, "n": 8192, "group": 128, "zeros": True},
        # a few drafted tokens or sequences at once, small groups, an odd number of outputs
        {"name": "w4_7x5003x4128", "op": "w4", "type": "bf16", "rows": 7, "m": 5003, "n": 4128, "group": 32, "zeros": True},
        # a verified tree of drafted tokens through a large projection
        {"name": "w4_32x14336x4096", "op": "w4", "type": "bf16", "rows": 32, "m": 14336, "n": 4096, "group": 64, "zeros": False},
        # the prompt of a few sequences, capped scores
        {"name": "attn_cap_4096", "op": "attn", "type": "bf16", "batch": 2, "heads_q": 16, "heads_kv": 4, "len_q": 4096, "len_kv": 4096,
         "dim": 128, "causal": True, "cap": 30.0, "bias": False, "prefix": False, "docs": 0, "pad": 0},
        # a later piece of a prompt behind what is known already, distances as a bias, odd lengths
        {"name": "attn_bias_piece", "op": "attn", "type": "f16", "batch": 3, "heads_q": 12, "heads_kv": 12, "len_q": 517, "len_kv": 1931,
         "dim": 64, "causal": True, "cap": 0.0, "bias": True, "prefix": False, "docs": 0, "pad": 0},
        # a training step on packed documents with padding behind them
        {"name": "train_docs_8192", "op": "train", "type": "bf16", "batch": 1, "heads_q": 16, "heads_kv": 8, "len_q": 8192, "len_kv": 8192,
         "dim": 128, "causal": True, "cap": 0.0, "bias": False, "prefix": False, "docs": 5, "pad": 100},
        # a training step with a prefix that every token sees, capped scores and distances, small heads and an odd length
        {"name": "train_prefix_1027", "op": "train", "type": "f16", "batch": 2, "heads_q": 8, "heads_kv": 8, "len_q": 1027, "len_kv": 1027,
         "dim": 80, "causal": True, "cap": 20.0, "bias": True, "prefix": True, "docs": 0, "pad": 0},
        # a training step on whole sequences
        {"name": "train_full_4096", "op": "train", "type": "bf16", "batch": 2, "heads_q": 16, "heads_kv": 16, "len_q": 4096, "len_kv": 4096,
         "dim": 128, "causal": True, "cap": 0.0, "bias": False, "prefix": False, "docs": 0, "pad": 0},
        # one new token for each of many sequences
        {"name": "tree_1_of_32", "op": "tree", "type": "bf16", "batch": 32, "drafts": 1, "heads_q": 32, "heads_kv": 8, "context": 6000,
         "page": 64, "dim": 128, "cap": 0.0, "bias": False},
        # a tree of drafted tokens for a few sequences, capped scores
        {"name": "tree_24_of_4", "op": "tree", "type": "bf16", "batch": 4, "drafts": 24, "heads_q": 16, "heads_kv": 4, "context": 3001,
         "page": 16, "dim": 128, "cap": 30.0, "bias": False},
        # one sequence with a long cache, distances as a bias
        {"name": "tree_5_long", "op": "tree", "type": "f16", "batch": 1, "drafts": 5, "heads_q": 8, "heads_kv": 2, "context": 120001,
         "page": 128, "dim": 64, "cap": 0.0, "bias": True},
    ]


def draw(rng):
    """One more case of the ranges above."""
    def spread(lo, hi):
        return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))

    op = rng.choice(["w4", "attn", "train", "tree"])
    case = {"op": op, "type": rng.choice(["f16", "bf16"])}
    if op == "w4":
        case |= {"rows": rng.choice([1, 1, 2, spread(3, 32)]), "m": spread(64, 16384), "n": 32 * spread(8, 512),
                 "group": rng.choice([32, 64, 128, 256]), "zeros": rng.random() < 0.5}
    elif op == "tree":
        heads_kv = rng.choice([1, 2, 4, 8])
        context = spread(1, 60000)
        case |= {"batch": max(1, min(spread(1, 32), 192000 // context)), "drafts": rng.choice([1, 1, spread(2, 64)]),
                 "heads_q": heads_kv * rng.choice([1, 2, 4, 8]), "heads_kv": heads_kv, "context": context,
                 "page": rng.choice([16, 32, 64, 128]), "dim": rng.choice([64, 80, 128]), "cap": rng.choice([0.0, 0.0, 30.0]),
                 "bias": rng.random() < 0.3}
    else:
        heads_kv = rng.choice([1, 2, 4, 8])
        length = spread(1, 4096)
        docs = rng.choice([0, 0, rng.randint(1, 6)]) if length >= 64 else 0
        prefix = docs == 0 and rng.random() < 0.3
        case |= {"batch": rng.randint(1, 2), "heads_q": heads_kv * rng.choice([1, 2]), "heads_kv": heads_kv, "len_q": length,
                 "len_kv": length if docs or rng.random() < 0.7 else length + spread(1, 1000), "dim": rng.choice([64, 72, 128]),
                 "causal": prefix or rng.random() < 0.75, "cap": rng.choice([0.0, 0.0, 25.0]), "bias": rng.random() < 0.3,
                 "prefix": prefix, "docs": docs, "pad": rng.randint(0, length // 8) if docs else 0}
    return case


# ---- what of a case's masks is settled by its sizes ---------------------------------------------------------------
def _doc_ids(case):
    """Documents one behind the other, of growing lengths, and -1 for the padding behind the last one."""
    length, used = case["len_q"], case["len_q"] - case["pad"]
    at = np.arange(length, dtype=np.float64)
    ids = np.floor(case["docs"] * np.sqrt((at + 0.5) / used)).astype(np.int32)
    return np.where(np.arange(length) < used, np.minimum(ids, case["docs"] - 1), -1).astype(np.int32)


def _prefixes(case):
    return (case["len_kv"] * (1 + np.arange(case["batch"])) // (2 + case["batch"])).astype(np.int32)


def _lens(case):
    """Tokens in the cache of each sequence: the context and less, down to about half of it."""
    return (case["context"] - (case["context"] // 2) * np.arange(case["batch"]) // case["batch"]).astype(np.int32)


def _parents(case):
    """Drafted token i hangs on token parent[i] of the tree (-1: on the last token of the cache)."""
    i = np.arange(case["drafts"])
    return np.where(i == 0, -1, (i - 1) // 2 * (i % 5 != 4) + (i - 1) * (i % 5 == 4)).astype(np.int64)


def _tree(case):
    """(ancestors as a truth matrix with the token itself, depth of each token) of the drafted tree."""
    t = case["drafts"]
    parents = torch.from_numpy(_parents(case))
    step = torch.zeros(t, t, dtype=torch.float64)
    has = torch.nonzero(parents >= 0).flatten()
    step[has, parents[has]] = 1.0
    sees = torch.linalg.inv(torch.eye(t, dtype=torch.float64) - step) > 0.5  # the sum of all powers of the parent relation
    return sees, sees.sum(1) - 1


def _slopes(case):
    """One slope to a head, each a step below the one before."""
    h = case["heads_q"]
    return torch.exp2(-8.0 * (torch.arange(h, dtype=torch.float32) + 1.0) / h)


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    dt = _TYPES[case["type"]]

    def normal(*shape, by=1.0):
        return (torch.randn(*shape, generator=g, device="cuda") * by).to(dt)

    s = {"case": case}
    if case["op"] == "w4":
        m, n, rows = case["m"], case["n"], case["rows"]
        groups = -(-n // case["group"])
        s["a"] = torch.randint(0, 256, (m, n // 2), generator=g, device="cuda", dtype=torch.uint8)
        s["scales"] = ((torch.rand(m, groups, generator=g, device="cuda") + 0.5) / (4.6 * math.sqrt(n))).to(dt)
        s["zeros"] = torch.randint(6, 11, (m, groups), generator=g, device="cuda", dtype=torch.uint8) if case["zeros"] else None
        s["x"] = normal(rows, n)
        s["y"] = torch.empty(rows, m, device="cuda", dtype=dt)
        return s
    s["scale"] = 1.0 / math.sqrt(case["dim"])
    s["slopes"] = _slopes(case).cuda() if case["bias"] else None
    hq, hk, d, b = case["heads_q"], case["heads_kv"], case["dim"], case["batch"]
    if case["op"] == "tree":
        t, page = case["drafts"], case["page"]
        lens = _lens(case)
        need = -(-(lens + t) // page)
        pages = int(need.sum())
        table = torch.zeros(b, int(need.max()), dtype=torch.int32)
        order = torch.randperm(pages, generator=torch.Generator().manual_seed(seed)).to(torch.int32)
        at = 0
        for i in range(b):
            table[i, :need[i]] = order[at:at + need[i]]
            at += int(need[i])
        sees, depth = _tree(case)
        bits = (sees.to(torch.int64) << torch.arange(t)).sum(1)  # bit j of word i: token i sees token j
        s["table"], s["lens"] = table.cuda(), torch.from_numpy(lens).cuda()
        s["tree"] = bits.expand(b, t).contiguous().cuda()
        s["depths"] = depth.to(torch.int32).expand(b, t).contiguous().cuda()
        s["q"] = normal(b, t, hq, d, by=2.0)
        s["k"], s["v"] = normal(pages, page, hk, d), normal(pages, page, hk, d)
        s["o"] = torch.empty_like(s["q"])
        return s
    lq, lk = case["len_q"], case["len_kv"]
    s["doc"] = torch.from_numpy(_doc_ids(case)).cuda().expand(b, lq).contiguous() if case["docs"] else None
    s["prefix"] = torch.from_numpy(_prefixes(case)).cuda() if case["prefix"] else None
    s["q"], s["k"], s["v"] = normal(b, lq, hq, d, by=2.0), normal(b, lk, hk, d), normal(b, lk, hk, d)
    s["o"] = torch.empty_like(s["q"])
    s["lse"] = torch.empty(b, hq, lq, device="cuda", dtype=torch.float32)
    if case["op"] == "train":
        s["do"] = normal(b, lq, hq, d)
        s["dq"], s["dk"], s["dv"] = torch.empty_like(s["q"]), torch.empty_like(s["k"]), torch.empty_like(s["v"])
    return s


# ---- the plain forms ---------------------------------------------------------------------------------------------
def _plain_w4(s):
    a, n, group = s["a"], s["case"]["n"], s["case"]["group"]
    q = torch.stack((a & 15, a >> 4), dim=2).reshape(a.shape[0], n).float()  # the low nibble is the even column
    q = torch.where(q > 7, q - 16, q) if s["zeros"] is None else q - s["zeros"].float().repeat_interleave(group, 1)[:, :n]
    w = q * s["scales"].float().repeat_interleave(group, 1)[:, :n]
    return (s["x"].float() @ w.t()).to(s["x"].dtype)


def _visible(s):
    """Which keys each query sees: [batch or 1, 1, len_q, len_kv]; None where it sees them all."""
    case = s["case"]
    i = torch.arange(case["len_q"], device="cuda")[:, None] + (case["len_kv"] - case["len_q"])
    j = torch.arange(case["len_kv"], device="cuda")[None, :]
    see = (j <= i)[None] if case["causal"] else torch.ones(1, case["len_q"], case["len_kv"], dtype=torch.bool, device="cuda")
    if s["prefix"] is not None:
        see = see | (j[None] < s["prefix"][:, None, None])
    if s["doc"] is not None:
        see = see & (s["doc"][:, :, None] == s["doc"][:, None, :]) & (s["doc"][:, :, None] >= 0)
    return see[:, None]


def _softmax(score, see):
    """(probabilities, log of the sum) of masked scores; a row that sees nothing has no probability and -inf."""
    score = torch.where(see, score, -math.inf)
    top = score.amax(-1, keepdim=True)
    e = torch.exp(score - torch.where(top > -math.inf, top, 0.0))
    total = e.sum(-1, keepdim=True)
    return e / torch.where(total > 0, total, 1.0), (top + torch.log(total))[..., 0]


def _plain_attn(s):
    case = s["case"]
    group = case["heads_q"] // case["heads_kv"]
    q = s["q"].float().transpose(1, 2)
    k = s["k"].float().transpose(1, 2).repeat_interleave(group, 1)
    v = s["v"].float().transpose(1, 2).repeat_interleave(group, 1)
    score = (q @ k.transpose(2, 3)) * s["scale"]
    tanh = torch.tanh(score / case["cap"]) if case["cap"] else None
    score = tanh * case["cap"] if case["cap"] else score
    if case["bias"]:
        i = torch.arange(case["len_q"], device="cuda")[:, None] + (case["len_kv"] - case["len_q"])
        far = (i - torch.arange(case["len_kv"], device="cuda")[None, :]).abs()
        score = score - s["slopes"][:, None, None] * far
    p, lse = _softmax(score, _visible(s))
    o = p @ v
    out = {"o": o.transpose(1, 2).to(s["q"].dtype), "lse": lse}
    if case["op"] == "attn":
        return out
    do = s["do"].float().transpose(1, 2)
    dp = do @ v.transpose(2, 3)
    ds = p * (dp - (p * dp).sum(-1, keepdim=True)) * s["scale"]
    ds = ds * (1 - tanh * tanh) if case["cap"] else ds
    back = (case["batch"], case["heads_kv"], group, case["len_kv"], case["dim"])
    out["dq"] = (ds @ k).transpose(1, 2).to(s["q"].dtype)
    out["dk"] = (ds.transpose(2, 3) @ q).reshape(back).sum(2).transpose(1, 2).to(s["q"].dtype)
    out["dv"] = (p.transpose(2, 3) @ do).reshape(back).sum(2).transpose(1, 2).to(s["q"].dtype)
    return out


def _plain_tree(s):
    case = s["case"]
    b, t, hk, page = case["batch"], case["drafts"], case["heads_kv"], case["page"]
    group = case["heads_q"] // hk
    keys = s["table"].shape[1] * page
    k = s["k"][s["table"].long()].reshape(b, keys, hk, -1).float().permute(0, 2, 3, 1)
    v = s["v"][s["table"].long()].reshape(b, keys, hk, -1).float().permute(0, 2, 1, 3)
    q = s["q"].float().reshape(b, t, hk, group, -1).permute(0, 2, 3, 1, 4).reshape(b, hk, group * t, -1)
    score = (q @ k).reshape(b, hk, group, t, keys) * s["scale"]
    score = torch.tanh(score / case["cap"]) * case["cap"] if case["cap"] else score
    at = torch.arange(keys, device="cuda")[None, :] - s["lens"][:, None]  # place behind the cached tokens
    draft = at.clamp(0, t - 1)
    words = s["tree"][:, :, None]
    in_tree = ((words >> draft[:, None, :]) & 1).bool() & (at >= 0)[:, None] & (at < t)[:, None]
    see = ((at < 0)[:, None] | in_tree)[:, None, None]
    if case["bias"]:
        where = torch.where(at < 0, at, torch.gather(s["depths"].long(), 1, draft))
        far = (s["depths"].long()[:, :, None] - where[:, None, :]).abs()
        score = score - s["slopes"].reshape(1, hk, group, 1, 1) * far[:, None, None]
    p, _ = _softmax(score, see)
    o = (p.reshape(b, hk, group * t, keys) @ v).reshape(b, hk, group, t, -1)
    return o.permute(0, 3, 1, 2, 4).reshape(s["q"].shape).to(s["q"].dtype)


# ---- the package's operators --------------------------------------------------------------------------------------
def _own(s):
    from rocwmma_b200 import api

    case = s["case"]
    if case["op"] == "w4":
        groups = s["scales"].shape[1]
        api.gemv_w4(case["m"], case["n"], case["rows"], s["a"], case["n"] // 2, s["scales"], groups, case["group"], s["x"], case["n"],
                    s["y"], case["m"], 1.0, 0.0, zeros=s["zeros"], ld_zeros=groups)
        return s["y"]
    if case["op"] == "tree":
        if "ws" not in s:
            need = api.attn_tree_workspace_bytes(case["batch"], case["drafts"], case["heads_q"], case["heads_kv"], case["dim"],
                                                 s["table"].shape[1] * case["page"])
            s["ws"] = torch.empty(need, dtype=torch.uint8, device="cuda")
        api.attn_tree(s["q"], s["k"], s["v"], s["table"], s["lens"], s["o"], s["scale"], tree=s["tree"], depths=s["depths"],
                      cap=case["cap"], slopes=s["slopes"], workspace=s["ws"])
        return s["o"]
    if "ws" not in s:
        need = api.attn_workspace_bytes(case["batch"], case["heads_q"], case["len_q"], case["len_kv"], case["op"] == "train")
        s["ws"] = torch.empty(need, dtype=torch.uint8, device="cuda")
    how = {"causal": case["causal"], "cap": case["cap"], "slopes": s["slopes"], "prefix": s["prefix"], "doc_q": s["doc"], "doc_kv": s["doc"],
           "workspace": s["ws"]}
    api.attn_fwd(s["q"], s["k"], s["v"], s["o"], s["lse"], s["scale"], **how)
    if case["op"] == "attn":
        return {"o": s["o"], "lse": s["lse"]}
    api.attn_bwd(s["q"], s["k"], s["v"], s["o"], s["do"], s["lse"], s["dq"], s["dk"], s["dv"], s["scale"], **how)
    return {"o": s["o"], "lse": s["lse"], "dq": s["dq"], "dk": s["dk"], "dv": s["dv"]}


def run(state):
    if own:
        return _own(state)
    op = state["case"]["op"]
    return _plain_w4(state) if op == "w4" else _plain_tree(state) if op == "tree" else _plain_attn(state)


# ---- what a pass cannot do without --------------------------------------------------------------------------------
def work(case):
    if case["op"] == "w4":
        m, n, rows = case["m"], case["n"], case["rows"]
        groups = -(-n // case["group"])
        return {"bytes": m * n // 2 + m * groups * (3 if case["zeros"] else 2) + 2 * rows * (n + m), "flops": 2 * rows * m * n}
    hq, hk, d, b = case["heads_q"], case["heads_kv"], case["dim"], case["batch"]
    if case["op"] == "tree":
        t = case["drafts"]
        cached = int(_lens(case).sum())
        seen = cached * t + b * int(_tree(case)[0].sum())
        return {"bytes": 4 * hk * d * (cached + b * t) + 4 * b * t * hq * d, "flops": 4 * hq * d * seen}
    lq, lk = case["len_q"], case["len_kv"]
    pairs = 0
    for i in range(b):
        at, j = np.arange(lq)[:, None] + (lk - lq), np.arange(lk)[None, :]
        see = j <= at if case["causal"] else np.ones((lq, lk), bool)
        if case["prefix"]:
            see = see | (j < _prefixes(case)[i])
        if case["docs"]:
            ids = _doc_ids(case)
            see = see & (ids[:, None] == ids[None, :]) & (ids >= 0)[:, None]
        pairs += int(see.sum())
    q_bytes, k_bytes, lse = 2 * b * lq * hq * d, 2 * b * lk * hk * d, 4 * b * hq * lq
    if case["op"] == "attn":
        return {"bytes": 2 * q_bytes + 2 * k_bytes + lse, "flops": 4 * hq * d * pairs}
    # forward, then five products of the backward pass; q, k, v, o, do and the row statistics in, o and three gradients out
    return {"bytes": 4 * q_bytes + 4 * k_bytes + lse, "flops": 14 * hq * d * pairs}


# ---- the definitions in 64 bits -----------------------------------------------------------------------------------
def exact(case, seed):
    s = prepare(case, seed)
    f64 = torch.float64
    if case["op"] == "w4":
        m, n = case["m"], case["n"]
        y = torch.empty(case["rows"], m, dtype=f64, device="cuda")
        of = torch.arange(n, device="cuda") // case["group"]
        for r in range(0, m, 1024):
            a = s["a"][r:r + 1024].to(torch.int64)
            w = torch.empty(a.shape[0], n, dtype=torch.int64, device="cuda")
            w[:, 0::2], w[:, 1::2] = a % 16, a // 16
            if case["zeros"]:
                w = w - s["zeros"][r:r + 1024].to(torch.int64)[:, of]
            else:
                w = (w + 8) % 16 - 8
            y[:, r:r + 1024] = torch.einsum("ik,jk->ij", s["x"].to(f64), w.to(f64) * s["scales"][r:r + 1024].to(f64)[:, of])
        return y
    b, hq, hk = case["batch"], case["heads_q"], case["heads_kv"]
    group = hq // hk

    def scores(q, k, far, slope):
        raw = torch.einsum("id,jd->ij", q, k) * s["scale"]
        out = case["cap"] * torch.tanh(raw / case["cap"]) if case["cap"] else raw
        return out - slope * far if case["bias"] else out, raw

    def weights(score, see):
        score = score.masked_fill(~see, -math.inf)
        lse = torch.logsumexp(score, 1)
        return torch.where(see, torch.exp(score - lse[:, None]), 0.0), lse

    slopes = s["slopes"].to(f64) if case["bias"] else torch.zeros(hq, dtype=f64, device="cuda")
    if case["op"] == "tree":
        o = torch.zeros(s["q"].shape, dtype=f64, device="cuda")
        t, page = case["drafts"], case["page"]
        sees, depth = _tree(case)
        for i in range(b):
            n = int(s["lens"][i])
            pages = s["table"][i, :-(-(n + t) // page)].long()
            see = torch.cat([torch.ones(t, n, dtype=torch.bool), sees], 1).cuda()
            where = torch.cat([torch.arange(n), n + depth]).cuda()
            far = ((n + depth).cuda()[:, None] - where[None, :]).abs().to(f64)
            for h in range(hq):
                k = s["k"][pages, :, h // group].reshape(-1, case["dim"])[:n + t].to(f64)
                v = s["v"][pages, :, h // group].reshape(-1, case["dim"])[:n + t].to(f64)
                p, _ = weights(scores(s["q"][i, :, h].to(f64), k, far, slopes[h])[0], see)
                o[i, :, h] = p @ v
        return o
    lq, lk = case["len_q"], case["len_kv"]
    out = {"o": torch.zeros(s["q"].shape, dtype=f64, device="cuda"), "lse": torch.zeros(b, hq, lq, dtype=f64, device="cuda")}
    if case["op"] == "train":
        out["dq"], out["dk"], out["dv"] = (torch.zeros(s[x].shape, dtype=f64, device="cuda") for x in "qkv")
    place, key = torch.arange(lq, device="cuda") + lk - lq, torch.arange(lk, device="cuda")
    far = (place[:, None] - key[None, :]).abs().to(f64)
    for i in range(b):
        see = place[:, None] >= key[None, :] if case["causal"] else torch.ones(lq, lk, dtype=torch.bool, device="cuda")
        if case["prefix"]:
            see = see | (key < s["prefix"][i])[None, :]
        if case["docs"]:
            ids = s["doc"][i]
            see = see & torch.eq(ids[:, None], ids[None, :]) & (ids != -1)[None, :]
        for h in range(hq):
            q, k, v = s["q"][i, :, h].to(f64), s["k"][i, :, h // group].to(f64), s["v"][i, :, h // group].to(f64)
            score, raw = scores(q, k, far, slopes[h])
            p, lse = weights(score, see)
            o = p @ v
            out["o"][i, :, h], out["lse"][i, h] = o, lse
            if case["op"] == "train":
                do = s["do"][i, :, h].to(f64)
                ds = p * (do @ v.t() - (do * o).sum(1, keepdim=True))
                if case["cap"]:
                    ds = ds / torch.cosh(raw / case["cap"]) ** 2  # the derivative of tanh
                out["dq"][i, :, h] = s["scale"] * (ds @ k)
                out["dk"][i, :, h // group] += s["scale"] * (ds.t() @ q)
                out["dv"][i, :, h // group] += p.t() @ do
    return out
