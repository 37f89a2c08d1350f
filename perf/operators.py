"""Workloads of the operators between dense token columns and sparse matrices.

A dense matrix holds one token per column (V scores, column-major, so a tensor of shape
(tokens, V)); a sparse matrix holds a few of those rows per token.  Measured are

  route            scores of experts -> the picked experts' weights (sparse), and its gradient
  topLogits        a teacher's logits -> its top logits (sparse) and the log-sum-exp
  distill          loss of a student's logits against a teacher's top logits: the forward pass,
                   the gradient, and both in one call

`run` computes them in plain torch operations, or, where `own` is true, through the package.
"""
import math

import torch

own = False

DTYPES = {"fp32": torch.float32, "bf16": torch.bfloat16, "fp16": torch.float16}
_SIZE = {"fp32": 4, "bf16": 2, "fp16": 2}


def listed():
    return [
        # one decoding step of a few sequences through a small mixture: latency only
        dict(name="route_decode", op="route", dtype="fp32", rows=64, cols=4, k=6, score="softmax", bias=False,
             groups=1, topgroups=1, grouptop=1, renorm=True, scale=1.0, padded=0),
        # a training batch through a mixture with a balancing bias and device groups, some padded tokens
        dict(name="route_batch", op="route", dtype="fp32", rows=256, cols=4096, k=8, score="sigmoid", bias=True,
             groups=8, topgroups=4, grouptop=2, renorm=True, scale=2.5, padded=100),
        # a long prefill in 16 bits, groups ranked by their best expert
        dict(name="route_long", op="route", dtype="bf16", rows=160, cols=65537, k=6, score="softmax", bias=False,
             groups=8, topgroups=3, grouptop=1, renorm=False, scale=16.0, padded=0),
        # the backward pass of the training batch
        dict(name="route_grad_batch", op="route_grad", dtype="fp32", rows=256, cols=4096, k=8, score="sigmoid",
             renorm=True, scale=2.5),
        # the backward pass where the weights keep the softmax over all experts (every score has a gradient)
        dict(name="route_grad_long", op="route_grad", dtype="bf16", rows=160, cols=65537, k=6, score="softmax",
             renorm=False, scale=16.0),
        # one token's candidates while decoding
        dict(name="top_one", op="top", dtype="fp32", rows=32768, cols=1, k=40, temperature=1.0, lse=False, padded=0),
        # an odd vocabulary in fp16, a ragged batch
        dict(name="top_odd", op="top", dtype="fp16", rows=100003, cols=257, k=64, temperature=2.0, lse=True, padded=3),
        # a teacher's batch written to a distillation set
        dict(name="top_large", op="top", dtype="bf16", rows=131072, cols=2048, k=64, temperature=1.0, lse=True,
             padded=72),
        # validation loss of a few tokens of a small vocabulary
        dict(name="distill_few", op="distill", dtype="fp32", rows=8192, cols=16, k=20, temperature=1.0, lse=False,
             padded=0),
        # validation loss against the teacher's own probabilities (not renormalised over its top)
        dict(name="distill_odd", op="distill", dtype="bf16", rows=100003, cols=1000, k=64, temperature=1.0, lse=True,
             padded=3),
        # the gradient from a saved forward pass, masked tokens and tokens without a teacher among them
        dict(name="distill_grad", op="distill_grad", dtype="fp32", rows=50001, cols=1500, k=100, temperature=2.0,
             lse=False, padded=0),
        # a training step's loss and gradient in one call
        dict(name="distill_step", op="distill_step", dtype="bf16", rows=131072, cols=2048, k=64, temperature=2.0,
             lse=False, padded=72),
    ]


def _logint(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["route", "route_grad", "top", "distill", "distill_grad", "distill_step"])
    dtype = rng.choice(["fp32", "bf16", "fp16"])
    if op in ("route", "route_grad"):
        groups = rng.choice([1, 1, 2, 4, 8])
        rows = groups * max(2, _logint(rng, 8, 512) // groups)
        cols = _logint(rng, 1, min(65537, 10485920 // rows))
        topgroups = rng.randint(1, groups)
        k = rng.randint(1, min(16, topgroups * (rows // groups)))
        case = dict(op=op, dtype=dtype, rows=rows, cols=cols, k=k, score=rng.choice(["softmax", "sigmoid"]),
                    renorm=rng.random() < 0.5, scale=rng.choice([1.0, 2.5]))
        if op == "route":
            case.update(bias=rng.random() < 0.5, groups=groups, topgroups=topgroups, grouptop=rng.choice([1, 2]),
                        padded=rng.choice([0, cols // 10]))
        return case
    rows = _logint(rng, 512, 131072)
    cols = _logint(rng, 1, min(8192, (1 << (27 if dtype == "fp32" else 28)) // rows))
    return dict(op=op, dtype=dtype, rows=rows, cols=cols, k=_logint(rng, 1, 128),
                temperature=rng.choice([1.0, 2.0]), lse=rng.random() < 0.5, padded=rng.choice([0, rows // 100]))


# ---------------------------------------------------------------------------------------- inputs

def _generator(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(int(seed))
    return g


def _fixed_pattern(cols, k):
    """pjc and pic of a matrix with k entries in every column."""
    pjc = torch.arange(0, cols * k + 1, k, dtype=torch.int32, device="cuda")
    pic = torch.arange(cols, dtype=torch.int32, device="cuda").repeat_interleave(k)
    return pjc, pic


def _strata(rows, cols, k, g):
    """k distinct rows per column in a random order: one from each of k equal strata."""
    u = torch.rand((cols, k), generator=g, device="cuda", dtype=torch.float64)
    i = torch.arange(k, device="cuda", dtype=torch.float64)
    lo = torch.floor(i * rows / k)
    hi = torch.floor((i + 1) * rows / k)
    r = (lo + torch.floor(u * (hi - lo))).to(torch.int64).clamp_(max=rows - 1)
    order = torch.rand((cols, k), generator=g, device="cuda").argsort(dim=1)
    return r.gather(1, order)


def prepare(case, seed):
    g = _generator(seed)
    rows, cols, k = case["rows"], case["cols"], case["k"]
    dt = DTYPES[case["dtype"]]
    s = dict(case=case)
    if case["op"] in ("route", "route_grad"):
        x = (1.5 * torch.randn((cols, rows), generator=g, device="cuda")).to(dt)
        if case.get("padded"):
            x[cols - case["padded"]:] = -math.inf
        s["x"] = x
        if case["op"] == "route":
            s["bias"] = 0.1 * torch.randn(rows, generator=g, device="cuda") if case["bias"] else None
            return s
        # the forward pass's picks and weights, and the gradient that reached them
        r = x.float().topk(k, dim=1).indices
        p = torch.softmax(x.float(), 1) if case["score"] == "softmax" else torch.sigmoid(x.float())
        w = p.gather(1, r)
        if case["renorm"]:
            w = w / w.sum(1, keepdim=True)
        s["pjc"], s["pic"] = _fixed_pattern(cols, k)
        s["pir"] = r.to(torch.int32).reshape(-1)
        s["weights"] = (w * case["scale"]).reshape(-1)
        s["dweights"] = torch.randn(cols * k, generator=g, device="cuda")
        return s
    x = (2.0 * torch.randn((cols, rows), generator=g, device="cuda", dtype=torch.float32))
    if case["op"] == "top":
        x = x.to(dt)
        if case["padded"]:
            x[:, rows - case["padded"]:] = -math.inf        # rows that only pad the vocabulary
        s["x"] = x
        return s
    # a teacher's k largest logits per token; the student has learned part of them
    live = rows - case["padded"]
    kk = min(k, live)
    r = _strata(live, cols, kk, g)
    z = 6.0 + 2.5 * torch.randn((cols, kk), generator=g, device="cuda")
    z = torch.sort(z, dim=1, descending=True).values
    x.scatter_(1, r, z + 1.5 * torch.randn((cols, kk), generator=g, device="cuda"))
    x = x.to(dt)
    if case["padded"]:
        x[:, live:] = -math.inf
    # every tenth token or so has no teacher (a prompt token, padding); the others have 1 to k entries
    count = torch.randint(1, kk + 1, (cols,), generator=g, device="cuda")
    count = torch.where(torch.rand(cols, generator=g, device="cuda") < 0.7, torch.full_like(count, kk), count)
    if cols > 1:
        count = torch.where(torch.rand(cols, generator=g, device="cuda") < 0.1, torch.zeros_like(count), count)
    keep = torch.arange(kk, device="cuda")[None, :] < count[:, None]
    s["x"] = x
    s["pir"] = r[keep].to(torch.int32)
    s["pdata"] = z[keep].contiguous()
    s["pic"] = torch.arange(cols, device="cuda", dtype=torch.int32).repeat_interleave(count)
    s["pjc"] = torch.zeros(cols + 1, dtype=torch.int32, device="cuda")
    s["pjc"][1:] = torch.cumsum(count, 0).to(torch.int32)
    s["tlse"] = None
    if case["lse"]:      # the teacher's whole vocabulary holds a little more than its top
        full = torch.logsumexp(z / case["temperature"], 1)
        s["tlse"] = (full + 0.05 + 0.1 * torch.rand(cols, generator=g, device="cuda")).contiguous()
    if case["op"] != "distill":
        # the mean over the tokens; gradients in fp16 carry a loss scale, as they have to
        w = torch.full((cols,), 1024.0 if case["dtype"] == "fp16" else 1.0 / cols, device="cuda")
        if cols > 1:
            w[torch.rand(cols, generator=g, device="cuda") < 0.05] = 0.0
        s["weights"] = w
    if case["op"] == "distill_grad":
        s["slse"] = torch.logsumexp(x.float() / case["temperature"], 1)
    return s


# ---------------------------------------------------------------------------------------- plain forms

def _plain_route(s):
    c, x = s["case"], s["x"].double()       # 64 bits: two scores next to each other must not change places
    T, E = x.shape
    top = x.amax(1, keepdim=True)
    if c["score"] == "softmax":
        e = torch.exp(x - torch.where(torch.isinf(top), torch.zeros_like(top), top))
        score = e / e.sum(1, keepdim=True).clamp_min(1e-300)
    else:
        score = 1.0 / (1.0 + torch.exp(-x))
    ranked = score if s["bias"] is None else score + s["bias"].double()
    free = x > -math.inf
    key = torch.where(free, x if s["bias"] is None else ranked, -math.inf)
    G = c["groups"]
    if G > 1:
        inside = torch.where(free, ranked, -math.inf).view(T, G, E // G)
        best = torch.sort(inside, dim=2, descending=True).values[:, :, :c["grouptop"]]
        none = best[:, :, 0] == -math.inf
        group = torch.where(best == -math.inf, 0.0, best).sum(2)
        group = torch.where(none, -math.inf, group)
        kept = torch.sort(group, dim=1, descending=True, stable=True).indices[:, :c["topgroups"]]
        mask = torch.zeros((T, G), dtype=torch.bool, device=x.device).scatter_(1, kept, True)
        key = torch.where(mask.repeat_interleave(E // G, dim=1), key, -math.inf)
    pick = torch.sort(key, dim=1, descending=True, stable=True).indices[:, :c["k"]]
    w = torch.where(key.gather(1, pick) > -math.inf, score.gather(1, pick), 0.0)
    if c["renorm"]:
        w = w / w.sum(1, keepdim=True).clamp_min(1e-300)
    pjc = torch.arange(0, T * c["k"] + 1, c["k"], dtype=torch.int32, device=x.device)
    pic = torch.arange(T, dtype=torch.int32, device=x.device).repeat_interleave(c["k"])
    return pick.to(torch.int32).reshape(-1), pic, pjc, (w * c["scale"]).float().reshape(-1)


def _plain_route_grad(s):
    c, x = s["case"], s["x"]
    T, E = x.shape
    pick = s["pir"].view(T, -1).long()
    w = s["weights"].view(T, -1)
    g = s["dweights"].view(T, -1)
    d = (w * g).sum(1, keepdim=True)
    if c["renorm"]:
        v = w * (g - d / c["scale"])
    else:
        v = w * g
    if c["score"] == "sigmoid":
        v = v / (1.0 + torch.exp(x.float().gather(1, pick)))
    if c["score"] == "softmax" and not c["renorm"]:
        xf = x.float()
        e = torch.exp(xf - xf.amax(1, keepdim=True))
        out = e / e.sum(1, keepdim=True) * -d
    else:
        out = torch.zeros((T, E), device=x.device)
    return out.scatter_add_(1, pick, v).to(x.dtype)


def _plain_lse(x, temperature):
    top = x.float().amax(1, keepdim=True)
    return (top[:, 0] / temperature) + torch.log(torch.exp((x.float() - top) / temperature).sum(1))


def _plain_top(s):
    c, x = s["case"], s["x"]
    T, V = x.shape
    k = min(c["k"], V)
    # one whole number per entry: the value's order above, the lower row first below
    b = (x.float() + 0.0).view(torch.int32).long()      # the sum makes one zero of the two
    b = torch.where(b < 0, b ^ 0x7FFFFFFF, b)
    b = (b << 32) + (0x7FFFFFFF - torch.arange(V, device=x.device))
    pick = 0x7FFFFFFF - (b.topk(k, dim=1).values & 0xFFFFFFFF)
    pjc = torch.arange(0, T * k + 1, k, dtype=torch.int32, device=x.device)
    pic = torch.arange(T, dtype=torch.int32, device=x.device).repeat_interleave(k)
    out = [pick.to(torch.int32).reshape(-1), pic, pjc, x.gather(1, pick).float().reshape(-1)]
    if c["lse"]:
        out.append(_plain_lse(x, c["temperature"]))
    return tuple(out)


def _plain_teacher(s, tau, T):
    """The teacher's probabilities per entry, their sum and log-sum-exp per token (zero without entries)."""
    ic = s["pic"].long()
    z = s["pdata"] / tau
    if s["tlse"] is None:
        top = torch.full((T,), -math.inf, device=z.device).scatter_reduce_(0, ic, z, "amax")
        tot = torch.zeros(T, device=z.device).index_add_(0, ic, torch.exp(z - top[ic]))
        lt = torch.where(tot > 0, top + torch.log(tot), 0.0)
    else:
        lt = s["tlse"]
    p = torch.exp(z - lt[ic])
    return ic, z, lt, p, torch.zeros(T, device=z.device).index_add_(0, ic, p)


def _plain_distill(s, ls):
    c, x = s["case"], s["x"]
    tau = c["temperature"]
    ic, z, lt, p, P = _plain_teacher(s, tau, x.shape[0])
    xr = x[ic, s["pir"].long()].float() / tau
    return torch.zeros_like(P).index_add_(0, ic, p * (z - xr)) + torch.where(P > 0, P * (ls - lt), 0.0)


def _plain_distill_grad(s, ls):
    c, x = s["case"], s["x"]
    tau = c["temperature"]
    ic, z, lt, p, P = _plain_teacher(s, tau, x.shape[0])
    w = s["weights"] / tau
    out = x.float().mul_(1.0 / tau) if x.dtype != torch.float32 else x / tau
    out.sub_(ls[:, None]).exp_().mul_((P * w)[:, None])
    out.index_put_((ic, s["pir"].long()), -p * w[ic], accumulate=True)
    return out.to(x.dtype)


def _run_plain(s):
    op = s["case"]["op"]
    if op == "route":
        return _plain_route(s)
    if op == "route_grad":
        return _plain_route_grad(s)
    if op == "top":
        return _plain_top(s)
    if op == "distill":
        ls = _plain_lse(s["x"], s["case"]["temperature"])
        return _plain_distill(s, ls), ls
    if op == "distill_grad":
        return _plain_distill_grad(s, s["slse"])
    ls = _plain_lse(s["x"], s["case"]["temperature"])
    return s["weights"] * _plain_distill(s, ls), _plain_distill_grad(s, ls)


# ---------------------------------------------------------------------------------------- the package's operators

def _run_own(s):
    from bidmat_b200 import tokens
    from bidmat_b200.mat import GHMat, GMat, GSMat

    c = s["case"]
    x = s["x"]
    T, V = x.shape
    X = GMat(x) if x.dtype == torch.float32 else GHMat(x)
    op = c["op"]
    if op == "route":
        bias = None if s["bias"] is None else GMat(s["bias"].view(1, V))
        S = tokens.route(X, c["k"], score=c["score"], bias=bias, groups=c["groups"], topgroups=c["topgroups"],
                         grouptop=c["grouptop"], renorm=c["renorm"], scale=c["scale"])
        return S.pir, S.pic, S.pjc, S.pdata
    if op == "route_grad":
        nnz = s["pir"].numel()
        S = GSMat(V, T, nnz, s["pir"], s["pic"], s["pjc"], s["weights"])
        dS = GSMat(V, T, nnz, s["pir"], s["pic"], s["pjc"], s["dweights"])
        return tokens.routeGrad(X, S, dS, score=c["score"], renorm=c["renorm"], scale=c["scale"]).t
    if op == "top":
        lse = GMat(torch.empty((T, 1), device=x.device)) if c["lse"] else None
        S = tokens.topLogits(X, min(c["k"], V), temperature=c["temperature"], lse=lse)
        out = (S.pir, S.pic, S.pjc, S.pdata)
        return out + (lse.t.view(T),) if c["lse"] else out
    Z = GSMat(V, T, s["pir"].numel(), s["pir"], s["pic"], s["pjc"], s["pdata"])
    tl = None if s["tlse"] is None else GMat(s["tlse"].view(T, 1))
    if op == "distill":
        loss, ls = tokens.distill(X, Z, temperature=c["temperature"], lse=tl)
        return loss.t.view(T), ls.t.view(T)
    w = GMat(s["weights"].view(T, 1))
    if op == "distill_grad":
        return tokens.distillGrad(X, Z, GMat(s["slse"].view(T, 1)), weights=w, temperature=c["temperature"], lse=tl).t
    loss, dX = tokens.distillWithGrad(X, Z, weights=w, temperature=c["temperature"], lse=tl)
    return loss.t.view(T), dX.t


def run(state):
    return _run_own(state) if own else _run_plain(state)


# ---------------------------------------------------------------------------------------- what a pass cannot do without

def work(case):
    V, T, k, es = case["rows"], case["cols"], min(case["k"], case["rows"]), _SIZE[case["dtype"]]
    dense = V * T
    op = case["op"]
    if op == "route":
        return {"bytes": dense * es + 12 * k * T + 4 * (T + 1) + (4 * V if case["bias"] else 0), "flops": 4 * dense}
    if op == "route_grad":
        whole = case["score"] == "softmax" and not case["renorm"]
        read = dense * es if whole else (k * T * es if case["score"] == "sigmoid" else 0)
        return {"bytes": read + dense * es + 12 * k * T + 4 * (T + 1), "flops": (4 * dense if whole else 0) + 6 * k * T}
    if op == "top":
        return {"bytes": dense * es + 12 * k * T + 4 * (T + 1) + (4 * T if case["lse"] else 0),
                "flops": (4 if case["lse"] else 1) * dense}
    # a tenth of the tokens has no entries, three tenths of the others have half of k on average
    entries = int(0.765 * k * T)
    teacher = 8 * entries + 4 * (T + 1) + (4 * T if case["lse"] else 0)
    if op == "distill":
        return {"bytes": dense * es + teacher + 8 * T, "flops": 3 * dense + 8 * entries}
    if op == "distill_grad":
        return {"bytes": 2 * dense * es + teacher + 8 * T, "flops": 3 * dense + 6 * entries}
    return {"bytes": 2 * dense * es + teacher + 8 * T, "flops": 6 * dense + 14 * entries}


# ---------------------------------------------------------------------------------------- the definitions in 64 bits

def _exact_route(s):
    """Expert by expert: the best remaining one is taken k times."""
    import numpy as np

    c = s["case"]
    x = s["x"].double().cpu().numpy()
    T, E = x.shape
    with np.errstate(over="ignore", invalid="ignore", divide="ignore"):
        if c["score"] == "softmax":
            m = x.max(axis=1, keepdims=True)
            p = np.exp(x - np.where(np.isfinite(m), m, 0.0))
            p /= np.maximum(p.sum(axis=1, keepdims=True), 1e-300)
        else:
            p = np.where(x >= 0, 1.0 / (1.0 + np.exp(-np.abs(x))), np.exp(-np.abs(x)) / (1.0 + np.exp(-np.abs(x))))
    b = np.zeros(E) if s["bias"] is None else s["bias"].double().cpu().numpy()
    order = x.copy() if s["bias"] is None else np.where(np.isneginf(x), -np.inf, p + b)
    G = c["groups"]
    every = np.arange(T)
    if G > 1:
        size = E // G
        cand = np.where(np.isneginf(x), -np.inf, p + b)
        value = np.empty((T, G))
        for j in range(G):
            part = cand[:, j * size:(j + 1) * size]
            hi = part.max(axis=1)
            value[:, j] = hi
            if c["grouptop"] == 2 and size > 1:
                part = part.copy()
                part[every, part.argmax(axis=1)] = -np.inf
                second = part.max(axis=1)
                value[:, j] = np.where(np.isneginf(second), hi, hi + second)
        kept = np.zeros((T, G), dtype=bool)
        for _ in range(c["topgroups"]):
            left = np.where(kept, -np.inf, value)
            j = left.argmax(axis=1)
            # among groups without any expert the first that is not yet kept
            j = np.where(np.isneginf(left[every, j]), kept.argmin(axis=1), j)
            kept[every, j] = True
        order = np.where(np.repeat(kept, size, axis=1), order, -np.inf)
    taken = np.zeros((T, E), dtype=bool)
    pir = np.empty((T, c["k"]), dtype=np.int32)
    w = np.zeros((T, c["k"]))
    for i in range(c["k"]):
        left = np.where(taken, -np.inf, order)
        j = left.argmax(axis=1)
        out = np.isneginf(left[every, j])
        j = np.where(out, taken.argmin(axis=1), j)
        taken[every, j] = True
        pir[:, i] = j
        w[:, i] = np.where(out, 0.0, p[every, j])
    if c["renorm"]:
        w /= np.maximum(w.sum(axis=1, keepdims=True), 1e-300)
    pjc = np.arange(T + 1, dtype=np.int32) * c["k"]
    pic = np.repeat(np.arange(T, dtype=np.int32), c["k"])
    return tuple(torch.from_numpy(a).cuda() for a in (pir.reshape(-1), pic, pjc, (w * c["scale"]).reshape(-1)))


def _exact_route_grad(s):
    """The weights' Jacobian applied column by column, from the scores themselves."""
    c, x = s["case"], s["x"].double()
    T = x.shape[0]
    pick = s["pir"].view(T, -1).long()
    g = s["dweights"].view(T, -1).double()
    w = s["weights"].view(T, -1).double()
    out = torch.zeros_like(x)
    if c["score"] == "softmax" and c["renorm"]:
        out.scatter_add_(1, pick, w * g - w * (w * g).sum(1, keepdim=True) / c["scale"])
    elif c["score"] == "softmax":
        p = torch.softmax(x, 1)
        up = torch.zeros_like(x).scatter_add_(1, pick, w * g)
        out = up - p * up.sum(1, keepdim=True)
    else:
        rest = torch.sigmoid(-x.gather(1, pick))
        if c["renorm"]:
            g = g - (w * g).sum(1, keepdim=True) / c["scale"]
        out.scatter_add_(1, pick, w * rest * g)
    return out


def _exact_top(s):
    c, x = s["case"], s["x"]
    T, V = x.shape
    k = min(c["k"], V)
    pir, val, lse = [], [], []
    for t in range(0, T, 64):
        d = x[t:t + 64].double()
        v, i = torch.sort(d, dim=1, descending=True, stable=True)
        pir.append(i[:, :k].to(torch.int32))
        val.append(v[:, :k])
        if c["lse"]:
            lse.append(torch.logsumexp(d / c["temperature"], 1))
    pjc = torch.arange(T + 1, dtype=torch.int32, device=x.device) * k
    pic = torch.arange(T, dtype=torch.int32, device=x.device)[:, None].expand(T, k).reshape(-1)
    out = (torch.cat(pir).reshape(-1), pic, pjc, torch.cat(val).reshape(-1))
    return out + (torch.cat(lse),) if c["lse"] else out


def _exact_distill(s, op):
    c, x = s["case"], s["x"]
    tau = c["temperature"]
    T, V = x.shape
    pjc = s["pjc"].tolist()
    loss, lses, grads = [], [], []
    for t in range(0, T, 64):
        u = min(T, t + 64)
        xs = x[t:u].double() / tau
        e0, e1 = pjc[t], pjc[u]
        at = (s["pic"][e0:e1].long() - t, s["pir"][e0:e1].long())
        # the teacher as dense columns: log probabilities, -inf where it says nothing
        z = torch.full_like(xs, -math.inf)
        z[at] = s["pdata"][e0:e1].double() / tau
        some = (z > -math.inf).any(1, keepdim=True)
        lt = torch.logsumexp(z, 1, keepdim=True) if s["tlse"] is None else s["tlse"][t:u, None].double()
        logp = torch.where(some, z - lt, -math.inf)
        p = torch.exp(logp)
        ls = torch.logsumexp(xs, 1, keepdim=True)
        if op == "distill_grad":
            ls = s["slse"][t:u, None].double()
        logq = xs - ls
        if op != "distill_grad":
            loss.append(torch.where(p > 0, p * (logp - logq), 0.0).sum(1))
            lses.append(ls[:, 0])
        if op != "distill":
            w = s["weights"][t:u, None].double() / tau
            grads.append(w * (p.sum(1, keepdim=True) * torch.exp(logq) - p))
    if op == "distill":
        return torch.cat(loss), torch.cat(lses)
    if op == "distill_grad":
        return torch.cat(grads)
    return s["weights"].double() * torch.cat(loss), torch.cat(grads)


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "route":
        return _exact_route(s)
    if case["op"] == "route_grad":
        return _exact_route_grad(s)
    if case["op"] == "top":
        return _exact_top(s)
    return _exact_distill(s, case["op"])
