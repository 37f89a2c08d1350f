"""Routing, top logits and distillation against their definitions in 64 bits (tokens_oracle).

Tolerances, fixed before the first run.  u = 2^-24 is half a step of fp32, h half a step of the output type.
  weights       |err| <= (16 + 2 max|x|) u |w|: the exponent's argument is off by at most 2 u max|x|, the rest
                is a handful of roundings
  log-sum-exp   |err| <= u (|L| + 2 range/t + V/256 + 16): the same for the exponents, and sums of V/512 terms
                or fewer per thread, twice that for joining them
  loss          |err| <= P * (the log-sum-exp's) + 4 u |loss| + 4 u: the entries are computed in 64 bits
  gradient      |err| <= |w|/t P q (the log-sum-exp's, relative, + 8 u + u |x|/t) + 4 u |w|/t p + h |grad| (+ half
                the smallest fp16)
Whole numbers, and logits that are passed through, have to be equal."""
import math

import numpy as np
import pytest
import torch

import tokens_oracle as oracle64
from bidmat_b200 import _lib, tokens
from bidmat_b200.mat import DDS, GHMat, GMat, GSMat, Mat

pytestmark = pytest.mark.gpu
U = 2.0 ** -24
DT = {"fp32": torch.float32, "bf16": torch.bfloat16, "fp16": torch.float16}
HALF = {n: torch.finfo(t).eps / 2 for n, t in DT.items()}          # a rounding, relative to the value
# half the smallest fp16; below 2^-126 an exponential leaves fp32's range and becomes 0, which is off by less than 2^-126
TINY = {"fp32": 2.0 ** -126, "bf16": 2.0 ** -126, "fp16": 2.0 ** -25}


def dense(a, dtype, device, pad=0):
    """A matrix object over `a` (ncols, nrows); pad > 0 puts that many foreign elements between columns."""
    t = torch.as_tensor(np.asarray(a), device=device).to(DT[dtype])
    if dtype == "fp32":
        return GMat(t.contiguous())
    if pad:
        wide = torch.full((t.shape[0], t.shape[1] + pad), float("nan"), dtype=t.dtype, device=device)
        wide[:, :t.shape[1]] = t
        return GHMat(wide[:, :t.shape[1]])
    return GHMat(t.contiguous())


def host(t):
    return t.float().cpu().numpy().astype(np.float64)


def row(v, device):
    return None if v is None else GMat(torch.as_tensor(np.asarray(v, np.float32), device=device).view(-1, 1))


def sparse(V, T, jc, ir, data, device):
    return GSMat.from_csc(V, T, torch.as_tensor(np.asarray(jc, np.int32), device=device),
                          torch.as_tensor(np.asarray(ir, np.int32), device=device),
                          torch.as_tensor(np.asarray(data, np.float32), device=device))


def close(got, want, tol, what):
    got, want, tol = (np.asarray(v, np.float64) for v in (got, want, tol))
    want = np.where(np.abs(want) > np.finfo(np.float32).max, np.copysign(np.inf, want), want)      # no number of fp32
    same = (np.isnan(got) & np.isnan(want)) | (got == want)
    with np.errstate(invalid="ignore"):
        bad = ~same & ~(np.abs(got - want) <= tol)
    if bad.any():
        i = tuple(int(v[0]) for v in np.nonzero(bad))
        raise AssertionError("%s: %d of %d outside, first at %s: got %r want %r tolerance %r"
                             % (what, bad.sum(), bad.size, i, got[i], want[i], np.broadcast_to(tol, got.shape)[i]))


def same_bits(a, b):
    return torch.equal(a.contiguous().view(torch.uint8), b.contiguous().view(torch.uint8))


# ------------------------------------------------------------------------------------------ routing

def check_route(x, dtype, device, k, score="softmax", bias=None, groups=1, topgroups=1, grouptop=2, renorm=True,
                scale=1.0, pad=0):
    X = dense(x, dtype, device, pad)
    xs = host(X.t)
    b = None if bias is None else GMat(torch.as_tensor(np.asarray(bias, np.float32), device=device).view(1, -1))
    S = tokens.route(X, k, score=score, bias=b, groups=groups, topgroups=topgroups, grouptop=grouptop, renorm=renorm,
                     scale=scale)
    T = xs.shape[0]
    pir, w = oracle64.route(xs, k, score, None if b is None else b.t.cpu().numpy()[0], groups, topgroups, grouptop, renorm,
                            np.float32(scale))
    assert np.array_equal(S.pjc.cpu().numpy(), np.arange(T + 1) * k)
    assert np.array_equal(S.pic.cpu().numpy(), np.repeat(np.arange(T), k))
    got = S.pir.cpu().numpy().reshape(T, k)
    assert np.array_equal(got, pir), (np.argwhere((got != pir).any(1))[:3], got[(got != pir).any(1)][:2],
                                      pir[(got != pir).any(1)][:2])
    finite = np.abs(np.where(np.isfinite(xs), xs, 0)).max()
    close(S.pdata.cpu().numpy().reshape(T, k), w, (16 + 2 * finite) * U * np.abs(w) + 2.0 ** -149, "weights")
    return X, S


@pytest.mark.parametrize("dtype", ["fp32", "bf16", "fp16"])
@pytest.mark.parametrize("E,T,k", [(1, 1, 1), (2, 5, 2), (7, 33, 3), (8, 64, 8), (33, 4, 5), (64, 4, 6), (65, 130, 9),
                                   (160, 257, 6), (256, 97, 8), (300, 31, 32), (1023, 9, 17), (1024, 40, 32)])
def test_route_sizes_and_types(cuda_device, dtype, E, T, k):
    rng = np.random.default_rng(E * 1000 + T)
    x = 1.5 * rng.standard_normal((T, E))
    for score in ("softmax", "sigmoid"):
        for renorm in (True, False):
            check_route(x, dtype, cuda_device, k, score=score, renorm=renorm, scale=2.5, pad=3)
            check_route(x, dtype, cuda_device, k, score=score, renorm=renorm, bias=0.1 * rng.standard_normal(E))


@pytest.mark.parametrize("E,groups,topgroups,grouptop,k", [(256, 8, 4, 2, 8), (256, 8, 4, 1, 8), (160, 8, 3, 1, 6), (12, 4, 1, 2, 3),
                                                           (12, 12, 5, 2, 5), (1024, 64, 7, 2, 32), (1024, 1024, 3, 1, 3),
                                                           (30, 3, 3, 2, 4), (6, 2, 1, 1, 3)])
@pytest.mark.parametrize("dtype", ["fp32", "bf16"])
def test_route_groups(cuda_device, dtype, E, groups, topgroups, grouptop, k):
    rng = np.random.default_rng(E + groups)
    x = 2.0 * rng.standard_normal((70, E))
    x[3] = -np.inf
    x[4, : E // 2] = -np.inf
    x[5] = -np.inf
    x[5, E - 1] = 0.25
    for score in ("softmax", "sigmoid"):
        for bias in (None, 0.2 * rng.standard_normal(E)):
            check_route(x, dtype, cuda_device, k, score=score, bias=bias, groups=groups, topgroups=topgroups, grouptop=grouptop)


@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
@pytest.mark.parametrize("biased", [False, True])
def test_route_ties_and_near_ties(cuda_device, score, biased):
    """Equal scores go by row; scores that fp32 cannot tell apart after the bias has been added still do not
    change places."""
    rng = np.random.default_rng(5)
    x = np.round(2.0 * rng.standard_normal((200, 96)) * 2) / 2               # many equal scores
    x[0] = 0.0
    x[1] = np.nextafter(np.float32(1.0), np.float32(2.0))
    x[1, 50] = 1.0
    base = np.float32(rng.standard_normal(100))
    y = np.repeat(base[:, None], 96, axis=1).astype(np.float32)              # columns of neighbours in fp32
    steps = rng.integers(-3, 4, size=y.shape)
    for s in range(1, 4):
        y = np.where(np.abs(steps) >= s, np.nextafter(y, np.where(steps > 0, np.inf, -np.inf).astype(np.float32)), y)
    x = np.concatenate([x, y])
    bias = np.where(np.arange(96) % 2 == 0, 0.25, 0.25) if biased else None
    check_route(x, "fp32", cuda_device, 12, score=score, bias=bias)
    check_route(x, "fp32", cuda_device, 12, score=score, bias=bias, groups=8, topgroups=4, renorm=False)
    if biased:
        # exact sums that differ by less than a step of fp32: s + b where b carries the opposite of most of s
        z = rng.standard_normal((64, 32))
        p = (np.exp(z) / np.exp(z).sum(1, keepdims=True) if score == "softmax" else 1 / (1 + np.exp(-z)))
        check_route(z.astype(np.float32), "fp32", cuda_device, 8, score=score, bias=(0.5 - p[7]).astype(np.float32))


@pytest.mark.parametrize("dtype", ["fp32", "bf16"])
@pytest.mark.parametrize("E,k", [(256, 8), (160, 6), (64, 3), (512, 8), (1024, 32), (256, 31)])
def test_route_columns_in_bad_orders(cuda_device, dtype, E, k):
    """Columns whose largest scores lie where few lanes have them, constant ones, and ones with fewer rows than picks."""
    rng = np.random.default_rng(E + k)
    x = rng.standard_normal((24, E))
    x[0] = 0.0                                                  # a mixture before its first step
    x[1] = np.round(x[1])
    x[2] = np.linspace(-3, 3, E)
    x[3] = np.linspace(3, -3, E)
    for i, m in enumerate((4, 8, 16, 32, 64)):
        x[4 + i, ::m] += 10.0
    x[9, : E // 2] += 10.0
    x[10, 8:16] += 10.0
    x[11] = np.where(np.arange(E) % 2 == 0, 1.0, -1.0)
    x[12, k - 1:] = -np.inf
    x[13, :-1] = -np.inf
    x[14] = -np.inf
    x[15] = 1.0
    x[15, 5] = 2.0
    x[16] = np.repeat(rng.standard_normal(E // 4), 4)
    bias = 0.1 * rng.standard_normal(E)
    for b in (None, bias, np.zeros(E)):
        for score in ("softmax", "sigmoid"):
            check_route(x, dtype, cuda_device, k, score=score, bias=b)
            check_route(x, dtype, cuda_device, k, score=score, bias=b, groups=8, topgroups=4, renorm=False)
            check_route(x, dtype, cuda_device, k, score=score, bias=b, groups=4, topgroups=2, grouptop=1)


def test_route_masks_infinities_and_nan(cuda_device):
    rng = np.random.default_rng(8)
    x = rng.standard_normal((40, 48)).astype(np.float32)
    low = np.finfo(np.float32).min
    x[0] = -np.inf
    x[1, 5:] = -np.inf
    x[2, 3] = np.nan
    x[3, 40] = np.inf
    x[4] = low
    x[5, 7:] = low
    x[6] = np.nan
    x[7] = 88.0 * np.sign(x[7])
    x[8] = -1000.0
    x[9] = np.linspace(-300, 300, 48)
    bias = 0.1 * rng.standard_normal(48)
    off = bias.copy()
    off[::2] = -np.inf
    off[1] = np.nan
    for b in (None, bias, off):
        for renorm in (True, False):
            check_route(x, "fp32", cuda_device, 8, score="softmax", bias=b, renorm=renorm, groups=4, topgroups=2)
            check_route(x, "fp32", cuda_device, 8, score="softmax", bias=b, renorm=renorm)
    # a sigmoid far below zero leaves the range of fp32: only finite weights are compared there
    x[4:10] = np.clip(x[4:10], -60, 60)
    for b in (None, bias, off):
        for renorm in (True, False):
            check_route(x, "fp32", cuda_device, 8, score="sigmoid", bias=b, renorm=renorm)


def grad_tolerance(x, S, w, g, want, renorm, scale, dtype):
    # D is a sum of at most 64 products, w and g are given: 70 u of the sum of absolute terms, and the exponent's 2 u max|x|
    T = x.shape[0]
    k = w.size // T
    mag = np.abs(w * g).reshape(T, k).sum(1, keepdims=True)
    finite = np.abs(np.where(np.isfinite(x), x, 0)).max()
    wmax = np.abs(w).reshape(T, k).max(1, keepdims=True) / (abs(scale) if renorm else 1.0)
    return (80 + 2 * finite) * U * (mag * np.maximum(wmax, 1.0) + np.abs(want)) + HALF[dtype] * np.abs(want) + TINY[dtype]


@pytest.mark.parametrize("dtype", ["fp32", "bf16", "fp16"])
@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
@pytest.mark.parametrize("renorm", [True, False])
def test_route_gradient_formula(cuda_device, dtype, score, renorm):
    for (E, T, k) in ((1, 3, 1), (5, 1, 2), (64, 4, 6), (97, 65, 32), (160, 300, 6), (256, 129, 8), (1024, 17, 8), (1001, 5, 3)):
        rng = np.random.default_rng(E + T)
        x = 1.5 * rng.standard_normal((T, E))
        if T > 2:
            x[2] = -np.inf
        X, S = check_route(x, dtype, cuda_device, k, score=score, renorm=renorm, scale=2.5, pad=5)
        dS = S.copy()
        dS.pdata = torch.as_tensor(rng.standard_normal(S.nnz).astype(np.float32), device=cuda_device)
        got = tokens.routeGrad(X, S, dS, score=score, renorm=renorm, scale=2.5)
        w, g = host(S.pdata), host(dS.pdata)
        want = oracle64.route_grad(host(X.t), S.pjc.cpu().numpy(), S.pir.cpu().numpy(), w, g, score, renorm, 2.5)
        close(host(got.t), want, grad_tolerance(host(X.t), S, w, g, want, renorm, 2.5, dtype), "routeGrad %d" % E)
        again = tokens.routeGrad(X, S, dS, score=score, renorm=renorm, scale=2.5)
        assert torch.equal(got.t, again.t)
        same = tokens.routeGrad(X, S, dS, score=score, renorm=renorm, scale=2.5, omat=X)     # in place
        assert same is X and torch.equal(X.t, got.t)


@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
@pytest.mark.parametrize("renorm", [True, False])
def test_route_gradient_against_differences(cuda_device, score, renorm):
    """Central differences of sum g * weights in 64 bits with the picks held: step 1e-4, third derivatives of
    order scale, so off by about 1e-8 * |g| * k, plus the kernel's own tolerance."""
    rng = np.random.default_rng(3)
    x = np.float32(rng.standard_normal((6, 20))).astype(np.float64)
    X, S = check_route(x, "fp32", cuda_device, 4, score=score, renorm=renorm, scale=1.5)
    dS = S.copy()
    g = rng.standard_normal(S.nnz).astype(np.float32)
    dS.pdata = torch.as_tensor(g, device=cuda_device)
    got = host(tokens.routeGrad(X, S, dS, score=score, renorm=renorm, scale=1.5).t)
    pir = S.pir.cpu().numpy().reshape(6, 4)

    def value(y):
        s = np.exp(y - y.max()) / np.exp(y - y.max()).sum() if score == "softmax" else 1 / (1 + np.exp(-y))
        return s

    want = np.zeros_like(x)
    for t in range(6):
        for e in range(20):
            f = []
            for d in (1e-4, -1e-4):
                y = x[t].copy()
                y[e] += d
                w = value(y)[pir[t]]
                f.append(1.5 * (w / w.sum() if renorm else w) @ g.reshape(6, 4)[t])
            want[t, e] = (f[0] - f[1]) / 2e-4
    close(got, want, 1e-7 * 4 * np.abs(g).max() + 100 * U, "routeGrad against differences")


def test_route_gradient_of_any_sparse_matrix(cuda_device):
    """Columns of any length, rows twice, rows outside: added up in order, left out."""
    rng = np.random.default_rng(4)
    E, counts = 50, [0, 1, 40, 100, 3, 0, 33]
    jc = np.concatenate([[0], np.cumsum(counts)]).astype(np.int32)
    ir = rng.integers(0, E, jc[-1]).astype(np.int32)
    ir[5], ir[60] = -1, E
    w = rng.uniform(0.1, 1.0, jc[-1]).astype(np.float32)
    g = rng.standard_normal(jc[-1]).astype(np.float32)
    x = rng.standard_normal((len(counts), E)).astype(np.float32)
    X = GMat(torch.as_tensor(x, device=cuda_device))
    S, dS = sparse(E, len(counts), jc, ir, w, cuda_device), sparse(E, len(counts), jc, ir, g, cuda_device)
    for score in ("softmax", "sigmoid"):
        for renorm in (True, False):
            got = host(tokens.routeGrad(X, S, dS, score=score, renorm=renorm).t)
            want = oracle64.route_grad(x, jc, ir, w, g, score, renorm, 1.0)
            tol = 200 * U * np.abs(w * g).sum()
            close(got, want, tol, "routeGrad of a ragged matrix")


# ------------------------------------------------------------------------------------------ top logits

def lse_tolerance(x, L, tau):
    V = x.shape[1]
    # what is masked, be it by a value like the lowest of the type, has no part in the exponents' rounding
    f = np.where(np.abs(x) < 1e30, x, 0.0)
    span = (f.max(1) - f.min(1)) / tau
    return U * (np.abs(np.where(np.isfinite(L), L, 0.0)) + 2 * span + V / 256.0 + 16)


def check_top(x, dtype, device, k, tau=1.0, pad=0):
    X = dense(x, dtype, device, pad)
    xs = host(X.t)
    T, V = xs.shape
    lse = row(np.zeros(T), device)
    S = tokens.topLogits(X, k, temperature=tau, lse=lse)
    pir, val, L = oracle64.top(xs, k, tau)
    assert np.array_equal(S.pjc.cpu().numpy(), np.arange(T + 1) * k)
    assert np.array_equal(S.pic.cpu().numpy(), np.repeat(np.arange(T), k))
    got = S.pir.cpu().numpy().reshape(T, k)
    assert np.array_equal(got, pir), np.argwhere((got != pir).any(1))[:5]
    assert np.array_equal(S.pdata.cpu().numpy().reshape(T, k), val.astype(np.float32), equal_nan=True)
    close(lse.t.cpu().numpy()[:, 0], L, lse_tolerance(xs, L, tau), "log-sum-exp")
    assert np.array_equal(tokens.topLogits(X, k).pir.cpu().numpy().reshape(T, k), pir)       # without the log-sum-exp
    return X, S, lse


@pytest.mark.parametrize("dtype", ["fp32", "bf16", "fp16"])
@pytest.mark.parametrize("V,T,k", [(1, 1, 1), (2, 3, 2), (31, 5, 31), (512, 4, 512), (513, 3, 512), (1000, 9, 17), (4096, 2, 100),
                                   (8191, 3, 64), (32768, 1, 40), (50001, 5, 128), (131072, 2, 512), (100003, 3, 1),
                                   (300007, 2, 50), (500009, 1, 70)])
def test_top_sizes_and_types(cuda_device, dtype, V, T, k):
    rng = np.random.default_rng(V + T)
    check_top(2.0 * rng.standard_normal((T, V)), dtype, cuda_device, k, pad=0)
    check_top(2.0 * rng.standard_normal((T, V)), dtype, cuda_device, k, tau=2.0, pad=5)


@pytest.mark.parametrize("dtype", ["fp32", "bf16"])
@pytest.mark.parametrize("V", [700, 40000, 140000, 520001])
def test_top_of_columns_in_bad_orders(cuda_device, dtype, V):
    """Ascending, descending, constant, two values, one spike, masked, equal large values at the far end."""
    k = 100
    up = np.linspace(-4, 4, V)
    cols = [up, up[::-1], np.zeros(V), np.where(np.arange(V) % 3 == 0, 1.0, 0.0), np.full(V, -np.inf), np.full(V, -5.0)]
    cols[5][V - 1] = 7.0
    c = np.full(V, -np.inf)
    c[V // 2: V // 2 + 10] = np.arange(10)
    cols.append(c)
    c = np.full(V, np.finfo(np.float32).min if dtype == "fp32" else -3.0e38)
    c[::97] = -1.0
    cols.append(c)
    c = np.zeros(V)
    c[V - 150:] = 3.0
    cols.append(c)
    c = np.where(np.arange(V) % 2 == 0, 0.0, -0.0)
    cols.append(c)
    c = up.copy()
    c[: V // 2] = up[V // 2 - 1: None if V % 2 == 0 else V - 2: 1][: V // 2]
    cols.append(c)
    c = np.tile(np.arange(50.0), V // 50 + 1)[:V]
    cols.append(c)
    check_top(np.stack(cols), dtype, cuda_device, k)


def test_top_nan_and_infinity(cuda_device):
    rng = np.random.default_rng(1)
    x = rng.standard_normal((5, 3001)).astype(np.float32)
    x[0, 7] = np.nan
    x[0, 3000] = -np.nan
    x[1, 5:9] = np.inf
    x[2] = np.nan
    x[3, 100:] = np.nan
    X = GMat(torch.as_tensor(x, device=cuda_device))
    pir, val, L = oracle64.top(x, 40, 1.0)
    lse = row(np.zeros(5), cuda_device)
    S = tokens.topLogits(X, 40, lse=lse)
    assert np.array_equal(S.pir.cpu().numpy().reshape(5, 40), pir)
    assert np.array_equal(S.pdata.cpu().numpy().reshape(5, 40), val.astype(np.float32), equal_nan=True)
    got = lse.t.cpu().numpy()[:, 0]
    assert np.isnan(got[[0, 2, 3]]).all() and not np.isfinite(got[1]) and abs(got[4] - L[4]) < 1e-5


# ------------------------------------------------------------------------------------------ distillation

def teacher(rng, V, counts, spread=2.5):
    jc = np.concatenate([[0], np.cumsum(counts)]).astype(np.int32)
    ir = np.concatenate([rng.permutation(V)[:n] for n in counts] + [np.zeros(0)]).astype(np.int32)
    return jc, ir, (6 + spread * rng.standard_normal(jc[-1])).astype(np.float32)


def check_distill(x, jc, ir, z, dtype, device, tau=1.0, tlse=None, weights=None, pad=0):
    X = dense(x, dtype, device, pad)
    xs = host(X.t)
    T, V = xs.shape
    Z = sparse(V, T, jc, ir, z, device)
    tau32 = float(np.float32(tau))
    loss64, L64, grad64, P = oracle64.distill(xs, jc, ir, z, tau32, tlse, weights)
    plain64 = oracle64.distill(xs, jc, ir, z, tau32, tlse)
    ltol = lse_tolerance(xs, L64, tau32)
    loss, L = tokens.distill(X, Z, temperature=tau, lse=row(tlse, device))
    close(L.t.cpu().numpy()[:, 0], L64, ltol, "log-sum-exp")
    close(loss.t.cpu().numpy()[:, 0], plain64[0], plain64[3] * ltol + 4 * U * (1 + np.abs(plain64[0])), "loss")
    w = np.ones(T) if weights is None else np.asarray(weights, np.float64)

    def gtol(g, rel):
        dense_part = np.abs(g) + 0.0
        p = np.zeros((T, V))
        for t in range(T):
            r = ir[jc[t]:jc[t + 1]]
            ok = (r >= 0) & (r < V)
            p[t, r[ok]] = np.abs(w[t]) / tau32 * P[t]
        f = np.abs(np.where(np.abs(xs) < 1e30, xs, 0)).max() / tau32
        return np.nan_to_num((dense_part + p) * (rel[:, None] + 8 * U + U * f) + 4 * U * p + HALF[dtype] * np.abs(g)) \
            + TINY[dtype] * (1 + np.nan_to_num(np.abs(w) / tau32 * P)[:, None])

    wl, dX = tokens.distillWithGrad(X, Z, weights=row(weights, device), temperature=tau, lse=row(tlse, device))
    close(wl.t.cpu().numpy()[:, 0], w * np.where(w == 0, 0, loss64), np.abs(w) * (P * ltol + 4 * U * (1 + np.abs(loss64))), "weighted loss")
    close(host(dX.t), grad64, gtol(grad64, ltol), "gradient of the fused pass")
    # the gradient from the saved log-sum-exp: compared with the formula at that saved value
    saved = host(L.t)[:, 0]
    g2 = oracle64.distill(xs, jc, ir, z, tau32, tlse, weights, slse=saved)[2]
    dX2 = tokens.distillGrad(X, Z, L, weights=row(weights, device), temperature=tau, lse=row(tlse, device))
    close(host(dX2.t), g2, gtol(g2, 4 * U * (1 + np.abs(np.where(np.isfinite(saved), saved, 0)))), "gradient from the saved pass")
    again = tokens.distillWithGrad(X, Z, weights=row(weights, device), temperature=tau, lse=row(tlse, device))
    assert same_bits(again[0].t, wl.t) and same_bits(again[1].t, dX.t)
    return X, Z, wl, dX


@pytest.mark.parametrize("dtype", ["fp32", "bf16", "fp16"])
@pytest.mark.parametrize("V,T,k", [(1, 1, 1), (3, 2, 3), (65, 7, 20), (1000, 3, 64), (1024, 2, 1000), (8192, 16, 20), (40001, 3, 100),
                                   (65536, 2, 64), (131072, 2, 64), (100003, 5, 7), (300007, 2, 50), (500009, 2, 60)])
def test_distill_sizes_and_types(cuda_device, dtype, V, T, k):
    rng = np.random.default_rng(V + 7 * T)
    counts = rng.integers(0, k + 1, T)
    counts[0] = k
    x = 2.0 * rng.standard_normal((T, V))
    jc, ir, z = teacher(rng, V, counts)
    for t in range(T):
        x[t, ir[jc[t]:jc[t + 1]]] = z[jc[t]:jc[t + 1]] + rng.standard_normal(counts[t])
    weights = rng.uniform(0.5, 2.0, T) * (1024.0 if dtype == "fp16" else 1.0)
    if T > 2:
        weights[1] = 0.0
    check_distill(x, jc, ir, z, dtype, cuda_device, tau=2.0, weights=np.float32(weights), pad=3)
    tlse = np.array([np.log(np.exp(z[jc[t]:jc[t + 1]].astype(np.float64)).sum()) + 0.2 if counts[t] else 1.0 for t in range(T)],
                    dtype=np.float32)
    check_distill(x, jc, ir, z, dtype, cuda_device, tau=1.0, tlse=tlse)


@pytest.mark.parametrize("dtype", ["fp32", "bf16", "fp16"])
@pytest.mark.parametrize("tau", [0.01, 0.3, 7.0, 500.0])
@pytest.mark.parametrize("V", [300, 20000, 70000])
def test_distill_temperatures_and_signs(cuda_device, dtype, tau, V):
    """Sharp and flat distributions, weights of both signs."""
    rng = np.random.default_rng(V)
    jc, ir, z = teacher(rng, V, [20, 1, 40])
    x = 2.0 * rng.standard_normal((3, V))
    for t in range(3):
        x[t, ir[jc[t]:jc[t + 1]]] = z[jc[t]:jc[t + 1]] + 0.2 * rng.standard_normal(jc[t + 1] - jc[t])
    check_distill(x, jc, ir, z, dtype, cuda_device, tau=tau, weights=np.float32([-tau, 0.5 * tau, -3.0 * tau]))


@pytest.mark.parametrize("dtype", ["fp32", "bf16"])
def test_distill_of_lowest_values_and_large_ones(cuda_device, dtype):
    """Columns masked with the lowest value, wholly or all but one row, and logits near the largest number: the
    distribution is the one of the differences."""
    V = 9000
    low = float(np.finfo(np.float32).min) if dtype == "fp32" else -3.3e38
    x = np.full((4, V), low)
    x[1, 17] = 0.0
    x[2] = 3.0e38 if dtype == "fp32" else 2.6e38
    x[3] = np.linspace(-1, 1, V)
    jc, ir, z = np.arange(0, 41, 10), np.tile(np.arange(10), 4).astype(np.int32), np.linspace(0, 1, 40).astype(np.float32)
    X = dense(x, dtype, cuda_device)
    Z = sparse(V, 4, jc, ir, z, cuda_device)
    loss, L = tokens.distill(X, Z)
    _, dX = tokens.distillWithGrad(X, Z)
    # from the differences: next to 3e38 a log-sum-exp loses its logarithm in 64 bits as well
    xs = host(X.t)
    d = np.exp(xs - xs.max(1, keepdims=True))
    want = d / d.sum(1, keepdims=True)
    for t in range(4):
        p = np.exp(z[jc[t]:jc[t + 1]].astype(np.float64))
        want[t, :10] -= p / p.sum()
    lse = xs.max(1) + np.log(d.sum(1))
    close(host(L.t)[:, 0], lse, 4 * U * np.abs(lse) + 64 * U, "log-sum-exp")
    close(host(dX.t), want, (HALF[dtype] + 64 * U) * np.abs(want) + 64 * U / 10, "gradient")


@pytest.mark.parametrize("dtype", ["fp32", "bf16", "fp16"])
@pytest.mark.parametrize("V,T,k", [(5, 3, 5), (999, 40, 64), (70001, 3, 700), (300007, 2, 5), (400003, 3, 300)])
def test_distill_gradient_in_place(cuda_device, dtype, V, T, k):
    rng = np.random.default_rng(V)
    jc, ir, z = teacher(rng, V, rng.integers(0, k + 1, T))
    ir[::7] = ir[0]                                    # rows twice
    Z = sparse(V, T, jc, ir, z, cuda_device)
    for pad in (0, 3):
        X = dense(rng.standard_normal((T, V)), dtype, cuda_device, pad)
        loss, want = tokens.distillWithGrad(X, Z, temperature=2.0)
        _, L = tokens.distill(X, Z, temperature=2.0)
        want2 = tokens.distillGrad(X, Z, L, temperature=2.0)
        Y = type(X)(X.t.clone(memory_format=torch.preserve_format))
        assert tokens.distillGrad(Y, Z, L, temperature=2.0, omat=Y) is Y and same_bits(Y.t, want2.t)
        loss2, dX = tokens.distillWithGrad(X, Z, temperature=2.0, omat=X)
        assert dX is X and same_bits(X.t, want.t) and same_bits(loss.t, loss2.t)


def test_distill_masks_and_infinities(cuda_device):
    rng = np.random.default_rng(12)
    V, n = 5003, 12
    low = float(np.finfo(np.float32).min)
    x = rng.standard_normal((n, V))
    jc, ir, z = teacher(rng, V, [30] * n)
    x[0, 4000:] = -np.inf
    x[1, :] = -np.inf
    x[2, 17] = np.nan
    x[3, 18] = np.inf
    x[4, 100:] = low
    x[5] = -np.inf
    x[5, ir[jc[5]:jc[6]]] = 1.0                       # only the teacher's rows are open
    z[jc[6]:jc[7]] = -np.inf                           # a teacher without a finite logit
    z[jc[7]:jc[7] + 5] = -np.inf
    x[8, ir[jc[8]]] = -np.inf                          # a row the teacher wants and the student forbids
    x[9] = 80.0 * np.sign(x[9])
    x[10] = low                                        # a mask of the lowest value that leaves nothing: uniform
    weights = np.ones(n, np.float32)
    weights[2] = 0.0                                   # the NaN column carries no weight
    check_distill(x, jc, ir, z, "fp32", cuda_device, weights=weights)
    check_distill(x, jc, ir, z, "bf16", cuda_device, tau=0.5)
    check_distill(x, jc, ir, z, "fp32", cuda_device, tlse=np.full(n, 12.0, np.float32))


def test_distill_rows_twice_and_rows_outside(cuda_device):
    rng = np.random.default_rng(13)
    V, counts = 2000, [50, 600, 1, 0, 1500, 7]
    jc = np.concatenate([[0], np.cumsum(counts)]).astype(np.int32)
    ir = rng.integers(0, V // 8, jc[-1]).astype(np.int32)          # most rows come several times
    z = rng.standard_normal(jc[-1]).astype(np.float32)
    x = rng.standard_normal((6, V))
    for dtype in ("fp32", "bf16"):
        check_distill(x, jc, ir, z, dtype, cuda_device)
    ir[3], ir[700] = V, -1
    X, Z, loss, dX = check_distill(x, jc, ir, z, "fp32", cuda_device)
    bad, good = [0, 4], [1, 2, 3, 5]                               # entry 700 belongs to column 4
    assert torch.isnan(loss.t[bad]).all() and torch.isnan(dX.t[bad]).all() and torch.isfinite(dX.t[good]).all()


def test_distill_without_entries(cuda_device):
    x = np.random.default_rng(2).standard_normal((4, 999))
    jc, none = np.zeros(5, np.int32), np.zeros(0, np.int32)
    X, Z, loss, dX = check_distill(x, jc, none, np.zeros(0, np.float32), "bf16", cuda_device)
    assert float(loss.t.abs().sum()) == 0.0 and float(dX.t.float().abs().sum()) == 0.0


def test_distill_gradient_against_differences(cuda_device):
    """Central differences of the loss in 64 bits, step 1e-4: off by the third derivative times 1e-8 / 6."""
    rng = np.random.default_rng(21)
    V, T, tau = 40, 3, 1.5
    x = rng.standard_normal((T, V)).astype(np.float32)
    jc, ir, z = teacher(rng, V, [10, 1, 6])
    w = np.float32([1.0, 0.5, -2.0])
    _, _, _, dX = check_distill(x, jc, ir, z, "fp32", cuda_device, tau=tau, weights=w)
    want = np.zeros((T, V))
    for t in range(T):
        for v in range(V):
            f = []
            for d in (1e-4, -1e-4):
                y = x.astype(np.float64)
                y[t, v] += d
                f.append(float(oracle64.distill(y, jc, ir, z, tau, None, w)[0][t]) * float(w[t]))
            want[t, v] = (f[0] - f[1]) / 2e-4
    close(host(dX.t), want, 1e-8 + 60 * U, "gradient against differences")


# ------------------------------------------------------------------------------------------ together, and around

def test_a_sparse_mixture_trains_through_the_products(cuda_device):
    """scores -> route -> A * S, and back: B.xT(S) for A, DDS for the weights, routeGrad for the scores; against
    64-bit automatic differentiation with the same picks.  Sums of at most 64 products per element in fp32:
    200 u of the largest sum of absolute terms."""
    rng = np.random.default_rng(30)
    E, T, k, d = 48, 70, 4, 32
    x = rng.standard_normal((T, E)).astype(np.float32)
    a = rng.standard_normal((E, d)).astype(np.float32)
    up = rng.standard_normal((T, d)).astype(np.float32)
    X, A, G = (GMat(torch.as_tensor(v, device=cuda_device)) for v in (x, a, up))
    for score, renorm in (("softmax", True), ("softmax", False), ("sigmoid", True), ("sigmoid", False)):
        S = tokens.route(X, k, score=score, renorm=renorm, scale=1.5)
        C = A * S
        dA = G.xT(S)
        dX = tokens.routeGrad(X, S, DDS(A, G, S), score=score, renorm=renorm, scale=1.5)
        tx = torch.tensor(x, dtype=torch.float64, requires_grad=True)
        ta = torch.tensor(a, dtype=torch.float64, requires_grad=True)
        s = torch.softmax(tx, 1) if score == "softmax" else torch.sigmoid(tx)
        pick = S.pir.cpu().long().view(T, k)
        w = s.gather(1, pick)
        w = 1.5 * (w / w.sum(1, keepdim=True) if renorm else w)
        out = torch.einsum("tk,tkd->td", w, ta[pick])
        out.backward(torch.tensor(up, dtype=torch.float64))
        for got, want, what in ((C.t, out.detach(), "A * S"), (dA.t, ta.grad, "gradient of A"), (dX.t, tx.grad, "gradient of X")):
            want = want.numpy()
            close(host(got), want, 200 * U * max(8.0, np.abs(want).max() * 8), what)
        by_expert = S.t                                        # the tokens of every expert
        jc = by_expert.pjc.cpu().numpy()
        assert np.array_equal(np.diff(jc), np.bincount(S.pir.cpu().numpy(), minlength=E))


def test_a_teacher_is_distilled_into_a_student(cuda_device):
    """topLogits of a teacher -> distillWithGrad of a student in bf16; the teacher itself has loss 0 on its
    own probabilities up to what its top leaves out."""
    rng = np.random.default_rng(31)
    T, V, k = 20, 5000, 50
    teach = GHMat(torch.as_tensor(3 * rng.standard_normal((T, V)), device=cuda_device).to(torch.bfloat16))
    stud = GHMat(torch.as_tensor(rng.standard_normal((T, V)), device=cuda_device).to(torch.bfloat16))
    lse = row(np.zeros(T), cuda_device)
    Z = tokens.topLogits(teach, k, lse=lse)
    jc, ir, z = Z.pjc.cpu().numpy(), Z.pir.cpu().numpy(), Z.pdata.cpu().numpy()
    check_distill(host(stud.t), jc, ir, z, "bf16", cuda_device, tlse=host(lse.t)[:, 0])
    loss, _ = tokens.distill(teach, Z, lse=lse)
    assert float(loss.t.abs().max()) <= 64 * U * 16          # p (log p - log p): two log-sum-exps of the same column
    loss, _ = tokens.distill(teach, Z)
    kept = torch.zeros(T, dtype=torch.float64).index_add_(0, Z.pic.cpu().long(),
                                                          torch.exp(Z.pdata.cpu().double() - lse.t.cpu().double()[Z.pic.cpu().long(), 0]))
    close(host(loss.t)[:, 0], -torch.log(kept).numpy(), 64 * U * 16, "loss of the renormalised top")


def test_calls_are_captured_and_replayed_with_new_inputs(cuda_device):
    rng = np.random.default_rng(40)
    T, V, E, k = 33, 9001, 64, 6
    xs = [torch.as_tensor(rng.standard_normal((T, V)), device=cuda_device).to(torch.bfloat16) for _ in range(3)]
    rs = [torch.as_tensor(rng.standard_normal((T, E)), device=cuda_device, dtype=torch.float32) for _ in range(3)]
    x, r = xs[0].clone(), rs[0].clone()

    def work():
        lse = GMat(torch.empty((T, 1), device=cuda_device))
        S = tokens.topLogits(GHMat(x), 20, lse=lse)
        loss, L = tokens.distill(GHMat(x), S, temperature=2.0)
        dX = tokens.distillGrad(GHMat(x), S, L, temperature=2.0)
        both = tokens.distillWithGrad(GHMat(x), S, lse=lse)
        R = tokens.route(GMat(r), k, groups=4, topgroups=2)
        dR = tokens.routeGrad(GMat(r), R, R, renorm=True)
        return [S.pir, S.pdata, lse.t, loss.t, L.t, dX.t, both[0].t, both[1].t, R.pir, R.pdata, dR.t]

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    graphs = []
    with torch.cuda.stream(side):
        work()
        side.synchronize()
        for _ in range(2):                                     # two graphs of the same calls live at once
            g = torch.cuda.CUDAGraph()
            with torch.cuda.graph(g, stream=side):
                out = work()
            graphs.append((g, out))
    torch.cuda.synchronize()
    for i in (1, 2):
        x.copy_(xs[i])
        r.copy_(rs[i])
        torch.cuda.synchronize()
        for g, _ in graphs:
            g.replay()
        torch.cuda.synchronize()
        want = work()
        torch.cuda.synchronize()
        for _, out in graphs:
            for p, q in zip(out, want):
                assert same_bits(p, q)


def test_calls_on_two_streams_at_once(cuda_device):
    rng = np.random.default_rng(41)
    xs = [torch.as_tensor(rng.standard_normal((64, 30011)), device=cuda_device).to(torch.bfloat16) for _ in range(2)]
    alone = []
    for x in xs:
        S = tokens.topLogits(GHMat(x), 64)
        alone.append((S, tokens.distillWithGrad(GHMat(x), S)))
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    got = [[], []]
    for _ in range(4):
        for i, st in enumerate(streams):
            with torch.cuda.stream(st):
                S = tokens.topLogits(GHMat(xs[i]), 64)
                got[i].append((S, tokens.distillWithGrad(GHMat(xs[i]), S)))
    torch.cuda.synchronize()
    for i in range(2):
        for S, (loss, dX) in got[i]:
            assert torch.equal(S.pir, alone[i][0].pir)
            assert torch.equal(loss.t, alone[i][1][0].t) and torch.equal(dX.t, alone[i][1][1].t)


def test_outputs_leave_their_surroundings_alone(cuda_device):
    """Rows between the columns of a strided output, and what lies before and behind every array."""
    rng = np.random.default_rng(42)
    T, V = 9, 1003
    for dtype in (torch.bfloat16, torch.float16):
        x = torch.as_tensor(rng.standard_normal((T, V)), device=cuda_device).to(dtype)
        wide = torch.full((T + 2, V + 13), 7.0, dtype=dtype, device=cuda_device)
        out = GHMat(wide[1:T + 1, 6:6 + V])
        Z = tokens.topLogits(GHMat(x), 30)
        ref = tokens.distillWithGrad(GHMat(x), Z)[1]
        tokens.distillWithGrad(GHMat(x), Z, omat=out)
        assert torch.equal(out.t, ref.t)
        mask = torch.ones_like(wide, dtype=torch.bool)
        mask[1:T + 1, 6:6 + V] = False
        assert bool((wide[mask] == 7.0).all())
        _, L = tokens.distill(GHMat(x), Z)
        ref = tokens.distillGrad(GHMat(x), Z, L)
        tokens.distillGrad(GHMat(x), Z, L, omat=out)
        assert torch.equal(out.t, ref.t) and bool((wide[mask] == 7.0).all())
        r = GHMat(x[:, :100])
        S = tokens.route(r, 5)
        out = GHMat(wide[1:T + 1, 6:106])
        tokens.routeGrad(r, S, S, omat=out)
        assert bool((wide[:, 6 + V:] == 7.0).all()) and bool((wide[0] == 7.0).all()) and bool((wide[T + 1] == 7.0).all())


def test_recycled_outputs_and_an_old_plan(cuda_device):
    """`omat` takes the new pattern; a transposed structure prepared for the old one is not used for it."""
    rng = np.random.default_rng(43)
    x1, x2 = (GMat(torch.as_tensor(rng.standard_normal((50, 24)), device=cuda_device, dtype=torch.float32)) for _ in range(2))
    B = GMat(torch.as_tensor(rng.standard_normal((50, 32)), device=cuda_device, dtype=torch.float32))
    S = tokens.route(x1, 3)
    S.prepareT(32)
    B.xT(S)
    S2 = tokens.route(x2, 3, omat=S)
    assert S2 is S
    fresh = tokens.route(x2, 3)
    assert torch.equal(S.pir, fresh.pir) and torch.equal(B.xT(S).t, B.xT(fresh).t)


def test_offsets_beyond_31_bits(cuda_device):
    """The last columns of a matrix of more than 2^31 elements equal the same columns alone."""
    V, T = 131072, 16500
    x = torch.zeros((T, V), dtype=torch.bfloat16, device=cuda_device)
    last = torch.randn((4, V), device=cuda_device).to(torch.bfloat16)
    x[T - 4:] = last
    X, Y = GHMat(x), GHMat(last)
    S, s = tokens.topLogits(X, 16), tokens.topLogits(Y, 16)
    assert torch.equal(S.pir[-64:], s.pir) and torch.equal(S.pir[:16].cpu(), torch.arange(16, dtype=torch.int32))
    loss, L = tokens.distill(X, S)
    l2, L2 = tokens.distill(Y, s)
    # a column alone may be split over more of the machine, so its sum may be in another order
    assert float((L.t[-4:] - L2.t).abs().max()) <= 2 * U * (16 + V / 256) and float((loss.t[-4:] - l2.t).abs().max()) <= 2 * U * (16 + V / 256)
    both = tokens.distillWithGrad(X, S)[1]
    want = tokens.distillWithGrad(Y, s)[1]
    diff = (both.t[-4:].float() - want.t.float()).abs()
    assert bool((diff <= 2 * HALF["bf16"] * want.t.float().abs() + 1e-9).all())
    del both
    g = tokens.distillGrad(X, S, L)
    assert bool(((g.t[-4:].float() - want.t.float()).abs() <= 2 * HALF["bf16"] * want.t.float().abs() + 1e-9).all())
    E = 1024
    T = (1 << 31) // E + 5
    xr = torch.zeros((T, E), dtype=torch.bfloat16, device=cuda_device)
    xr[-3:] = torch.randn((3, E), device=cuda_device).to(torch.bfloat16)
    R, r = tokens.route(GHMat(xr), 2), tokens.route(GHMat(xr[-3:].clone()), 2)
    assert torch.equal(R.pir[-6:], r.pir) and torch.equal(R.pdata[-6:], r.pdata)
    dR, dr = tokens.routeGrad(GHMat(xr), R, R), tokens.routeGrad(GHMat(xr[-3:].clone()), r, r)
    assert torch.equal(dR.t[-3:], dr.t)


def test_mirror_refuses_wrong_operands(cuda_device):
    f = torch.zeros((4, 64), device=cuda_device)
    X, H = GMat(f), GHMat(f.to(torch.bfloat16))
    S = tokens.route(X, 4)
    v = GMat(torch.zeros((4, 1), device=cuda_device))
    wrong = GMat(torch.zeros((5, 1), device=cuda_device))
    other = GSMat(63, 4, S.nnz, S.pir, S.pic, S.pjc, S.pdata)
    for call in (lambda: tokens.route(f, 4), lambda: tokens.route(X, 0), lambda: tokens.route(X, 65),
                 lambda: tokens.route(X, 33), lambda: tokens.route(X, 4, score="tanh"), lambda: tokens.route(X, 4, groups=7),
                 lambda: tokens.route(X, 9, groups=8, topgroups=1), lambda: tokens.route(X, 4, grouptop=3, groups=2),
                 lambda: tokens.route(X, 4, bias=v), lambda: tokens.route(X, 4, scale=0.0),
                 lambda: tokens.route(X, 4, scale=float("nan")), lambda: tokens.route(X, 5, omat=S),
                 lambda: tokens.routeGrad(X, other, S), lambda: tokens.routeGrad(X, S, tokens.route(X, 5)),
                 lambda: tokens.routeGrad(X, S, S, omat=H), lambda: tokens.routeGrad(X, f, S),
                 lambda: tokens.topLogits(X, 0), lambda: tokens.topLogits(X, 65), lambda: tokens.topLogits(X, 4, temperature=0.0),
                 lambda: tokens.topLogits(X, 4, lse=wrong), lambda: tokens.topLogits(S, 4),
                 lambda: tokens.distill(X, other), lambda: tokens.distill(X, S, lse=wrong),
                 lambda: tokens.distill(X, S, temperature=float("inf")), lambda: tokens.distillGrad(X, S, None),
                 lambda: tokens.distillGrad(X, S, v, weights=wrong), lambda: tokens.distillGrad(X, S, v, omat=H),
                 lambda: tokens.distillWithGrad(X, S, weights=wrong), lambda: tokens.distillWithGrad(X, f),
                 lambda: GHMat(f), lambda: GHMat(H.t.t()), lambda: GHMat(H.t.cpu()), lambda: GHMat(H.t[0])):
        with pytest.raises(RuntimeError):
            call()
    Mat.debugStructure = True
    try:
        S.pir[3] = 64
        with pytest.raises(RuntimeError):
            tokens.distill(X, S)
    finally:
        Mat.debugStructure = False
    none = GMat(torch.zeros((0, 64), device=cuda_device))
    E = tokens.route(none, 4)
    assert E.nnz == 0 and int(E.pjc[0]) == 0 and tokens.topLogits(none, 4).nnz == 0
    assert tokens.routeGrad(none, E, E).ncols == 0 and tokens.distill(none, E)[0].ncols == 0
    assert tokens.distillWithGrad(none, E)[1].ncols == 0
    assert math.isfinite(float(tokens.distill(X, tokens.topLogits(X, 3))[0].t.sum()))
    assert _lib.lib.bidmat_b200_launch_count() > 0
