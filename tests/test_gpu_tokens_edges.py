"""Corners of the operators on token columns: long lists, columns in place, large and masked values, near ties.

Against definitions in 64 bits (tokens_oracle), with the tolerances named at each test, where u = 2^-24 is half a
step of fp32 and h half a step of the output type (2^-24 fp32, 2^-8 bf16, 2^-11 fp16)."""
import sys
import threading

import numpy as np
import pytest
import torch

import tokens_oracle as oracle64
from bidmat_b200 import tokens
from bidmat_b200.mat import GHMat, GMat, GSMat
from test_gpu_tokens import check_route, grad_tolerance

pytestmark = pytest.mark.gpu
U = 2.0 ** -24
DT = {"fp32": torch.float32, "bf16": torch.bfloat16, "fp16": torch.float16}
HALF = {n: torch.finfo(t).eps / 2 for n, t in DT.items()}


def matrix(t):
    return GMat(t) if t.dtype == torch.float32 else GHMat(t)


# ------------------------------------------------------------------------------------------ top logits

@pytest.mark.parametrize("dtype", ["fp32", "bf16"])
@pytest.mark.parametrize("V,T,k", [(9000, 40, 512), (70001, 6, 512), (131072, 2, 300), (40000, 500, 230)])
def test_top_with_long_lists(cuda_device, dtype, V, T, k):
    """Columns that keep the list near the length at which it is cut: ascending rows, steps, and rows in no order with
    many picks.  Whole numbers and the logits themselves are equal, also from call to call."""
    g = torch.Generator(device=cuda_device)
    g.manual_seed(V + k)
    x = torch.randn((T, V), generator=g, device=cuda_device)
    x[0] = torch.linspace(-4, 4, V, device=cuda_device)
    if T > 3:
        x[1] = torch.arange(V, device=cuda_device) // 700 * 0.125
        x[2] = torch.sort(x[2]).values
        x[3] = x[3].abs() + torch.arange(V, device=cuda_device) / V
    x = x.to(DT[dtype])
    S = tokens.topLogits(matrix(x), k)
    v, i = torch.sort(x.float(), dim=1, descending=True, stable=True)
    assert torch.equal(S.pir.view(T, k), i[:, :k].to(torch.int32))
    assert torch.equal(S.pdata.view(T, k), v[:, :k])
    for _ in range(20):
        again = tokens.topLogits(matrix(x), k)
        assert torch.equal(again.pir, S.pir) and torch.equal(again.pdata, S.pdata)


# ------------------------------------------------------------------------------------------ distillation

def row(v, device):
    return None if v is None else GMat(torch.as_tensor(np.asarray(v, np.float32), device=device).view(-1, 1))


def sparse(V, T, jc, ir, data, device):
    return GSMat.from_csc(V, T, torch.as_tensor(np.asarray(jc, np.int32), device=device),
                          torch.as_tensor(np.asarray(ir, np.int32), device=device),
                          torch.as_tensor(np.asarray(data, np.float32), device=device))


@pytest.mark.parametrize("dtype", ["fp32", "bf16", "fp16"])
@pytest.mark.parametrize("V,T,k", [(9000, 2, 500), (131072, 1, 4000), (60001, 3, 1500), (131072, 700, 200)])
def test_distill_in_place_with_entries_in_every_part(cuda_device, dtype, V, T, k):
    """Columns that are split over CTAs, with many entries, most of them at the far end: the loss and the gradient are the
    bits of the call that leaves the logits alone."""
    g = torch.Generator(device=cuda_device)
    g.manual_seed(V + T)
    x = torch.randn((T, V), generator=g, device=cuda_device).to(DT[dtype])
    ir = torch.cat([torch.arange(0, V - k // 2, (V - k // 2) // (k - k // 2), device=cuda_device)[: k - k // 2],
                    torch.arange(V - k // 2, V, device=cuda_device)])
    z = torch.randn((T, k), generator=g, device=cuda_device)
    Z = sparse(V, T, np.arange(T + 1) * k, ir.repeat(T).cpu().numpy(), z.flatten().cpu().numpy(), cuda_device)
    loss, dX = tokens.distillWithGrad(matrix(x), Z, temperature=2.0)
    assert bool(torch.isfinite(loss.t).all())
    for _ in range(30):
        y = matrix(x.clone())
        again, _ = tokens.distillWithGrad(y, Z, temperature=2.0, omat=y)
        assert torch.equal(again.t, loss.t) and torch.equal(y.t, dX.t)


# ------------------------------------------------------------------------------------------ large maxima
#
# Exponents are those of the differences from the largest logit, however large it is against the temperature.  The
# definition is taken from the differences too: next to 1e20 the ordinary one loses its logarithms in 64 bits as well.
# With d = (max - x)/t, of which what is beyond 104 leaves the range of fp32:
#   sum of exponentials, relative   e = u (2 max d + V/256 + 16): an argument is off by at most 2 u d (its own rounding and that
#                                   of log2(e)/t), ex2 by 4 u, a thread adds V/512 terms or fewer, the rest is for joining them
#   log-sum-exp                     e + u |L|
#   loss                            e + 4 u (1 + |loss|)
#   gradient                        |w|/t (q (e + u (2 d + 8)) + 4 u p) + h |gradient|, and half the smallest number
# and from a saved log-sum-exp S, where q = exp(x/t - S) may be far from a distribution, with d = |x/t - S| + u |S|:
#   gradient                        |w|/t (q (u (2 d + 12) + 2^-50 |S|) + 4 u p) + h |gradient|
# 16-bit gradients may have their factor in the exponent, two roundings of at most 2^-16 and 2^-17 there: (2^-16 + 2^-17) log 2
# of q besides.
FACTOR = {"fp32": 0.0, "bf16": (2.0 ** -16 + 2.0 ** -17) * np.log(2), "fp16": (2.0 ** -16 + 2.0 ** -17) * np.log(2)}
SMALLEST = {"fp32": 2.0 ** -126, "bf16": 2.0 ** -126, "fp16": 2.0 ** -25}


def close(got, want, tol, what):
    got, want, tol = (np.asarray(v, np.float64) for v in (got, want, tol))
    bad = ~(np.abs(got - want) <= tol)
    if bad.any():
        i = tuple(int(v[0]) for v in np.nonzero(bad))
        raise AssertionError("%s: %d of %d outside, first at %s: got %r want %r tolerance %r"
                             % (what, bad.sum(), bad.size, i, got[i], want[i], np.broadcast_to(tol, got.shape)[i]))


def by_differences(x, t):
    """(d, q, log of the sum of exp(-d)) of the rows of x"""
    d = (x.max(1, keepdims=True) - x) / t
    e = np.exp(-d)
    s = e.sum(1, keepdims=True)
    return d, e / s, np.log(s[:, 0])


def large_columns(dtype, t, V, rng):
    if t < 0.1:
        at = [14.0, -60.0, 300.0, -3000.0]
    else:
        at = [300.0, -3e3, 3e4, -6e4]
        if dtype != "fp16":
            at += [-1e5, 1e6, -1e7, 1e8, -1e8, -1e9, 1e10, -1e20, 1e30, -1e37, 2e38]
    at = [a for a in at for _ in range(2)]
    x = np.array(at)[:, None] + np.where(np.arange(len(at)) % 2, 3.0 * t, 0.0)[:, None] * rng.standard_normal((len(at), V))
    return torch.as_tensor(x, device="cuda").to(DT[dtype])


@pytest.mark.parametrize("V", [300, 9001, 60000, 300007])
@pytest.mark.parametrize("t", [1.0, 2.5, 1e-4, 1e-7])
@pytest.mark.parametrize("dtype", ["fp32", "bf16", "fp16"])
def test_log_sum_exp_of_large_maxima(cuda_device, dtype, t, V):
    x = large_columns(dtype, t, V, np.random.default_rng(V))
    T, t32 = x.shape[0], float(np.float32(t))
    xs = x.double().cpu().numpy()
    d, _, logs = by_differences(xs, t32)
    L = xs.max(1) / t32 + logs
    tol = U * (2 * np.minimum(d, 104).max(1) + V / 256 + 16) + U * np.abs(L)
    lse = row(np.zeros(T), cuda_device)
    tokens.topLogits(matrix(x), 5, temperature=t, lse=lse)
    close(lse.t.cpu().numpy()[:, 0], L, tol, "log-sum-exp of topLogits")
    Z = sparse(V, T, np.arange(T + 1), np.zeros(T), np.zeros(T), cuda_device)
    _, out = tokens.distill(matrix(x), Z, temperature=t)
    close(out.t.cpu().numpy()[:, 0], L, tol, "log-sum-exp of distill")


def check_large_gradients(device, dtype, t, V):
    rng = np.random.default_rng(V + 1)
    x = large_columns(dtype, t, V, rng)
    T, t32 = x.shape[0], float(np.float32(t))
    xs = x.double().cpu().numpy()
    k = min(V, 200)
    ir = np.stack([rng.permutation(V)[:k] for _ in range(T)])
    z = np.float32(t * rng.standard_normal((T, k)))
    w = np.full(T, np.float32(t * (1024 if dtype == "fp16" else 1)))
    Z = sparse(V, T, np.arange(T + 1) * k, ir.ravel(), z.ravel(), device)
    d, q, logs = by_differences(xs, t32)
    _, pz, logz = by_differences(z.astype(np.float64), t32)
    p = np.zeros((T, V))
    np.put_along_axis(p, ir, pz, 1)
    wt = w.astype(np.float64)[:, None] / t32
    e = U * (2 * np.minimum(d, 104).max(1) + V / 256 + 16)
    zd, xd = (z.max(1, keepdims=True).astype(np.float64) - z) / t32, np.take_along_axis(d, ir, 1)
    loss = (pz * (xd - zd)).sum(1) + logs - logz
    want = wt * (q - p)
    got, dX = tokens.distillWithGrad(matrix(x), Z, weights=row(w, device), temperature=t)
    close(dX.t.double().cpu().numpy(), want, wt * (q * (e[:, None] + U * (2 * np.minimum(d, 104) + 8) + FACTOR[dtype]) + 4 * U * p)
          + HALF[dtype] * np.abs(want) + SMALLEST[dtype] * (1 + wt), "gradient")
    out, L = tokens.distill(matrix(x), Z, temperature=t)
    S = L.t.double().cpu().numpy()
    some = (np.abs(S[:, 0]) <= 2e8) & np.isfinite(S[:, 0])
    S = S[some]
    q = np.exp(xs[some] / t32 - S)
    far = np.minimum(np.abs(xs[some] / t32 - S) + U * np.abs(S), 104)
    want = wt[some] * (q - p[some])
    dX = tokens.distillGrad(matrix(x), Z, L, weights=row(w, device), temperature=t)
    close(dX.t.double().cpu().numpy()[some], want, wt[some] * (q * (U * (2 * far + 12) + 2.0 ** -50 * np.abs(S) + FACTOR[dtype]) + 4 * U * p[some])
          + HALF[dtype] * np.abs(want) + SMALLEST[dtype] * (1 + wt[some]), "gradient from the saved log-sum-exp")
    return loss, e, out.t.cpu().numpy()[:, 0], w, got.t.cpu().numpy()[:, 0], np.abs(xs).max(1) / t32


@pytest.mark.parametrize("V", [300, 9001, 60000, 300007])
@pytest.mark.parametrize("t", [1.0, 2.5, 1e-4, 1e-7])
def test_gradients_of_large_maxima(cuda_device, t, V):
    loss, e, out, w, weighted, at = check_large_gradients(cuda_device, "fp32", t, V)
    tol, some = e + 4 * U * (1 + np.abs(loss)), at < 1e6
    close(out[some], loss[some], tol[some], "loss")
    close(weighted[some], (w * loss)[some], (w * tol)[some], "weighted loss")


@pytest.mark.parametrize("V", [300, 9001, 60000, 300007])
@pytest.mark.parametrize("t", [1.0, 2.5, 1e-4, 1e-7])
@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
def test_gradients_of_large_maxima_in_16_bits(cuda_device, dtype, t, V):
    check_large_gradients(cuda_device, dtype, t, V)


@pytest.mark.parametrize("V", [300, 60000, 300007])
@pytest.mark.parametrize("t", [1.0, 2.5])
@pytest.mark.parametrize("dtype", ["fp32", "bf16", "fp16"])
def test_loss_of_large_logits(cuda_device, dtype, t, V):
    """The student's logits, the teacher's or both next to a large number, masks that leave nothing among them."""
    loss, e, out, w, weighted, _ = check_large_gradients(cuda_device, dtype, t, V)
    tol = e + 4 * U * (1 + np.abs(loss))
    close(out, loss, tol, "loss")
    close(weighted, w * loss, w * tol, "weighted loss")
    rng = np.random.default_rng(V + 2)
    t32, k = float(np.float32(t)), min(V, 200)
    low = torch.finfo(DT[dtype]).min
    xs = [0.0, 0.0, 0.0, 0.0, low, low, -3e4, low]
    zs = [-1e9, -1e20, torch.finfo(torch.float32).min, 1e7, torch.finfo(torch.float32).min, 0.0, -1e9, low]
    T = len(xs)
    x = torch.as_tensor(np.array(xs)[:, None] + rng.standard_normal((T, V)), device=cuda_device).to(DT[dtype])
    x = torch.clamp(x, min=low)
    z = np.float32(np.maximum(np.array(zs)[:, None] + rng.standard_normal((T, k)), float(np.finfo(np.float32).min)))
    ir = np.stack([rng.permutation(V)[:k] for _ in range(T)])
    Z = sparse(V, T, np.arange(T + 1) * k, ir.ravel(), z.ravel(), cuda_device)
    x64 = x.double().cpu().numpy()
    d, q, logs = by_differences(x64, t32)
    zd, pz, logz = by_differences(z.astype(np.float64), t32)
    loss = (pz * (np.take_along_axis(d, ir, 1) - zd)).sum(1) + logs - logz
    e = U * (2 * np.minimum(d, 104).max(1) + V / 256 + 16)
    out, L = tokens.distill(matrix(x), Z, temperature=t)
    close(out.t.cpu().numpy()[:, 0], loss, e + 4 * U * (1 + np.abs(loss)), "loss of a large teacher")
    w = np.full(T, np.float32(1024 * t))
    got, dX = tokens.distillWithGrad(matrix(x), Z, weights=row(w, cuda_device), temperature=t)
    close(got.t.cpu().numpy()[:, 0], w * loss, w * (e + 4 * U * (1 + np.abs(loss))), "weighted loss of a large teacher")
    p = np.zeros((T, V))
    np.put_along_axis(p, ir, pz, 1)
    wt = 1024.0 * t / t32
    want = wt * (q - p)
    close(dX.t.double().cpu().numpy(), want, wt * (q * (e[:, None] + U * (2 * np.minimum(d, 104) + 8) + FACTOR[dtype]) + 4 * U * p)
          + HALF[dtype] * np.abs(want) + SMALLEST[dtype] * (1 + wt), "gradient of a large teacher")


@pytest.mark.parametrize("dtype", ["fp32", "bf16"])
@pytest.mark.parametrize("V,k", [(1000, 30), (70001, 200), (400003, 5)])
def test_padded_tokens_of_a_teacher_are_nothing_to_learn_from(cuda_device, dtype, V, k):
    """A teacher's columns of -infinity have the log-sum-exp -infinity; the loss and the gradient there are 0, also where the
    student is masked as well, and the other columns are those of a batch without padding."""
    g = torch.Generator(device=cuda_device)
    g.manual_seed(V)
    teach, stud = (torch.randn((6, V), generator=g, device=cuda_device).to(DT[dtype]) for _ in range(2))
    teach[[1, 4, 5]] = -torch.inf
    stud[4] = -torch.inf
    lse = row(np.zeros(6), cuda_device)
    Z = tokens.topLogits(matrix(teach), k, lse=lse)
    assert torch.isneginf(lse.t[[1, 4, 5]]).all()
    loss, L = tokens.distill(matrix(stud), Z, lse=lse)
    wl, dX = tokens.distillWithGrad(matrix(stud), Z, lse=lse)
    dY = tokens.distillGrad(matrix(stud), Z, L, lse=lse)
    for out in (loss.t, wl.t, dX.t, dY.t):
        assert bool((out[[1, 4, 5]] == 0).all()) and bool(torch.isfinite(out).all())
    some = [0, 2, 3]
    lse = row(np.zeros(3), cuda_device)
    Z = tokens.topLogits(matrix(teach[some]), k, lse=lse)
    # split over more or fewer CTAs a column may be summed up in another order: both are within e of the definition
    e = 2 * U * (2 * float(stud[some].float().max() - stud[some].float().min()) + V / 256 + 16)
    ones = tokens.distill(matrix(stud[some]), Z, lse=lse)[0]
    assert bool((loss.t[some] - ones.t).abs().max() <= e + 8 * U * (1 + float(ones.t.abs().max())))


# ------------------------------------------------------------------------------------------ routing

def up(v):
    return np.nextafter(np.float32(v), np.float32(np.inf))


@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
@pytest.mark.parametrize("E,k", [(3, 1), (20, 5), (30, 8), (96, 1), (96, 12), (256, 8), (512, 16), (1024, 32)])
def test_route_a_better_row_behind_identical_ones(cuda_device, score, E, k):
    """Rows with the same score and bias around the k-th place, and behind them one that is better by less than fp32 can
    tell after the bias has been added.  Weights and picks as in 64 bits."""
    rng = np.random.default_rng(E + k)
    places = sorted({E - 1, E // 2, k, 0} & set(range(E)))
    x = np.ones((len(places) + 4, E), np.float32)
    for i, p in enumerate(places):
        x[i, p] = up(1.0)
    x[-4] = 0.0
    x[-3] = 0.5 * rng.integers(0, 2, E)
    x[-2, : k // 2] = 3.0                                   # some picks far above, the rest among identical ones
    x[-2, E - 1] = up(1.0)
    x[-1] = np.where(rng.random(E) < 0.2, up(1.0), 1.0)
    one = np.zeros(E)
    one[E - 1] = 1e-9
    steps = 0.25 + 2.0 ** -30 * rng.integers(0, 3, E)      # bias that moves in small fixed steps
    for bias in (np.full(E, 0.25), one, steps, np.zeros(E)):
        check_route(x, "fp32", cuda_device, k, score=score, bias=bias)
        if E % 4 == 0 and k <= E // 2:
            check_route(x, "fp32", cuda_device, k, score=score, bias=bias, groups=4, topgroups=2, renorm=False)
    for bias in (one, steps):
        check_route(np.round(2 * rng.standard_normal((300, E))) / 2, "bf16", cuda_device, k, score=score, bias=bias)


@pytest.mark.parametrize("E,groups,k", [(32, 8, 4), (64, 16, 8), (256, 8, 8), (512, 16, 16), (1024, 64, 32)])
@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
def test_route_groups_whose_sums_cancel(cuda_device, score, E, groups, k):
    """Biases that force rows on and off by +-1000, so that a group's sum is small against its parts and their roundings
    in fp32 (1e-4 there) are larger than the differences between the groups; picks and weights as in 64 bits."""
    rng = np.random.default_rng(E + groups)
    x = 0.05 * rng.standard_normal((4000 if E <= 64 else 500, E))
    size = E // groups
    for on, off in ((1000.0, -1000.0), (37.5, -37.5), (1e6, -1e6)):
        bias = np.full(E, -2e6)
        bias[::size] = on
        bias[1::size] = off
        check_route(x, "fp32", cuda_device, min(k, size), score=score, bias=bias, groups=groups, topgroups=1 + groups // 2)
        check_route(x, "bf16", cuda_device, 1, score=score, bias=bias + 0.001 * rng.standard_normal(E), groups=groups, topgroups=2)


@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
@pytest.mark.parametrize("E,groups", [(256, 8), (1024, 16)])
def test_route_groups_masked_by_the_lowest_bias(cuda_device, score, E, groups):
    """Whole groups with the lowest number as their bias come behind all others and before groups of nothing but -infinity."""
    rng = np.random.default_rng(E)
    x = rng.standard_normal((50, E))
    size = E // groups
    x[10:, :size] = -np.inf                                 # group 0: nothing to pick from
    x[20:, size:2 * size - 1] = -np.inf                     # group 1: one row is left
    bias = 0.1 * rng.standard_normal(E)
    bias[2 * size:4 * size] = np.finfo(np.float32).min      # groups 2 and 3: masked
    for top in (1, 2, groups - 2, groups - 1, groups):
        for grouptop in (1, 2):
            check_route(x, "fp32", cuda_device, 3, score=score, bias=bias, groups=groups, topgroups=top, grouptop=grouptop)


@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
@pytest.mark.parametrize("E,groups,k", [(8, 2, 3), (24, 4, 3), (30, 5, 7), (32, 4, 8)])
def test_route_few_rows_masked_by_the_lowest_bias(cuda_device, score, E, groups, k):
    """Up to 32 rows of which fewer than k are unmasked: the masked ones follow by row, then those without a score."""
    rng = np.random.default_rng(E)
    x = rng.standard_normal((60, E))
    x[20:40, ::3] = -np.inf
    x[40:, : E // 2] = -np.inf
    for open_rows in (1, 2, k - 1):
        bias = np.full(E, np.finfo(np.float32).min)
        bias[rng.permutation(E)[:open_rows]] = 0.25
        for dtype in ("fp32", "bf16"):
            check_route(x, dtype, cuda_device, k, score=score, bias=bias)
            for top in range(1 + (k - 1) // (E // groups), groups + 1):
                check_route(x, dtype, cuda_device, k, score=score, bias=bias, groups=groups, topgroups=top)


@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
@pytest.mark.parametrize("scale", [1e-39, -3e-39, 2.0 ** -127, 1e30, -0.5])
@pytest.mark.parametrize("E", [40, 300])
def test_route_gradient_of_tiny_and_large_scales(cuda_device, score, scale, E):
    """Scales whose reciprocal is no number of fp32 among them; weights and their gradients make up for the scale, so that
    the gradient of the scores is of ordinary size.  Tolerance as for other scales."""
    rng = np.random.default_rng(E)
    x = rng.standard_normal((20, E))
    scale = float(np.float32(scale))
    X = matrix(torch.as_tensor(x, device=cuda_device, dtype=torch.float32))
    S = tokens.route(X, 6, score=score, scale=scale)
    dS = S.copy()
    dS.pdata = torch.as_tensor((rng.standard_normal(S.nnz) * min(abs(1.0 / scale), 1e38)).astype(np.float32), device=cuda_device)
    got = tokens.routeGrad(X, S, dS, score=score, scale=scale).t.double().cpu().numpy()
    xs, w, g = (v.double().cpu().numpy() for v in (X.t, S.pdata, dS.pdata))
    want = oracle64.route_grad(xs, S.pjc.cpu().numpy(), S.pir.cpu().numpy(), w, g, score, True, scale)
    assert np.abs(want).max() > 0.001          # a weight of 1e-39/6 and a gradient of 1e38 make 1/60, times 1 - s of a large sigmoid
    close(got, want, grad_tolerance(xs, S, w, g, want, True, scale, "fp32"), "routeGrad at scale %g" % scale)


@pytest.mark.parametrize("dtype", ["fp32", "bf16", "fp16"])
@pytest.mark.parametrize("E,k", [(16, 1), (32, 4), (48, 6), (64, 8), (96, 8), (96, 12), (128, 16), (160, 20), (256, 32), (512, 32)])
def test_route_of_few_vectors(cuda_device, dtype, E, k):
    """Aligned columns with about as many 16-byte vectors as picks: right, and in the time of columns that are read one
    element at a time or so.  When they all went the long way in 64 bits they took two to five times that."""
    rng = np.random.default_rng(E + k)
    check_route(1.5 * rng.standard_normal((200, E)), dtype, cuda_device, k)
    x = (1.5 * torch.randn((65536, E + 8), device=cuda_device)).to(DT[dtype])
    wide = matrix(x[:, :E].contiguous())
    if dtype == "fp32":                                     # another base address, which is not that of a vector
        flat = torch.empty(wide.t.numel() + 1, device=cuda_device)
        narrow = matrix(flat[1:].view(wide.t.shape).copy_(wide.t))
    else:
        narrow = matrix(x[:, 1:E + 1])

    def time(X):
        times = []
        for _ in range(12):
            a, b = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
            a.record()
            for _ in range(8):
                tokens.route(X, k)
            b.record()
            torch.cuda.synchronize()
            times.append(a.elapsed_time(b))
        return min(times)

    assert any(time(wide) < 2.0 * time(narrow) for _ in range(3))


@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
@pytest.mark.parametrize("E,k", [(12, 3), (40, 6), (300, 16)])
def test_route_weights_of_tiny_scores(cuda_device, score, E, k):
    """Picks that are all tiny, forced by a bias (softmax) or for want of better ones (sigmoid), some of them next to the end
    of fp32's range: their shares are still those of 64 bits."""
    rng = np.random.default_rng(E)
    x = np.full((64, E), -np.inf)
    at = np.linspace(-100, -20, 64)
    x[:, :k] = at[:, None] - 25.0 * rng.random((64, k))
    bias = None
    if score == "softmax":
        x[:, k] = 0.0
        bias = np.zeros(E)
        bias[:k] = 4.0 + 0.125 * np.arange(k)
    check_route(x, "fp32", cuda_device, k, score=score, bias=bias)
    check_route(x, "fp32", cuda_device, k, score=score, bias=bias, scale=2.5)


# ------------------------------------------------------------------------------------------ several at once

def test_calls_of_different_sizes_from_two_host_threads(cuda_device):
    """The same kernels with different amounts of shared memory, called from two threads at once: every call is launched and
    gives what it gives alone."""
    from bidmat_b200 import _lib

    def scores(E):
        return matrix(torch.randn((8, E), device=cuda_device))

    def arguments(X, S, stream):
        return (X.nrows, X.ncols, X.pdata, X.nrows, 0, 32, 0, 0, 1, 1, 2, 1, 1.0, S.pir.data_ptr(), S.pic.data_ptr(),
                S.pjc.data_ptr(), S.pdata.data_ptr(), stream.cuda_stream)

    jobs = []
    for E, V in ((1024, 32768), (700, 20000)):
        x = matrix(torch.randn((300, V), device=cuda_device).to(torch.bfloat16))
        r, Z = scores(E), tokens.topLogits(x, 4)
        jobs.append((r, tokens.route(r, 32), x, Z, tokens.distillWithGrad(x, Z)))
    torch.cuda.synchronize()
    failed, start = [], threading.Barrier(2, timeout=60)

    def run(r, S, x, Z, want):
        try:
            torch.cuda.set_device(cuda_device)
            stream, T, out = torch.cuda.Stream(), S.copy(), matrix(torch.empty_like(x.t))
            args = arguments(r, T, stream)
            torch.cuda.synchronize()
            start.wait()
            for i in range(30000):
                err = _lib.lib.bidmat_b200_route(*args)
                assert err == 0, _lib.error_string(err)
                if i % 500 == 0:
                    stream.synchronize()
            with torch.cuda.stream(stream):
                for i in range(300):
                    loss, _ = tokens.distillWithGrad(x, Z, omat=out)
            stream.synchronize()
            assert torch.equal(T.pir, S.pir) and torch.equal(T.pdata, S.pdata)
            assert torch.equal(loss.t, want[0].t) and torch.equal(out.t, want[1].t)
        except Exception as e:                              # the thread's, for the test to raise
            failed.append(e)

    before = sys.getswitchinterval()
    sys.setswitchinterval(1e-5)
    try:
        threads = [threading.Thread(target=run, args=job) for job in jobs]
        for t in threads:
            t.start()
        for t in threads:
            t.join()
    finally:
        sys.setswitchinterval(before)
    assert not failed, failed
