"""Definitions in 64 bits of the operators between token columns and sparse matrices, in numpy.
Dense matrices are (ncols, nrows) arrays, sparse ones (jc, ir, data)."""
import numpy as np


def route(x, k, score, bias, groups, topgroups, grouptop, renorm, scale):
    x = np.asarray(x, np.float64)
    T, E = x.shape
    pir, w = np.zeros((T, k), np.int32), np.zeros((T, k))
    size = E // groups
    for t in range(T):
        col = x[t]
        if np.isnan(col).any() or np.isposinf(col).any():
            pir[t], w[t] = np.arange(k), np.nan
            continue
        live = ~np.isneginf(col)
        s = np.zeros(E)
        if score == "softmax":
            if live.any():
                e = np.exp(col - col.max())
                s = e / e.sum()
        else:
            s[live] = 1.0 / (1.0 + np.exp(-col[live]))
        rank = s + (0.0 if bias is None else np.asarray(bias, np.float64))
        rank = np.where(live & ~np.isnan(rank), rank, -np.inf)
        key = rank if bias is not None else col
        if groups > 1:
            val = []
            for g in range(groups):
                b = sorted((v for v in rank[g * size:(g + 1) * size] if v > -np.inf), reverse=True)[:grouptop]
                val.append(sum(b) if b else -np.inf)
            keep = sorted(range(groups), key=lambda g: (-val[g], g))[:topgroups]
            mask = np.isin(np.arange(E) // size, keep)
            rank = np.where(mask, rank, -np.inf)
        key = np.where(rank > -np.inf, key, -np.inf)
        order = sorted(range(E), key=lambda e: (-key[e], e))[:k]
        pir[t] = order
        w[t] = np.where(key[order] > -np.inf, s[order], 0.0)
        if renorm and w[t].sum() > 0:
            w[t] /= w[t].sum()
    return pir, w * scale


def route_grad(x, jc, ir, w, g, score, renorm, scale):
    x, w, g = (np.asarray(a, np.float64) for a in (x, w, g))
    T, E = x.shape
    out = np.zeros((T, E))
    for t in range(T):
        js = range(jc[t], jc[t + 1])
        D = sum(w[j] * g[j] for j in js)
        if score == "softmax" and not renorm and np.isfinite(x[t].max()):
            e = np.exp(x[t] - x[t].max())
            out[t] = -D * e / e.sum()
        for j in js:
            if not 0 <= ir[j] < E:
                continue
            v = w[j] * (g[j] - (D / scale if renorm else 0.0))
            if score == "sigmoid":
                v /= 1.0 + np.exp(x[t, ir[j]])
            out[t, ir[j]] += v
    return out


def top(x, k, tau):
    x = np.asarray(x, np.float64)
    T, V = x.shape
    pir, val, lse = np.zeros((T, k), np.int32), np.zeros((T, k)), np.zeros(T)
    for t in range(T):
        key = np.where(np.isnan(x[t]), np.inf, x[t])
        o = np.lexsort((np.arange(V), -key, ~np.isnan(x[t])))[:k]
        pir[t], val[t] = o, x[t][o]
        m = np.nanmax(x[t]) if not np.isnan(x[t]).any() else np.nan
        u = 0.0 if np.isneginf(m) else m
        with np.errstate(divide="ignore", invalid="ignore"):
            lse[t] = u / tau + np.log(np.exp((x[t] - u) / tau).sum())
    return pir, val, lse


def distill(x, jc, ir, z, tau, tlse=None, weights=None, slse=None):
    """(loss, L, gradient of sum weights * loss, P)"""
    x, z = np.asarray(x, np.float64), np.asarray(z, np.float64)
    T, V = x.shape
    loss, L, grad, mass = np.zeros(T), np.zeros(T), np.zeros((T, V)), np.zeros(T)
    with np.errstate(all="ignore"):
        for t in range(T):
            xs = x[t] / tau
            m = xs.max()
            u = 0.0 if np.isneginf(m) else m
            L[t] = u + np.log(np.exp(xs - u).sum())
            r, zs = ir[jc[t]:jc[t + 1]], z[jc[t]:jc[t + 1]] / tau
            w = 1.0 if weights is None else float(weights[t])
            if len(r) == 0 or np.isneginf(zs).all() or w == 0.0:
                continue
            lt = float(tlse[t]) if tlse is not None else zs.max() + np.log(np.exp(zs - zs.max()).sum())
            p = np.exp(zs - lt)
            P = mass[t] = p.sum()
            if P == 0.0:
                continue
            if ((r < 0) | (r >= V)).any():
                loss[t], grad[t], mass[t] = np.nan, np.nan, np.nan
                continue
            loss[t] = sum(pi * ((zi - lt) - (xs[ri] - L[t])) for pi, zi, ri in zip(p, zs, r) if pi > 0)
            if np.isneginf(m) or not np.isfinite(L[t]):
                loss[t] = np.nan
            grad[t] = P * np.exp(xs - (L[t] if slse is None else float(slse[t])))
            np.add.at(grad[t], r, -p)
            grad[t] *= w / tau
    return loss, L, grad, mass
