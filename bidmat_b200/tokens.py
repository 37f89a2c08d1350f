"""Operators of language models between dense token columns and sparse matrices.

A dense matrix (GMat in fp32, GHMat in bf16 or fp16) holds one token per column: the scores of
its experts, or its logits over the vocabulary.  A GSMat of the same size holds a few rows of every
token: the experts it goes to with their weights, or a teacher's largest logits.

  route           scores -> weights of the picked experts        routeGrad   its gradient
  topLogits       logits -> the k largest of every token
  distill         loss of a student against a teacher's top logits
  distillGrad     its gradient from a saved forward pass
  distillWithGrad both with one read of the logits

The sparse results work with the products of bidmat_b200.mat: with S = route(X, k), A * S mixes the
columns of A that every token was routed to, B.xT(S) is the gradient of A, DDS(A, B, S) the gradient of
the weights (which routeGrad takes on to the scores) and S.t lists the tokens of every expert.

Like GSMat.t and TransposedPlan.run the calls run on torch's current stream and return without
waiting for it, so they can be captured into a CUDA graph; vectors with one value per token are
1 x ncols GMats.  Formulas, ranges and the treatment of infinities and NaN: include/bidmat_b200.h.
"""
import torch

from . import _lib
from .mat import GHMat, GMat, GSMat, _check, _ptr

_L = _lib.lib

# torch.cuda.current_stream(i).cuda_stream without making the stream object, which takes as long as the rest of a call
_raw_stream = torch._C._cuda_getCurrentRawStream

F32, BF16, F16 = 0, 1, 2
_DTYPES = {torch.float32: F32, torch.bfloat16: BF16, torch.float16: F16}
_SCORES = {"softmax": 0, "sigmoid": 1}


def _dense(X, what):
    """(matrix, leading dimension, type code)"""
    if isinstance(X, GMat):
        return X, X.nrows, F32
    if isinstance(X, GHMat):
        return X, X.ld, _DTYPES[X.t.dtype]
    raise RuntimeError("%s: expected a GMat or GHMat" % what)


def _score(name, what):
    if name not in _SCORES:
        raise RuntimeError("%s: score is 'softmax' or 'sigmoid', not %r" % (what, name))
    return _SCORES[name]


def _same_device(what, device, *mats):
    for m in mats:
        if m is not None and (m.device if isinstance(m, GSMat) else m.t.device) != device:
            raise RuntimeError("%s: operands on different devices" % what)


def _sparse(S, X, what):
    if not isinstance(S, GSMat):
        raise RuntimeError("%s: expected a GSMat" % what)
    if S.nrows != X.nrows or S.ncols != X.ncols:
        raise RuntimeError("%s: dimensions mismatch (%d %d) (%d %d)" % (what, X.nrows, X.ncols, S.nrows, S.ncols))
    S._debug_check()


def _vector(v, ncols, what, name):
    """A 1 x ncols GMat, or None."""
    if v is None:
        return 0
    if not isinstance(v, GMat) or v.nrows != 1 or v.ncols != ncols:
        raise RuntimeError("%s: %s should be a 1 x %d GMat" % (what, name, ncols))
    return v.pdata


def _new_sparse(X, k, omat, what):
    nnz = k * X.ncols
    if omat is not None:
        if omat.nrows != X.nrows or omat.ncols != X.ncols or omat.nnz != nnz:
            raise RuntimeError("%s: dimensions mismatch in output GSMat" % what)
        _same_device(what, X.t.device, omat)
        omat._plans = {}       # another pattern from here on; matrices that share the old one keep theirs
        return omat
    dev = X.t.device
    if nnz > 0x7fffffff:
        raise RuntimeError("%s: %d entries do not fit 32-bit indices" % (what, nnz))
    # one allocation; the lists begin at multiples of 16 bytes
    n4 = (nnz + 3) & ~3
    pir, pic, data, pjc = torch.empty(3 * n4 + X.ncols + 1, dtype=torch.int32, device=dev).split((n4, n4, n4, X.ncols + 1))
    if n4 != nnz:
        pir, pic, data = pir[:nnz], pic[:nnz], data[:nnz]
    return GSMat(X.nrows, X.ncols, nnz, pir, pic, pjc, data.view(torch.float32))


def _new_dense(X, omat, what):
    if omat is None:
        t = torch.empty((X.ncols, X.nrows), dtype=X.t.dtype, device=X.t.device)
        return GMat(t) if isinstance(X, GMat) else GHMat(t)
    if type(omat) is not type(X) or omat.t.dtype != X.t.dtype or omat.nrows != X.nrows or omat.ncols != X.ncols:
        raise RuntimeError("%s: dimensions or types mismatch in output" % what)
    _same_device(what, X.t.device, omat)
    return omat


def _row(ncols, device):
    return GMat(torch.empty((ncols, 1), dtype=torch.float32, device=device))


def _call(fn, device, what, *args):
    if device.index == torch.cuda.current_device():
        err = fn(*args, _raw_stream(device.index))
    else:
        with torch.cuda.device(device):
            err = fn(*args, _raw_stream(device.index))
    if err != 0:
        _check(err, what)


def route(X, k, score="softmax", bias=None, groups=1, topgroups=1, grouptop=2, renorm=True, scale=1.0, omat=None):
    """The k experts of every token as a GSMat of their weights (rows: experts, columns: tokens).
    `bias` (nrows x 1 GMat) is added to the scores for the choice only; with `groups` > 1 only the experts
    of the `topgroups` best groups compete, a group counting as the sum of its `grouptop` best."""
    what = "route"
    X, ld, dt = _dense(X, what)
    sc = _score(score, what)
    if not 1 <= k <= min(32, X.nrows) or X.nrows > 1024:
        raise RuntimeError("route: k = %d of %d experts (at most 32 of 1024)" % (k, X.nrows))
    if (groups < 1 or X.nrows % groups or not 1 <= topgroups <= groups or grouptop not in (1, 2)
            or k > topgroups * (X.nrows // groups)):
        raise RuntimeError("route: %d of %d groups cannot give %d of %d experts" % (topgroups, groups, k, X.nrows))
    if bias is not None and (not isinstance(bias, GMat) or bias.nrows != X.nrows or bias.ncols != 1):
        raise RuntimeError("route: the bias should be a %d x 1 GMat" % X.nrows)
    _same_device(what, X.t.device, bias)
    S = _new_sparse(X, k, omat, what)
    _call(_L.bidmat_b200_route, X.t.device, "route:", X.nrows, X.ncols, X.pdata, ld, dt, k, sc,
          0 if bias is None else bias.pdata, groups, topgroups, grouptop, 1 if renorm else 0, scale,
          _ptr(S.pir), _ptr(S.pic), _ptr(S.pjc), _ptr(S.pdata))
    return S


def routeGrad(X, S, dS, score="softmax", renorm=True, scale=1.0, omat=None):
    """The gradient of the scores X from the gradient dS of the weights S = route(X, ...) (a GSMat of S's
    pattern, as DDS gives it).  `omat` may be X."""
    what = "routeGrad"
    X, ld, dt = _dense(X, what)
    sc = _score(score, what)
    _sparse(S, X, what)
    if not isinstance(dS, GSMat) or dS.nnz != S.nnz:
        raise RuntimeError("routeGrad: dS should be a GSMat with the %d entries of S" % S.nnz)
    if not 1 <= X.nrows <= 1024:
        raise RuntimeError("routeGrad: %d experts (at most 1024)" % X.nrows)
    _same_device(what, X.t.device, S, dS)
    out = _new_dense(X, omat, what)
    _call(_L.bidmat_b200_route_grad, X.t.device, "routeGrad:", X.nrows, X.ncols, S.nnz, X.pdata, ld, dt, sc,
          1 if renorm else 0, scale, _ptr(S.pir), _ptr(S.pjc), _ptr(S.pdata), _ptr(dS.pdata), out.pdata,
          out.ld if isinstance(out, GHMat) else out.nrows)
    return out


def topLogits(X, k, temperature=1.0, lse=None, omat=None):
    """The k largest logits of every token as a GSMat, largest first, equal ones by row.  `lse`, a 1 x ncols
    GMat, receives the log-sum-exp of every column of X / temperature: with it `distill` takes the
    probabilities over the whole vocabulary instead of those over the k entries."""
    what = "topLogits"
    X, ld, dt = _dense(X, what)
    if not 1 <= k <= min(512, X.nrows):
        raise RuntimeError("topLogits: k = %d of %d rows (at most 512)" % (k, X.nrows))
    pl = _vector(lse, X.ncols, what, "lse")
    _same_device(what, X.t.device, lse)
    S = _new_sparse(X, k, omat, what)
    _call(_L.bidmat_b200_top_logits, X.t.device, "topLogits:", X.nrows, X.ncols, X.pdata, ld, dt, k, temperature,
          _ptr(S.pir), _ptr(S.pic), _ptr(S.pjc), _ptr(S.pdata), pl)
    return S


def distill(X, Z, temperature=1.0, lse=None):
    """(loss, log-sum-exp) of every token: the divergence of the student's logits X from the teacher's top
    logits Z, as 1 x ncols GMats.  `lse` (1 x ncols) normalises the teacher's probabilities; without it they
    sum to one over the entries of Z.  A token without entries has loss 0."""
    what = "distill"
    X, ld, dt = _dense(X, what)
    _sparse(Z, X, what)
    pl = _vector(lse, X.ncols, what, "lse")
    _same_device(what, X.t.device, Z, lse)
    loss, out = _row(X.ncols, X.t.device), _row(X.ncols, X.t.device)
    _call(_L.bidmat_b200_distill, X.t.device, "distill:", X.nrows, X.ncols, Z.nnz, X.pdata, ld, dt, temperature,
          _ptr(Z.pir), _ptr(Z.pjc), _ptr(Z.pdata), pl, loss.pdata, out.pdata)
    return loss, out


def distillGrad(X, Z, slse, weights=None, temperature=1.0, lse=None, omat=None):
    """The gradient in X of the sum over the tokens of weights * distill(X, Z, temperature, lse)[0], from the
    log-sum-exp `slse` that distill returned.  `omat` may be X."""
    what = "distillGrad"
    X, ld, dt = _dense(X, what)
    _sparse(Z, X, what)
    if slse is None:
        raise RuntimeError("distillGrad: needs the log-sum-exp that distill returned")
    ps, pw, pl = (_vector(v, X.ncols, what, n) for v, n in ((slse, "slse"), (weights, "weights"), (lse, "lse")))
    _same_device(what, X.t.device, Z, slse, weights, lse)
    out = _new_dense(X, omat, what)
    _call(_L.bidmat_b200_distill_grad, X.t.device, "distillGrad:", X.nrows, X.ncols, Z.nnz, X.pdata, ld, dt,
          temperature, _ptr(Z.pir), _ptr(Z.pjc), _ptr(Z.pdata), pl, ps, pw, out.pdata,
          out.ld if isinstance(out, GHMat) else out.nrows)
    return out


def distillWithGrad(X, Z, weights=None, temperature=1.0, lse=None, omat=None):
    """(weights * loss, gradient of its sum in X) with one read of X: the training step's form, for weights
    that are known before the loss (a mean over the tokens, a mask, a loss scale).  `omat` may be X."""
    what = "distillWithGrad"
    X, ld, dt = _dense(X, what)
    _sparse(Z, X, what)
    pw, pl = _vector(weights, X.ncols, what, "weights"), _vector(lse, X.ncols, what, "lse")
    _same_device(what, X.t.device, Z, weights, lse)
    out = _new_dense(X, omat, what)
    loss = _row(X.ncols, X.t.device)
    _call(_L.bidmat_b200_distill_with_grad, X.t.device, "distillWithGrad:", X.nrows, X.ncols, Z.nnz, X.pdata, ld, dt,
          temperature, _ptr(Z.pir), _ptr(Z.pjc), _ptr(Z.pdata), pl, pw, loss.pdata, out.pdata,
          out.ld if isinstance(out, GHMat) else out.nrows)
    return loss, out
