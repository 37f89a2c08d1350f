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
from .mat import GHMat, GMat, GSMat, Mat, _check

_L = _lib.lib

# torch.cuda.current_stream(i).cuda_stream without making the stream object, which takes as long as the rest of a call
_raw_stream = torch._C._cuda_getCurrentRawStream

F32, BF16, F16 = 0, 1, 2
_DTYPES = {torch.float32: F32, torch.bfloat16: BF16, torch.float16: F16}
_SCORES = {"softmax": 0, "sigmoid": 1}


def _dense(X, what):
    """(tensor, rows, columns, leading dimension, type code) of a dense operand"""
    if isinstance(X, GMat):
        t = X.t
        n, m = t.shape
        return t, m, n, m, F32
    if isinstance(X, GHMat):
        t = X.t
        n, m = t.shape
        return t, m, n, X.ld, _DTYPES[t.dtype]
    raise RuntimeError("%s: expected a GMat or GHMat" % what)


def _matrix(cls, t):
    """A GMat or GHMat over a tensor that was made for it here."""
    M = cls.__new__(cls)
    M.t = t
    return M


def _score(name, what):
    if name not in _SCORES:
        raise RuntimeError("%s: score is 'softmax' or 'sigmoid', not %r" % (what, name))
    return _SCORES[name]


def _same_device(what, device, *mats):
    for m in mats:
        if m is not None and (m.pjc if isinstance(m, GSMat) else m.t).device != device:
            raise RuntimeError("%s: operands on different devices" % what)


def _sparse(S, nrows, ncols, what):
    if not isinstance(S, GSMat):
        raise RuntimeError("%s: expected a GSMat" % what)
    if S.nrows != nrows or S.ncols != ncols:
        raise RuntimeError("%s: dimensions mismatch (%d %d) (%d %d)" % (what, nrows, ncols, S.nrows, S.ncols))
    if Mat.debugStructure:
        S._debug_check()


def _vector(v, ncols, what, name):
    """The address of a 1 x ncols GMat, 0 for None."""
    if v is None:
        return 0
    if not isinstance(v, GMat) or v.t.shape != (ncols, 1):
        raise RuntimeError("%s: %s should be a 1 x %d GMat" % (what, name, ncols))
    return v.t.data_ptr()


def _new_sparse(t, nrows, ncols, k, omat, what):
    nnz = k * ncols
    if omat is not None:
        if omat.nrows != nrows or omat.ncols != ncols or omat.nnz != nnz:
            raise RuntimeError("%s: dimensions mismatch in output GSMat" % what)
        _same_device(what, t.device, omat)
        omat._plans = {}       # another pattern from here on; matrices that share the old one keep theirs
        return omat
    if nnz > 0x7fffffff:
        raise RuntimeError("%s: %d entries do not fit 32-bit indices" % (what, nnz))
    # one allocation; the lists begin at multiples of 16 bytes
    n4 = (nnz + 3) & ~3
    pir, pic, data, pjc = torch.empty(3 * n4 + ncols + 1, dtype=torch.int32, device=t.device).split((n4, n4, n4, ncols + 1))
    if n4 != nnz:
        pir, pic, data = pir[:nnz], pic[:nnz], data[:nnz]
    return GSMat(nrows, ncols, nnz, pir, pic, pjc, data.view(torch.float32))


def _new_dense(X, t, omat, what):
    """(matrix, leading dimension) of an output like X"""
    if omat is None:
        return _matrix(type(X), torch.empty(t.shape, dtype=t.dtype, device=t.device)), t.shape[1]
    if type(omat) is not type(X) or omat.t.dtype != t.dtype or omat.t.shape != t.shape:
        raise RuntimeError("%s: dimensions or types mismatch in output" % what)
    _same_device(what, t.device, omat)
    return omat, omat.ld if isinstance(omat, GHMat) else t.shape[1]


def _row(ncols, device):
    return _matrix(GMat, torch.empty((ncols, 1), dtype=torch.float32, device=device))


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
    t, nrows, ncols, ld, dt = _dense(X, what)
    sc = _score(score, what)
    if not 1 <= k <= min(32, nrows) or nrows > 1024:
        raise RuntimeError("route: k = %d of %d experts (at most 32 of 1024)" % (k, nrows))
    if (groups < 1 or nrows % groups or not 1 <= topgroups <= groups or grouptop not in (1, 2)
            or k > topgroups * (nrows // groups)):
        raise RuntimeError("route: %d of %d groups cannot give %d of %d experts" % (topgroups, groups, k, nrows))
    if bias is not None and (not isinstance(bias, GMat) or bias.t.shape != (1, nrows)):
        raise RuntimeError("route: the bias should be a %d x 1 GMat" % nrows)
    _same_device(what, t.device, bias)
    S = _new_sparse(t, nrows, ncols, k, omat, what)
    _call(_L.bidmat_b200_route, t.device, "route:", nrows, ncols, t.data_ptr(), ld, dt, k, sc,
          0 if bias is None else bias.t.data_ptr(), groups, topgroups, grouptop, 1 if renorm else 0, scale,
          S.pir.data_ptr(), S.pic.data_ptr(), S.pjc.data_ptr(), S.pdata.data_ptr())
    return S


def routeGrad(X, S, dS, score="softmax", renorm=True, scale=1.0, omat=None):
    """The gradient of the scores X from the gradient dS of the weights S = route(X, ...) (a GSMat of S's
    pattern, as DDS gives it).  `omat` may be X."""
    what = "routeGrad"
    t, nrows, ncols, ld, dt = _dense(X, what)
    sc = _score(score, what)
    _sparse(S, nrows, ncols, what)
    if not isinstance(dS, GSMat) or dS.nnz != S.nnz:
        raise RuntimeError("routeGrad: dS should be a GSMat with the %d entries of S" % S.nnz)
    if not 1 <= nrows <= 1024:
        raise RuntimeError("routeGrad: %d experts (at most 1024)" % nrows)
    _same_device(what, t.device, S, dS)
    out, ldo = _new_dense(X, t, omat, what)
    _call(_L.bidmat_b200_route_grad, t.device, "routeGrad:", nrows, ncols, S.nnz, t.data_ptr(), ld, dt, sc,
          1 if renorm else 0, scale, S.pir.data_ptr(), S.pjc.data_ptr(), S.pdata.data_ptr(), dS.pdata.data_ptr(),
          out.t.data_ptr(), ldo)
    return out


def topLogits(X, k, temperature=1.0, lse=None, omat=None):
    """The k largest logits of every token as a GSMat, largest first, equal ones by row.  `lse`, a 1 x ncols
    GMat, receives the log-sum-exp of every column of X / temperature: with it `distill` takes the
    probabilities over the whole vocabulary instead of those over the k entries."""
    what = "topLogits"
    t, nrows, ncols, ld, dt = _dense(X, what)
    if not 1 <= k <= min(512, nrows):
        raise RuntimeError("topLogits: k = %d of %d rows (at most 512)" % (k, nrows))
    pl = _vector(lse, ncols, what, "lse")
    _same_device(what, t.device, lse)
    S = _new_sparse(t, nrows, ncols, k, omat, what)
    _call(_L.bidmat_b200_top_logits, t.device, "topLogits:", nrows, ncols, t.data_ptr(), ld, dt, k, temperature,
          S.pir.data_ptr(), S.pic.data_ptr(), S.pjc.data_ptr(), S.pdata.data_ptr(), pl)
    return S


def distill(X, Z, temperature=1.0, lse=None):
    """(loss, log-sum-exp) of every token: the divergence of the student's logits X from the teacher's top
    logits Z, as 1 x ncols GMats.  `lse` (1 x ncols) normalises the teacher's probabilities; without it they
    sum to one over the entries of Z.  A token without entries has loss 0."""
    what = "distill"
    t, nrows, ncols, ld, dt = _dense(X, what)
    _sparse(Z, nrows, ncols, what)
    pl = _vector(lse, ncols, what, "lse")
    _same_device(what, t.device, Z, lse)
    loss, out = _row(ncols, t.device), _row(ncols, t.device)
    _call(_L.bidmat_b200_distill, t.device, "distill:", nrows, ncols, Z.nnz, t.data_ptr(), ld, dt, temperature,
          Z.pir.data_ptr(), Z.pjc.data_ptr(), Z.pdata.data_ptr(), pl, loss.t.data_ptr(), out.t.data_ptr())
    return loss, out


def distillGrad(X, Z, slse, weights=None, temperature=1.0, lse=None, omat=None):
    """The gradient in X of the sum over the tokens of weights * distill(X, Z, temperature, lse)[0], from the
    log-sum-exp `slse` that distill returned.  `omat` may be X."""
    what = "distillGrad"
    t, nrows, ncols, ld, dt = _dense(X, what)
    _sparse(Z, nrows, ncols, what)
    if slse is None:
        raise RuntimeError("distillGrad: needs the log-sum-exp that distill returned")
    ps, pw, pl = (_vector(v, ncols, what, n) for v, n in ((slse, "slse"), (weights, "weights"), (lse, "lse")))
    _same_device(what, t.device, Z, slse, weights, lse)
    out, ldo = _new_dense(X, t, omat, what)
    _call(_L.bidmat_b200_distill_grad, t.device, "distillGrad:", nrows, ncols, Z.nnz, t.data_ptr(), ld, dt, temperature,
          Z.pir.data_ptr(), Z.pjc.data_ptr(), Z.pdata.data_ptr(), pl, ps, pw, out.t.data_ptr(), ldo)
    return out


def distillWithGrad(X, Z, weights=None, temperature=1.0, lse=None, omat=None):
    """(weights * loss, gradient of its sum in X) with one read of X: the training step's form, for weights
    that are known before the loss (a mean over the tokens, a mask, a loss scale).  `omat` may be X."""
    what = "distillWithGrad"
    t, nrows, ncols, ld, dt = _dense(X, what)
    _sparse(Z, nrows, ncols, what)
    pw, pl = _vector(weights, ncols, what, "weights"), _vector(lse, ncols, what, "lse")
    _same_device(what, t.device, Z, weights, lse)
    out, ldo = _new_dense(X, t, omat, what)
    loss = _row(ncols, t.device)
    _call(_L.bidmat_b200_distill_with_grad, t.device, "distillWithGrad:", nrows, ncols, Z.nnz, t.data_ptr(), ld, dt,
          temperature, Z.pir.data_ptr(), Z.pjc.data_ptr(), Z.pdata.data_ptr(), pl, pw, loss.t.data_ptr(), out.t.data_ptr(), ldo)
    return loss, out
