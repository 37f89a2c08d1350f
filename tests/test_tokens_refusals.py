"""What the operators on token columns refuse is decided on the host before anything is launched, so the
C entry points can be asked without a GPU; every refused call here passes addresses that are never read."""
import ctypes

import pytest

INVALID = 1                        # cudaErrorInvalidValue
P = 4096                           # an aligned address that no refused call touches
NAN, INF = float("nan"), float("inf")


def lib():
    from bidmat_b200 import _lib
    return _lib.lib


ROUTE = dict(nrows=64, ncols=4, X=P, ldx=64, dtype=0, k=6, score=0, bias=0, ngroups=8, topgroups=2, grouptop=2, renorm=1,
             scale=1.0, Sir=P, Sic=P, Sjc=P, Sdata=P, stream=0)
ROUTE_GRAD = dict(nrows=64, ncols=4, nnz=24, X=P, ldx=64, dtype=0, score=0, renorm=1, scale=1.0, Sir=P, Sjc=P, Sdata=P,
                  dS=P, dX=P, lddx=64, stream=0)
TOP = dict(nrows=100, ncols=4, X=P, ldx=100, dtype=1, k=10, temperature=1.0, Sir=P, Sic=P, Sjc=P, Sdata=P, lse=P, stream=0)
DISTILL = dict(nrows=100, ncols=4, nnz=24, X=P, ldx=100, dtype=1, temperature=1.0, Zir=P, Zjc=P, Zdata=P, Zlse=0, loss=P,
               Xlse=P, stream=0)
DISTILL_GRAD = dict(nrows=100, ncols=4, nnz=24, X=P, ldx=100, dtype=2, temperature=1.0, Zir=P, Zjc=P, Zdata=P, Zlse=0,
                    Xlse=P, weights=0, dX=P, lddx=100, stream=0)
DISTILL_BOTH = dict(nrows=100, ncols=4, nnz=24, X=P, ldx=100, dtype=0, temperature=1.0, Zir=P, Zjc=P, Zdata=P, Zlse=0,
                    weights=0, loss=P, dX=P, lddx=100, stream=0)


@pytest.mark.parametrize("base,name,changes", [
    (ROUTE, "route", [dict(nrows=0), dict(nrows=-1), dict(nrows=1025, ldx=1025, ngroups=1, topgroups=1), dict(ncols=-1),
                      dict(X=0), dict(X=P + 2), dict(ldx=63), dict(dtype=3), dict(dtype=-1), dict(k=0), dict(k=-1),
                      dict(k=17), dict(k=33, ngroups=1, topgroups=1), dict(score=2), dict(score=-1), dict(ngroups=0),
                      dict(ngroups=7), dict(topgroups=0), dict(topgroups=9), dict(grouptop=0), dict(grouptop=3),
                      dict(scale=0.0), dict(scale=NAN), dict(scale=INF), dict(Sir=0), dict(Sic=0), dict(Sjc=0),
                      dict(Sdata=0), dict(ncols=2147483647, k=2)]),
    (ROUTE_GRAD, "route_grad", [dict(nrows=0), dict(nrows=1025, ldx=1025, lddx=1025), dict(ncols=-1), dict(nnz=-1),
                                dict(X=0), dict(ldx=63), dict(lddx=63), dict(X=P + 1), dict(dX=P + 2), dict(dX=0),
                                dict(dtype=3), dict(score=2), dict(scale=0.0), dict(scale=NAN), dict(Sir=0),
                                dict(Sjc=0), dict(Sdata=0), dict(dS=0), dict(ldx=80)]),
    (TOP, "top_logits", [dict(nrows=0), dict(nrows=9, ldx=9), dict(ncols=-1), dict(X=0), dict(X=P + 1), dict(ldx=99),
                         dict(dtype=4), dict(k=0), dict(k=513, nrows=1000, ldx=1000), dict(temperature=0.0),
                         dict(temperature=-1.0), dict(temperature=1e-39), dict(nrows=2147483647, ldx=2147483647),
                         dict(temperature=NAN), dict(temperature=INF), dict(Sir=0), dict(Sic=0),
                         dict(Sjc=0), dict(Sdata=0), dict(ncols=2147483647)]),
    (DISTILL, "distill", [dict(nrows=0), dict(ncols=-1), dict(nnz=-1), dict(X=0), dict(X=P + 1), dict(ldx=99),
                          dict(dtype=3), dict(temperature=0.0), dict(temperature=1e-39), dict(temperature=NAN),
                          dict(nrows=2147483647, ldx=2147483647), dict(ncols=2147483647), dict(Zir=0), dict(Zjc=0),
                          dict(Zdata=0), dict(loss=0), dict(Xlse=0)]),
    (DISTILL_GRAD, "distill_grad", [dict(nrows=0), dict(ncols=-1), dict(nnz=-1), dict(X=0), dict(ldx=99), dict(dtype=3),
                                    dict(temperature=-2.0), dict(temperature=INF), dict(Zir=0), dict(Zjc=0),
                                    dict(Zdata=0), dict(Xlse=0), dict(dX=0), dict(dX=P + 1), dict(lddx=99)]),
    (DISTILL_BOTH, "distill_with_grad", [dict(nrows=0), dict(ncols=-1), dict(nnz=-1), dict(X=0), dict(X=P + 2),
                                         dict(ldx=99), dict(dtype=3), dict(temperature=0.0), dict(Zir=0), dict(Zjc=0),
                                         dict(Zdata=0), dict(loss=0), dict(dX=0), dict(dX=P + 2), dict(lddx=99)]),
], ids=["route", "route_grad", "top_logits", "distill", "distill_grad", "distill_with_grad"])
def test_entry_points_refuse_before_any_launch(base, name, changes):
    fn = getattr(lib(), "bidmat_b200_" + name)
    before = lib().bidmat_b200_launch_count()
    for change in changes:
        args = dict(base, **change)
        assert set(args) == set(base)
        assert fn(*args.values()) == INVALID, change
    assert lib().bidmat_b200_launch_count() == before


def test_no_columns_is_a_successful_no_op():
    L = lib()
    assert L.bidmat_b200_route_grad(*dict(ROUTE_GRAD, ncols=0, nnz=0, X=0, dX=0, Sjc=0, Sir=0).values()) == 0
    assert L.bidmat_b200_distill(*dict(DISTILL, ncols=0, nnz=0, X=0, loss=0).values()) == 0
    assert L.bidmat_b200_distill_grad(*dict(DISTILL_GRAD, ncols=0, nnz=0, X=0, dX=0).values()) == 0
    assert L.bidmat_b200_distill_with_grad(*dict(DISTILL_BOTH, ncols=0, nnz=0, X=0, dX=0).values()) == 0


def test_signatures_have_as_many_arguments_as_the_lists_above():
    from bidmat_b200 import _lib
    for base, name in ((ROUTE, "route"), (ROUTE_GRAD, "route_grad"), (TOP, "top_logits"), (DISTILL, "distill"),
                       (DISTILL_GRAD, "distill_grad"), (DISTILL_BOTH, "distill_with_grad")):
        assert len(_lib._SIGNATURES["bidmat_b200_" + name][1]) == len(base)
    assert ctypes.sizeof(ctypes.c_longlong) == 8
