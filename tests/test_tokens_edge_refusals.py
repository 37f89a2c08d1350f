"""Sizes next to the limits that the operators on token columns refuse on the host, before anything is launched."""
import pytest

from test_tokens_refusals import DISTILL, DISTILL_BOTH, DISTILL_GRAD, INVALID, ROUTE_GRAD, lib


@pytest.mark.parametrize("base,name", [(ROUTE_GRAD, "route_grad"), (DISTILL, "distill"), (DISTILL_GRAD, "distill_grad"),
                                       (DISTILL_BOTH, "distill_with_grad")], ids=lambda v: v if isinstance(v, str) else "")
@pytest.mark.parametrize("nnz", [2 ** 31 - 1, 2 ** 31 - 65535])
def test_entries_that_leave_no_room_for_a_loops_step(base, name, nnz):
    before = lib().bidmat_b200_launch_count()
    assert getattr(lib(), "bidmat_b200_" + name)(*dict(base, nnz=nnz).values()) == INVALID
    assert lib().bidmat_b200_launch_count() == before
