"""Corners of the operators on token columns: long lists, columns in place, large and masked values, near ties.

Against definitions in 64 bits (tokens_oracle), with the tolerances named at each test, where u = 2^-24 is half a
step of fp32 and h half a step of the output type (2^-24 fp32, 2^-8 bf16, 2^-11 fp16)."""
import numpy as np
import pytest
import torch

import tokens_oracle as oracle64
from bidmat_b200 import tokens
from bidmat_b200.mat import GHMat, GMat

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
