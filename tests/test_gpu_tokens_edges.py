"""Corners of the operators on token columns: long lists, columns in place, large and masked values, near ties.

Against definitions in 64 bits (tokens_oracle), with the tolerances named at each test, where u = 2^-24 is half a
step of fp32 and h half a step of the output type (2^-24 fp32, 2^-8 bf16, 2^-11 fp16)."""
import numpy as np
import pytest
import torch

import tokens_oracle as oracle64
from bidmat_b200 import tokens
from bidmat_b200.mat import GHMat, GMat, GSMat

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
