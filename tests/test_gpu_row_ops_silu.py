"""silu of the row operators over the whole range of its argument."""
import pytest
import torch

from row_ops_ref import EPS32
from test_gpu_row_ops import DEV, F32, ops       # noqa: F401 (ops: fixture)

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("m", [1, 300])
def test_silu_over_its_range(ops, m):            # noqa: F811
    """act(0 + bias). exp(-v) = 2^(-v log2 e): the product is rounded, which in the exponent of e is |v| half steps, and so is the constant
    (1.44269502 for 1.44269504, 1.34e-8 of it: 0.23 half steps for each unit of v); the rest is a few half steps. Below -87.3 the result is 0 in place of
    less than 1.1e-36."""
    v = torch.cat([torch.linspace(-120, 100, 4401), torch.tensor([0.0, -0.0, 1e-30, -1e-30, 1e-44, 3e38, -3e38, float("inf")])])
    n = v.numel()
    a, w = ops.quantize_fp8(torch.zeros(m, 16, device=DEV)), ops.quantize_fp8(torch.zeros(n, 16, device=DEV), 128)
    y = ops.matmul_fp8(a, w, v.to(DEV), act="silu", dtype=F32).cpu().double()
    want = v.double() * torch.sigmoid(v.double())
    tol = EPS32 * (8 + 1.23 * v.double().abs().clamp(max=100)) * want.abs() + 1.1e-36
    assert (y == y[:1]).all()
    assert torch.isinf(y[0, -1]) and ((y[0] - want).abs()[:-1] <= tol[:-1]).all()
    bad = torch.tensor([float("nan"), -float("inf")], device=DEV)      # -inf * 0, as the formula has it
    y = ops.matmul_fp8(a, ops.quantize_fp8(torch.zeros(2, 16, device=DEV), 128), bad, act="silu", dtype=F32)
    assert torch.isnan(y).all()
