"""Calls of the row operators that are refused, or have to hold, because of who calls: derivatives, traces, threads, streams, branches."""
import pytest
import torch

from test_gpu_row_ops import DEV, gen, ops       # noqa: F401 (ops: fixture)

pytestmark = pytest.mark.gpu


def test_derivatives_and_traces_are_refused(ops):          # noqa: F811
    from torch.autograd import forward_ad
    E = ops.LssvcHipError
    x, v = torch.randn(32, 64, device=DEV), torch.ones(64, device=DEV)
    q, w = ops.quantize_fp8(x), ops.quantize_fp8(torch.randn(64, 64, device=DEV), 128)
    with forward_ad.dual_level():
        d, dv = forward_ad.make_dual(x, x), forward_ad.make_dual(v, v)
        one = torch.ones(32, 1, device=DEV)
        for call in (lambda: ops.group_norm(d, 4), lambda: ops.group_norm(x, 4, dv), lambda: ops.group_norm(x, 4, None, dv), lambda: ops.group_norm(x, 4, out=d),
                     lambda: ops.group_norm_fp8(d, 4), lambda: ops.quantize_fp8(d), lambda: ops.matmul_fp8(q, w, dv), lambda: ops.matmul_fp8(q, w, residual=d),
                     lambda: ops.Fp8Rows(q.values, forward_ad.make_dual(one, one))):
            with pytest.raises(E, match="tangent"):
                call()
        assert torch.equal(ops.group_norm(x, 4, v), ops.group_norm(x, 4, v))       # others' levels do not matter
    for trace in (lambda: torch.jit.trace(lambda x: ops.group_norm(x, 4), x), lambda: torch.func.vmap(lambda x: ops.quantize_fp8(x).values.float())(x[None]),
                  lambda: torch.jit.trace(lambda x: ops.matmul_fp8(q, w, residual=x), x)):
        with pytest.raises((E, RuntimeError)):
            trace()
    values = q.values.clone().requires_grad_()
    with pytest.raises(E, match="gradient"):
        ops.Fp8Rows(values, q.scale)
    with torch.no_grad():
        assert ops.Fp8Rows(values, q.scale).rows == 32
