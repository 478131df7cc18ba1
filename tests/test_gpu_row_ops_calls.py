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


def test_a_branch_keeps_what_it_reads_until_it_is_joined(ops):      # noqa: F811
    """Inputs that the caller drops while a branch on a side stream still reads them: their memory goes to nobody else before the join."""
    import gc
    import weakref
    from lssvc_amd.hip_ops import Fork
    g = gen(3)
    x, b = torch.randn(4000, 64, generator=g).to(DEV), torch.randn(64, generator=g).to(DEV)
    want = ops.group_norm(x, 4, None, b)
    w = ops.quantize_fp8(torch.randn(64, 64, generator=g).to(DEV), 128)
    q = ops.quantize_fp8(want)
    want = ops.matmul_fp8(q, w, b, residual=want)
    fork = Fork(torch.device(DEV), enabled=True, tag="row_ops")
    x, b, w = x.clone(), b.clone(), ops.quantize_fp8(w.dequantize(), 128)
    refs = [weakref.ref(x), weakref.ref(b), weakref.ref(w.values)]
    with fork.branch(0):
        y = ops.group_norm(x, 4, None, b)
        q = ops.quantize_fp8(y)
        refs.append(weakref.ref(y))
        y = ops.matmul_fp8(q, w, b, residual=y)
        del x, b, w, q
    gc.collect()
    assert all(r() is not None for r in refs)
    noise = [torch.full((4000, 64), float("nan"), device=DEV) for _ in range(4)]       # what would get the memory
    fork.join(0)
    gc.collect()
    assert all(r() is None for r in refs)
    assert torch.equal(y, want) and len(noise) == 4


def test_arguments_of_other_types(ops):          # noqa: F811
    """Numbers of any kind are taken; what is none is refused with the operators' own error."""
    import numpy as np
    x = torch.randn(32, 64, device=DEV)
    q, w = ops.quantize_fp8(x), ops.quantize_fp8(torch.randn(48, 64, device=DEV), 128)
    y = ops.group_norm(x, 4, eps=1.0, act="lrelu", slope=2.0, images=2)
    assert torch.equal(y, ops.group_norm(x, np.int32(4), eps=1, act="lrelu", slope=np.float32(2), images=np.int64(2)))
    for call in (lambda: ops.group_norm(x, 4.0), lambda: ops.group_norm(x, None), lambda: ops.group_norm(x, "4"), lambda: ops.group_norm(x, 4, images=1.5),
                 lambda: ops.group_norm(x, 4, eps=None), lambda: ops.group_norm(x, 4, eps=torch.tensor(1e-5, device=DEV)), lambda: ops.group_norm(x, 4, act=[]),
                 lambda: ops.group_norm(x, 4, slope="0.1"), lambda: ops.group_norm_fp8(x, 4.0), lambda: ops.quantize_fp8(x, 1.0), lambda: ops.quantize_fp8(x, None),
                 lambda: ops.matmul_fp8(q, w, slope=None), lambda: ops.matmul_fp8(q, w, act=1), lambda: ops.matmul_fp8(q, w, dtype="bf16"), lambda: ops.matmul_fp8(q, w, dtype=[]),
                 lambda: ops.matmul_fp8(q, w, out=torch.empty(32, 48, device=DEV), dtype=[]), lambda: ops.matmul_fp8(ops.Fp8Rows.empty(32, 64, "cpu"), w),
                 lambda: ops.matmul_fp8(q, ops.Fp8Rows.empty(48, 64, "cpu", 128)), lambda: ops.quantize_fp8(x, out=ops.Fp8Rows.empty(32, 64, "cpu")),
                 lambda: ops.Fp8Rows(q.values, q.scale, 1.0)):
        with pytest.raises(ops.LssvcHipError):
            call()
    assert torch.equal(ops.group_norm(x, 4, eps=1.0, act="lrelu", slope=2.0, images=2), y)


def test_on_a_torch_with_other_inner_names(ops, monkeypatch):      # noqa: F811
    from test_row_ops_calls import without_private_names
    other = without_private_names(monkeypatch)
    x = torch.randn(3000, 64, device=DEV)
    with torch.cuda.stream(torch.cuda.Stream()):
        torch.cuda.current_stream().wait_stream(torch.cuda.default_stream())
        y = other.group_norm(x, 4, act="silu")
    torch.cuda.synchronize()
    assert torch.equal(y, ops.group_norm(x, 4, act="silu"))


def test_wrappers_without_memory_are_refused(ops):         # noqa: F811
    """A tensor that only wraps others has the address 0, which to the library means no weight: it must not be left out in silence."""
    class Wrapper(torch.Tensor):
        @staticmethod
        def __new__(cls, t):
            return torch.Tensor._make_wrapper_subclass(cls, t.shape, strides=t.stride(), dtype=t.dtype, device=t.device)

        @classmethod
        def __torch_dispatch__(cls, f, types, args=(), kwargs=None):
            raise RuntimeError("not looked into")
    x, v = torch.randn(32, 64, device=DEV), torch.ones(64, device=DEV)
    q, w = ops.quantize_fp8(x), ops.quantize_fp8(torch.randn(64, 64, device=DEV), 128)
    wx, wv = Wrapper(x), Wrapper(v)
    for call in (lambda: ops.group_norm(x, 4, wv), lambda: ops.group_norm(x, 4, None, wv), lambda: ops.group_norm_fp8(x, 4, wv), lambda: ops.matmul_fp8(q, w, wv),
                 lambda: ops.group_norm(wx, 4), lambda: ops.quantize_fp8(wx), lambda: ops.matmul_fp8(q, w, residual=wx), lambda: ops.group_norm(x, 4, out=wx)):
        with pytest.raises((ops.LssvcHipError, RuntimeError)):
            call()
    with pytest.raises(ops.LssvcHipError, match="no memory of its own"):
        ops.group_norm(x, 4, wv)


def test_scales_with_room_behind_a_row(ops):               # noqa: F811
    """e8m0 scales of 2 and 5 blocks a row at a pitch of 4 and 8: read in place, whatever stands between the rows; without room for the last row's, copied."""
    g = gen(9)
    for m, n, k, pitch in ((40, 300, 200, 4), (1500, 1300, 600, 8), (1, 70, 130, 4)):
        q, w = ops.quantize_fp8(torch.randn(m, k, generator=g).to(DEV)), ops.quantize_fp8(torch.randn(n, k, generator=g).to(DEV), 128)
        want = ops.matmul_fp8(q, w)
        store = torch.full((m, pitch), 255, dtype=torch.uint8, device=DEV)               # (NaN, were it used)
        kb = q.scale.shape[1]
        store[:, :kb] = q.scale.contiguous().view(torch.uint8)
        scale = store.view(torch.float8_e8m0fnu)[:, :kb]
        a = ops.Fp8Rows(q.values, scale)
        assert a.scale.data_ptr() == store.data_ptr()
        assert torch.equal(ops.matmul_fp8(a, w), want)
        short = store.flatten()[:(m - 1) * pitch + kb].clone().as_strided((m, kb), (pitch, 1)).view(torch.float8_e8m0fnu)
        a = ops.Fp8Rows(q.values, short)
        assert a.scale.data_ptr() != short.data_ptr()
        assert torch.equal(ops.matmul_fp8(a, w), want)


@pytest.mark.parametrize("images,c,groups,dtype,fp8", [(2200000, 64, 8, torch.float32, False), (2200000, 1024, 64, torch.bfloat16, True), (1900000, 8200, 1, torch.float16, False)])
def test_more_images_than_a_launch_holds(ops, images, c, groups, dtype, fp8):       # noqa: F811
    """Every row an image of its own (a norm per pixel): more workgroups than a launch's threads can be counted for."""
    few = 1000
    rows = (torch.randn(few, c, generator=gen(c)) * 3 + 1).to(dtype).to(DEV)
    want = ops.group_norm_fp8(rows, groups, act="relu", images=few) if fp8 else ops.group_norm(rows, groups, act="relu", images=few)
    x = torch.empty(images, c, dtype=dtype, device=DEV)
    x.view(images // few, few, c)[:] = rows
    if fp8:
        q = ops.group_norm_fp8(x, groups, act="relu", images=images)
        same = lambda at: torch.equal(q.values[at].view(torch.uint8), want.values.view(torch.uint8)) and torch.equal(q.scale[at].view(torch.uint8), want.scale.view(torch.uint8))
    else:
        ops.group_norm(x, groups, act="relu", images=images, out=x)
        same = lambda at: torch.equal(x[at], want)
    for k in range(0, images // few, 50):
        assert same(slice(k * few, (k + 1) * few)), k
    assert same(slice(images - few, images))
