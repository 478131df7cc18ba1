"""What the row operators refuse is refused on the host, before anything is launched: these calls need no GPU."""
import ctypes as C

import pytest
import torch

from row_ops_ref import quantize64


def rows(ptr=4096, rows=8, ld=64, cols=64, dtype=0):
    from lssvc_amd import _lib
    return C.byref(_lib.Rows(ptr, rows, ld, cols, dtype))


def fp8(values=4096, scale=8192, rows=8, ld=64, scale_ld=4, cols=64, block_rows=1, e8m0=1, reserved=0):
    from lssvc_amd import _lib
    return C.byref(_lib.Fp8(values, scale, rows, ld, scale_ld, cols, block_rows, e8m0, reserved))


def refused(rc, text):
    from lssvc_amd import _lib
    assert rc != 0
    assert text in _lib.lib.lssvc_last_error().decode(), _lib.lib.lssvc_last_error()


def norm(x=None, images=1, groups=4, eps=1e-5, act=0, y="same", y8=None, ws=None, nws=0):
    from lssvc_amd import _lib
    x = rows() if x is None else x
    y = rows(ptr=1 << 20) if y == "same" else y
    return _lib.lib.lssvc_group_norm(x, images, groups, None, None, eps, act, 0.01, y, y8, ws, nws, None)


def test_group_norm_refusals():
    refused(norm(images=3), "images")
    refused(norm(images=0), "images")
    refused(norm(groups=5), "groups")
    refused(norm(groups=0), "groups")
    refused(norm(groups=-4), "groups")
    refused(norm(eps=-1.0), "eps")
    refused(norm(eps=float("nan")), "eps")
    refused(norm(act=4), "activation")
    refused(norm(y=None), "exactly one")
    refused(norm(y8=fp8()), "exactly one")
    refused(norm(x=rows(dtype=3)), "type")
    refused(norm(x=rows(ptr=4098)), "aligned")
    refused(norm(x=rows(ld=63)), "bad rows")
    refused(norm(x=rows(cols=0)), "bad rows")
    refused(norm(x=rows(rows=-1)), "bad rows")
    refused(norm(x=rows(ptr=0)), "bad rows")
    refused(norm(y=rows(ptr=1 << 20, rows=7)), "shape")
    refused(norm(y=rows(ptr=1 << 20, dtype=1)), "shape")
    refused(norm(y=rows(ptr=4096 + 256)), "overlap")                     # one row later
    refused(norm(x=rows(ld=128), y=rows(ptr=4096 + 4, ld=128)), "overlap")
    refused(norm(y=None, y8=fp8(cols=63)), "8-bit output is")
    refused(norm(y=None, y8=fp8(ld=72)), "multiple of 16")
    refused(norm(y=None, y8=fp8(values=4104)), "16-byte aligned")
    refused(norm(y=None, y8=fp8(scale_ld=3)), "multiple of 4")
    refused(norm(y=None, y8=fp8(e8m0=0)), "e8m0")
    refused(norm(y=None, y8=fp8(block_rows=128)), "1 x 128")
    refused(norm(y=None, y8=fp8(values=4096 + 2032)), "overlaps an input")
    refused(norm(y=None, y8=fp8(values=1 << 20, scale=4100)), "overlaps an input")
    refused(norm(x=rows(ld=1 << 32)), "out of range")
    big = rows(rows=1 << 20)
    refused(norm(x=big, y=rows(ptr=1 << 30, rows=1 << 20)), "workspace")
    refused(norm(x=big, y=rows(ptr=1 << 30, rows=1 << 20), ws=1 << 29, nws=64), "workspace")
    refused(norm(x=big, y=rows(ptr=1 << 30, rows=1 << 20), ws=(1 << 30) + 4096, nws=1 << 30), "overlaps")
    refused(norm(x=big, y=rows(ptr=1 << 30, rows=1 << 20), ws=8192, nws=1 << 30), "overlaps")


def test_group_norm_workspace_size():
    from lssvc_amd import _lib
    size = _lib.lib.lssvc_group_norm_workspace_bytes
    assert size(540, 1, 64, 8, 0, 0) == 0                                # held by the workgroups
    assert size(1 << 20, 1, 64, 8, 0, 0) > 0
    for bad in ((0, 1, 64, 8, 0, 0), (10, 3, 64, 8, 0, 0), (10, 1, 64, 7, 0, 0), (10, 1, 64, 8, 9, 0), (10, 0, 64, 8, 0, 0)):
        assert size(*bad) == 0


def test_quantize_refusals():
    from lssvc_amd import _lib
    q = lambda x, y: _lib.lib.lssvc_quantize_fp8(x, y, None)
    refused(q(rows(rows=7), fp8()), "8-bit output is")
    refused(q(rows(), fp8(block_rows=64)), "block_rows")
    refused(q(rows(dtype=7), fp8()), "type")
    refused(q(rows(ptr=4097), fp8()), "aligned")
    refused(q(rows(), fp8(scale=8193)), "4-byte")
    refused(q(rows(), fp8(scale=0)), "no 8-bit output")
    refused(q(rows(), fp8(reserved=1)), "e8m0")
    refused(q(rows(ptr=4096), fp8()), "overlap")
    refused(q(rows(ptr=8192 - 2044), fp8(values=1 << 20)), "overlap")                 # the scales, by four bytes
    refused(q(rows(ptr=1 << 20), fp8(values=8192 - 512 + 16)), "overlap")             # values and scales
    refused(q(rows(cols=(1 << 30) + 1, ld=1 << 31), fp8()), "out of range")


def test_matmul_refusals():
    from lssvc_amd import _lib
    f = lambda a=None, w=None, act=0, res=None, y=None: _lib.lib.lssvc_matmul_fp8(
        a or fp8(), w or fp8(rows=32, block_rows=128), None, act, 0.01, res, y or rows(ptr=1 << 20, cols=32, ld=32), None)
    refused(f(w=fp8(rows=32)), "scales for 1 rows")
    refused(f(a=fp8(block_rows=128)), "scales for 128 rows")
    refused(f(w=fp8(rows=32, cols=63, block_rows=128)), "columns")
    refused(f(w=fp8(rows=32, block_rows=128, e8m0=0)), "e8m0")
    refused(f(w=fp8(rows=0, block_rows=128)), "no rows")
    refused(f(act=9), "activation")
    refused(f(y=rows(ptr=1 << 20, cols=33, ld=40)), "output")
    refused(f(y=rows(ptr=1 << 20, cols=32, ld=31)), "bad rows")
    refused(f(y=rows(ptr=1 << 20, cols=32, ld=32, dtype=5)), "type")
    refused(f(y=rows(ptr=0, cols=32, ld=32)), "bad rows")
    refused(f(y=rows(ptr=(1 << 20) + 2, cols=32, ld=32)), "aligned")
    refused(f(y=rows(ptr=4096 + 256, cols=32, ld=32)), "overlaps an operand")         # the values of a and w
    refused(f(y=rows(ptr=8192, cols=32, ld=32)), "overlaps an operand")               # their scales
    refused(f(res=rows(ptr=(1 << 22) + 2, cols=32, ld=32)), "aligned")
    refused(f(a=fp8(rows=1 << 31), y=rows(ptr=1 << 20, rows=1 << 31, cols=32, ld=32)), "too large")
    refused(f(a=fp8(ld=1 << 22)), "too large")
    refused(f(res=rows(ptr=1 << 22, cols=31, ld=32)), "residual")
    refused(f(res=rows(ptr=1 << 22, cols=32, ld=32, dtype=1)), "residual")
    refused(f(res=rows(ptr=(1 << 20) + 64, cols=32, ld=32)), "overlap")
    refused(f(a=fp8(ld=72)), "multiple of 16")
    refused(f(a=fp8(ld=48)), "multiple of 16")
    refused(f(a=fp8(values=4100)), "16-byte")
    refused(f(a=fp8(scale_ld=2)), "scale layout")
    refused(f(a=fp8(scale_ld=0, e8m0=0)), "scale layout")
    refused(f(a=fp8(values=0)), "no data")
    refused(f(a=fp8(cols=0)), "bad operand")


def test_python_refusals_without_a_gpu():
    from lssvc_amd import row_ops
    E = row_ops.LssvcHipError
    x = torch.randn(8, 64)
    for call in (lambda: row_ops.group_norm(x, 4), lambda: row_ops.quantize_fp8(x), lambda: row_ops.group_norm("x", 4), lambda: row_ops.matmul_fp8(x, x),
                 lambda: row_ops.Fp8Rows(x, x), lambda: row_ops.Fp8Rows(x.to(torch.float8_e4m3fn), torch.ones(8, 1)), lambda: row_ops.Fp8Rows.empty(4, 0, "cpu"),
                 lambda: row_ops.Fp8Rows.empty(4, 4, "cpu", 2)):
        with pytest.raises(E):
            call()
    q = row_ops.Fp8Rows.empty(5, 40, "cpu")
    assert q.values.shape == (5, 40) and q.values.stride(0) == 48 and q.scale.shape == (5, 1) and q.scale.stride(0) == 4


def test_reference_quantiser_on_known_values():
    """The test-side definition itself: maxima at the border of two scales, ties, subnormals."""
    x = torch.zeros(4, 128)
    x[0, 0], x[1, 0], x[2, 0], x[3, 0] = 448.0, 449.0, 1.0, 1e-45
    x[0, 1:5] = torch.tensor([17.0, 19.0, 2.0 ** -10, 3 * 2.0 ** -10])       # ties: 16 / 20, 0 / 2^-8
    v, e = quantize64(x, 1)
    assert e.flatten().tolist() == [0, 1, -8, -126]
    assert v[0, :5].tolist() == [448, 16, 20, 0, 2.0 ** -8] and v[1, 0] == 224 and v[2, 0] == 256
