"""Row operators: group norm with an activation, 8-bit blocks, and the matrix product of 8-bit rows.

They work on ROWS of channels -- what a channels-last map of any batch is -- in fp32, fp16 or bf16, and serve transform blocks that
normalise over channel groups and take their pointwise products in 8 bits:

    q = row_ops.group_norm_fp8(x, 32, gamma, beta, act="silu", images=n)     # one pass: normalise, activate, 8-bit blocks
    h = row_ops.matmul_fp8(q, w1, b1, act="lrelu")                           # w1 = row_ops.quantize_fp8(weight, block_rows=128), once
    y = row_ops.matmul_fp8(row_ops.quantize_fp8(h), w2, b2, residual=x)

Rows are given as one of
    hip_ops.T                                   an H x W x C fp32 view (a slice of a wider buffer too)
    torch.Tensor (rows, C)                      any pitch between rows, channels adjacent
    torch.Tensor (N, C, H, W)                   torch.channels_last memory, or a channel slice of such a tensor
and come back as the same kind. Everything is enqueued on the current stream of the tensors' device; nothing synchronises. The
operators are forward operators (a tensor that requires a gradient is refused) and are not part of compiled frame plans.
"""
import ctypes as C

import torch

from . import _lib, hip_ops
from ._lib import LssvcHipError, Rows, Fp8, check, lib
from .hip_ops import T

BLOCK = 128                                   # columns that share a scale (and rows, in a weight)
_DTYPE = {torch.float32: _lib.F32, torch.float16: _lib.F16, torch.bfloat16: _lib.BF16}
_ACT = {None: _lib.ACT_NONE, "lrelu": _lib.ACT_LRELU, "relu": _lib.ACT_RELU, "silu": _lib.ACT_SILU}
_E4M3, _E8M0 = torch.float8_e4m3fn, torch.float8_e8m0fnu


def _refuse(what, *args):
    raise LssvcHipError(what % args)


def _no_grad(x, name):
    if x.requires_grad and torch.is_grad_enabled():
        _refuse("row_ops: %s requires a gradient and these operators have none (use torch.no_grad() or detach())", name)


def _rows(x, name):
    """-> the lssvc_rows of a T or tensor."""
    if isinstance(x, T):
        if x.split:
            _refuse("row_ops: %s is a pre-split view", name)
        v = x.v
        return Rows(v.ptr, x.H * x.W, x.ld, x.C, _lib.F32)
    if not isinstance(x, torch.Tensor):
        _refuse("row_ops: %s is neither a T nor a tensor: %s", name, type(x).__name__)
    dt = _DTYPE.get(x.dtype)
    if dt is None:
        _refuse("row_ops: %s has type %s (fp32, fp16 or bf16 expected)", name, x.dtype)
    if not x.is_cuda:
        _refuse("row_ops: %s is on %s: there is no CPU path", name, x.device)
    _no_grad(x, name)
    if x.dim() == 2:
        rows, cols = x.shape
        ld, step = x.stride()
        if (step != 1 and cols > 1) or (ld < cols and rows > 1):
            _refuse("row_ops: the channels of %s are not adjacent (strides %s)", name, tuple(x.stride()))
        return Rows(x.data_ptr(), rows, ld if rows > 1 else cols, cols, dt)
    if x.dim() == 4:
        n, c, h, w = x.shape
        sn, sc, sh, sw = x.stride()
        ld = sw if w > 1 else sh if h > 1 else sn if n > 1 else c
        if (sc != 1 and c > 1) or ld < c or (h > 1 and sh != w * ld) or (n > 1 and sn != h * w * ld):
            _refuse("row_ops: %s is not channels-last (shape %s, strides %s)", name, tuple(x.shape), tuple(x.stride()))
        return Rows(x.data_ptr(), n * h * w, ld, c, dt)
    _refuse("row_ops: %s has %d dimensions (rows x channels, or N x C x H x W)", name, x.dim())


def _vector(x, name, n, device):
    if x is None:
        return None
    if not (isinstance(x, torch.Tensor) and x.dtype == torch.float32 and x.dim() == 1 and x.shape[0] == n and (n == 1 or x.stride(0) == 1) and x.device == device):
        _refuse("row_ops: %s has to be %d adjacent fp32 values on %s", name, n, device)
    _no_grad(x, name)
    return x.data_ptr()


def _act_code(act):
    code = _ACT.get(act)
    if code is None:
        _refuse("row_ops: unknown activation %r (None, 'lrelu', 'relu', 'silu')", act)
    return code


class _On:
    """The launch context of one call: the tensors' device is made current if it is not."""
    __slots__ = ("guard",)

    def __init__(self, device):
        if hip_ops.PLAN_RECORDER is not None:
            _refuse("row_ops: not part of compiled frame plans")
        self.guard = None if device.index == torch.cuda.current_device() else torch.cuda.device(device)

    def __enter__(self):
        if self.guard is not None:
            self.guard.__enter__()

    def __exit__(self, *exc):
        if self.guard is not None:
            self.guard.__exit__(*exc)
        return False


def _same_device(device, **others):
    for name, x in others.items():
        if x is not None and x.device != device:
            _refuse("row_ops: %s is on %s, the input on %s", name, x.device, device)


class Fp8Rows:
    """8-bit rows (OCP e4m3) with a scale for each block of `block_rows` x 128 values: 1 for activations, 128 for weights.

    values  (rows, cols) torch.float8_e4m3fn
    scale   (ceil(rows / block_rows), ceil(cols / 128)): torch.float8_e8m0fnu (powers of two: what quantize_fp8 makes, and the faster
            product) or torch.float32 (any scale, e.g. a checkpoint's)

    Tensors that the kernels can read as they are stay where they are; others (columns that are no multiple of 16, odd pitches or
    bases) are copied once, here, into rows with zeros behind the last column."""
    __slots__ = ("values", "scale", "rows", "cols", "block_rows", "_c", "_keep")

    def __init__(self, values, scale, block_rows=1):
        if not isinstance(values, torch.Tensor) or values.dtype != _E4M3 or values.dim() != 2 or not values.is_cuda:
            _refuse("Fp8Rows: values have to be a (rows, cols) torch.float8_e4m3fn tensor on the GPU")
        if not isinstance(scale, torch.Tensor) or scale.dtype not in (_E8M0, torch.float32) or scale.dim() != 2 or scale.device != values.device:
            _refuse("Fp8Rows: scale has to be a 2-d torch.float8_e8m0fnu or torch.float32 tensor on the values' device")
        if block_rows not in (1, BLOCK):
            _refuse("Fp8Rows: block_rows is 1 or %d, got %r", BLOCK, block_rows)
        rows, cols = values.shape
        want = (-(-rows // block_rows), -(-cols // BLOCK))
        if cols < 1 or tuple(scale.shape) != want:
            _refuse("Fp8Rows: scale is %s, expected %s for %d x %d values in %d x %d blocks", tuple(scale.shape), want, rows, cols, block_rows, BLOCK)
        _no_grad(scale, "scale")
        if rows and not (cols % 16 == 0 and values.stride(1) == 1 and (rows == 1 or values.stride(0) % 16 == 0 and values.stride(0) >= cols) and values.data_ptr() % 16 == 0):
            values = _padded(values, 16)
        if rows and scale.dtype == _E8M0 and not (want[1] % 4 == 0 and scale.stride(1) == 1 and scale.data_ptr() % 4 == 0
                                                  and (want[0] == 1 or scale.stride(0) % 4 == 0 and scale.stride(0) >= want[1])):
            scale = _padded(scale, 4)
        elif rows and scale.dtype == torch.float32 and not ((scale.stride(1) == 1 or want[1] == 1) and (want[0] == 1 or scale.stride(0) >= want[1])):
            scale = scale.contiguous()
        self._set(values, scale, block_rows)

    def _set(self, values, scale, block_rows):
        rows, cols = values.shape
        kb = -(-cols // BLOCK)
        self.values, self.scale, self.rows, self.cols, self.block_rows = values, scale, rows, cols, block_rows
        e8m0 = scale.dtype == _E8M0
        ld = values.stride(0) if rows > 1 else -(-cols // 16) * 16
        sld = scale.stride(0) if scale.shape[0] > 1 else (-(-kb // 4) * 4 if e8m0 else kb)
        self._c = Fp8(values.data_ptr(), scale.data_ptr(), rows, ld, sld, cols, block_rows, 1 if e8m0 else 0, 0)

    @property
    def device(self):
        return self.values.device

    @staticmethod
    def empty(rows, cols, device, block_rows=1):
        """Uninitialised rows with e8m0 scales, for `out=` of the operators that write 8-bit rows."""
        if block_rows not in (1, BLOCK):
            _refuse("Fp8Rows: block_rows is 1 or %d, got %r", BLOCK, block_rows)
        if rows < 0 or cols < 1:
            _refuse("Fp8Rows: %d x %d values", rows, cols)
        ld, br, kb = -(-cols // 16) * 16, -(-rows // block_rows), -(-cols // BLOCK)
        values = torch.empty(rows, ld, dtype=_E4M3, device=device)
        scale = torch.empty(br, -(-kb // 4) * 4, dtype=_E8M0, device=device)
        self = Fp8Rows.__new__(Fp8Rows)
        self._set(values[:, :cols] if ld != cols else values, scale[:, :kb] if scale.shape[1] != kb else scale, block_rows)
        return self

    def dequantize(self, dtype=torch.float32):
        """The (rows, cols) values the blocks stand for, in plain torch operations (for inspection and tests)."""
        s = self.scale.contiguous()
        s = s if s.dtype == torch.float32 else (s.view(torch.uint8).to(torch.int32) << 23).view(torch.float32)
        s = s.repeat_interleave(self.block_rows, 0)[:self.rows].repeat_interleave(BLOCK, 1)[:, :self.cols]
        return (self.values.float() * s).to(dtype)


def _padded(x, to):
    """A copy of 8-bit rows in a buffer whose pitch is the next multiple of `to` bytes, zeros behind the last column."""
    store = torch.zeros(x.shape[0], -(-x.shape[1] // to) * to, dtype=torch.uint8, device=x.device)
    store[:, :x.shape[1]] = x.contiguous().view(torch.uint8)
    return store.view(x.dtype)[:, :x.shape[1]]


def _empty_like(x, rows, cols, dtype):
    if isinstance(x, T):
        return T.empty(x.H, x.W, cols, x.device)
    if x.dim() == 4:
        return torch.empty((x.shape[0], cols, x.shape[2], x.shape[3]), dtype=dtype, device=x.device, memory_format=torch.channels_last)
    return torch.empty((rows, cols), dtype=dtype, device=x.device)


def _fp8_out(out, rows, cols, device, block_rows):
    if out is None:
        return Fp8Rows.empty(rows, cols, device, block_rows)
    if not isinstance(out, Fp8Rows) or out.rows != rows or out.cols != cols or out.block_rows != block_rows:
        _refuse("row_ops: out has to be Fp8Rows.empty(%d, %d, device, block_rows=%d)", rows, cols, block_rows)
    _same_device(device, out=out)
    return out


def _stream(device):
    return torch.cuda.current_stream(device).cuda_stream


def _group_norm(x, groups, weight, bias, eps, act, slope, images, out, fp8):
    xr = _rows(x, "x")
    dev = x.device
    if images is None:
        images = x.shape[0] if not isinstance(x, T) and x.dim() == 4 else 1
    elif not isinstance(x, T) and x.dim() == 4 and images != x.shape[0]:
        _refuse("group_norm: images=%d, but x has %d", images, x.shape[0])
    code = _act_code(act)
    wp, bp = _vector(weight, "weight", xr.cols, dev), _vector(bias, "bias", xr.cols, dev)
    with _On(dev):
        if fp8:
            out = _fp8_out(out, xr.rows, xr.cols, dev, 1)
            yr, y8 = None, C.byref(out._c)
        else:
            if out is None:
                out = _empty_like(x, xr.rows, xr.cols, getattr(x, "dtype", None))
            _same_device(dev, out=out)
            yr, y8 = C.byref(_rows(out, "out")), None
        if xr.rows == 0:
            images = 1
        need = lib.lssvc_group_norm_workspace_bytes(xr.rows, images, xr.cols, groups, xr.dtype, 1 if fp8 else 0)
        ws = torch.empty(need, dtype=torch.uint8, device=dev) if need else None
        check(lib.lssvc_group_norm(C.byref(xr), images, groups, wp, bp, eps, code, slope, yr, y8,
                                   ws.data_ptr() if need else None, need, _stream(dev)))
    return out


def group_norm(x, groups, weight=None, bias=None, *, eps=1e-5, act=None, slope=0.01, images=None, out=None):
    """act(group_norm(x)): statistics over the rows of each of `images` images and the C / groups channels of a group, in fp32;
    weight / bias: C fp32 values. images: for 2-d rows and T (default 1); a 4-d tensor brings its own. out: rows of x's shape and type,
    x itself allowed. act: None, 'lrelu' (slope), 'relu', 'silu'."""
    return _group_norm(x, groups, weight, bias, eps, act, slope, images, out, False)


def group_norm_fp8(x, groups, weight=None, bias=None, *, eps=1e-5, act=None, slope=0.01, images=None, out=None):
    """quantize_fp8(act(group_norm(x))) in the pass that normalises: the fp32 result goes into 1 x 128 blocks and is not written itself."""
    return _group_norm(x, groups, weight, bias, eps, act, slope, images, out, True)


def quantize_fp8(x, block_rows=1, out=None):
    """x as 8-bit blocks: block_rows=1 (1 x 128) for activations, 128 (128 x 128) for weights. Of each block the scale is the smallest
    power of two s >= 2^-126 with max |x| <= 448 s (1 for a block of zeros), values are e4m3(x / s) to nearest even. A value that is not
    finite becomes NaN and does not move the scale."""
    xr = _rows(x, "x")
    if block_rows not in (1, BLOCK):
        _refuse("quantize_fp8: block_rows is 1 or %d, got %r", BLOCK, block_rows)
    with _On(x.device):
        out = _fp8_out(out, xr.rows, xr.cols, x.device, block_rows)
        check(lib.lssvc_quantize_fp8(C.byref(xr), C.byref(out._c), _stream(x.device)))
    return out


def matmul_fp8(a, w, bias=None, *, act=None, slope=0.01, residual=None, out=None, dtype=None):
    """act(a @ w.T + bias) + residual. a: Fp8Rows (M, K) of 1 x 128 blocks; w: Fp8Rows (N, K) of 128 x 128 blocks; both with e8m0 or both
    with fp32 scales. Sums in fp32, one rounding to the output's type. bias: N fp32 values. residual, out: M rows of N channels
    (residual may be out). dtype: the output's type; by default that of out or residual, or bf16."""
    if not isinstance(a, Fp8Rows) or not isinstance(w, Fp8Rows):
        _refuse("matmul_fp8: operands are Fp8Rows (quantize_fp8, group_norm_fp8)")
    dev = a.values.device
    m, n = a.rows, w.rows
    code = _act_code(act)
    bp = _vector(bias, "bias", n, dev)
    rr = None
    if residual is not None:
        rr = _rows(residual, "residual")
    with _On(dev):
        if out is None:
            if dtype is None:
                dtype = torch.bfloat16 if residual is None else torch.float32 if isinstance(residual, T) else residual.dtype
            if residual is not None:
                out = _empty_like(residual, m, n, dtype)
            else:
                out = torch.empty((m, n), dtype=dtype, device=dev)
        yr = _rows(out, "out")
        if dtype is not None and _DTYPE.get(dtype) != yr.dtype:
            _refuse("matmul_fp8: dtype %s is not the output's", dtype)
        _same_device(dev, w=w, out=out, residual=residual)
        need = lib.lssvc_matmul_fp8_workspace_bytes(m, n, a.cols)
        ws = torch.empty(need, dtype=torch.uint8, device=dev) if need else None
        check(lib.lssvc_matmul_fp8(C.byref(a._c), C.byref(w._c), bp, code, slope, C.byref(rr) if rr is not None else None, C.byref(yr),
                                   ws.data_ptr() if need else None, need, _stream(dev)))
    return out
