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
operators are forward operators: a tensor that requires a gradient or carries a forward-mode tangent is refused, and so is a call inside
torch.jit.trace, make_fx or a torch.func transform. They are not part of compiled frame plans.
"""
import functools
import operator
import sys

import torch
from torch.autograd import forward_ad

from . import _lib, hip_ops
from ._lib import LssvcHipError, Rows, Fp8, check, lib
from .hip_ops import T

BLOCK = 128                                   # columns that share a scale (and rows, in a weight)
_DTYPE = {torch.float32: _lib.F32, torch.float16: _lib.F16, torch.bfloat16: _lib.BF16}
_ACT = {None: _lib.ACT_NONE, "lrelu": _lib.ACT_LRELU, "relu": _lib.ACT_RELU, "silu": _lib.ACT_SILU}
_MAX_COLS = 1 << 30
_E4M3, _E8M0 = torch.float8_e4m3fn, torch.float8_e8m0fnu


def _refuse(what, *args):
    raise LssvcHipError(what % args)


def _no_grad(x, name):
    if x.requires_grad and torch.is_grad_enabled():
        _refuse("row_ops: %s requires a gradient and these operators have none (use torch.no_grad() or detach())", name)


def _no_tangent(*tensors):
    """For calls inside a level of forward-mode differentiation, where x.requires_grad says nothing."""
    for x in tensors:
        if isinstance(x, torch.Tensor) and forward_ad.unpack_dual(x).tangent is not None:
            _refuse("row_ops: a tensor carries a forward-mode tangent and these operators have no derivative")


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
    if dt is None or x.layout is not torch.strided:
        _refuse("row_ops: %s has type %s (fp32, fp16 or bf16 expected)", name, x.dtype)
    if not x.is_cuda:
        _refuse("row_ops: %s is on %s: there is no CPU path", name, x.device)
    if x.requires_grad:
        _no_grad(x, name)
    shape = x.shape
    if len(shape) == 2:
        rows, cols = shape
        ld, step = x.stride()
        if (step != 1 and cols > 1) or (ld < cols and rows > 1):
            _refuse("row_ops: the channels of %s are not adjacent (strides %s)", name, tuple(x.stride()))
        if cols > _MAX_COLS:
            _refuse("row_ops: %s has %d channels", name, cols)
        return Rows(x.data_ptr(), rows, ld if rows > 1 else cols, cols, dt)
    if len(shape) == 4:
        n, c, h, w = shape
        sn, sc, sh, sw = x.stride()
        ld = sw if w > 1 else sh if h > 1 else sn if n > 1 else c
        if (sc != 1 and c > 1) or ld < c or (h > 1 and sh != w * ld) or (n > 1 and sn != h * w * ld):
            _refuse("row_ops: %s is not channels-last (shape %s, strides %s)", name, tuple(x.shape), tuple(x.stride()))
        if c > _MAX_COLS:
            _refuse("row_ops: %s has %d channels", name, c)
        return Rows(x.data_ptr(), n * h * w, ld, c, dt)
    _refuse("row_ops: %s has %d dimensions (rows x channels, or N x C x H x W)", name, x.dim())


def _vector(x, name, n, device):
    if not (isinstance(x, torch.Tensor) and x.dtype is torch.float32 and x.shape == (n,) and x.is_contiguous() and x.is_cuda and x.get_device() == device.index):
        _refuse("row_ops: %s has to be %d adjacent fp32 values on %s", name, n, device)
    if x.requires_grad:
        _no_grad(x, name)
    p = x.data_ptr()
    if not p:                                                      # (a wrapper of another tensor; no address would mean no weight)
        _refuse("row_ops: %s has no memory of its own: %s", name, type(x).__name__)
    return p


def _whole(v, name):
    try:
        return operator.index(v)
    except TypeError:
        _refuse("row_ops: %s has to be a whole number, got %r", name, v)


def _number(v, name):
    if isinstance(v, torch.Tensor):
        _refuse("row_ops: %s has to be a number, not a tensor (which would have to be waited for)", name)
    try:
        if not isinstance(v, str):
            return float(v)
    except (TypeError, ValueError):
        pass
    _refuse("row_ops: %s has to be a number, got %r", name, v)


def _act_code(act):
    code = _ACT.get(act) if act is None or isinstance(act, str) else None
    if code is None:
        _refuse("row_ops: unknown activation %r (None, 'lrelu', 'relu', 'silu')", act)
    return code


# torch.cuda.current_stream(device).cuda_stream without the Stream object, torch.cuda.current_device() without its look at whether the GPU is in
# use already (a tensor on it says so): 1.3 us of a call's 6 to 8. Both are names inside torch: a torch without them has the public ones.
_raw_stream = getattr(torch._C, "_cuda_getCurrentRawStream", None) or (lambda index: torch.cuda.current_stream(index).cuda_stream)
_current_device = getattr(torch._C, "_cuda_getDevice", None) or torch.cuda.current_device


# who else may be watching: a trace or transform sees a call's allocations and not its launches, and what it makes of them would be wrong without an
# error. (All four looks together: 0.2 us.)
_tracing = getattr(torch._C, "_is_tracing", torch.jit.is_tracing)
_transform = getattr(getattr(torch._C, "_functorch", None), "peek_interpreter_stack", lambda: None)
_modes = getattr(torch._C, "_len_torch_dispatch_stack", lambda: 0)


def _no_proxies():
    proxies = sys.modules.get("torch.fx.experimental.proxy_tensor")
    return proxies is None or proxies.get_proxy_mode() is None


def _elsewhere(device, *tensors):
    """Whether `device` has to be made current for a call (every entry point does that around itself). tensors: what the caller gave; in a branch of
    hip_ops.Fork they are alive until it is joined, as the engine's views are."""
    keep = hip_ops._TLS.keep
    if keep is not None:
        keep.extend(tensors)
    if _tracing() or _transform() is not None or _modes() and not _no_proxies():
        _refuse("row_ops: these operators cannot be traced or transformed (torch.jit.trace, make_fx, torch.func)")
    if getattr(forward_ad, "_current_level", 0) >= 0:              # (not known: look)
        _no_tangent(*tensors)
    if hip_ops.recording():
        _refuse("row_ops: not part of compiled frame plans")
    if device.index is None:
        _refuse("row_ops: operands on %s: there is no CPU path", device)
    return device.index != _current_device()


class Fp8Rows:
    """8-bit rows (OCP e4m3) with a scale for each block of `block_rows` x 128 values: 1 for activations, 128 for weights.

    values  (rows, cols) torch.float8_e4m3fn
    scale   (ceil(rows / block_rows), ceil(cols / 128)): torch.float8_e8m0fnu (powers of two: what quantize_fp8 makes, and the faster
            product) or torch.float32 (any scale, e.g. a checkpoint's)

    Tensors that the kernels can read as they are stay where they are: values of a multiple of 16 columns, their base and the pitch multiples
    of 16 (a pitch that is a multiple of 128 is up to 1.9x faster in the product); fp32 scales; e8m0 scales at a base and a pitch that are multiples
    of 4, with memory up to the last row's next one. Others are copied once, here, into rows with zeros behind the last column."""
    __slots__ = ("_values", "_scale", "_store", "rows", "cols", "block_rows", "device", "_c")

    def __init__(self, values, scale, block_rows=1):
        if not isinstance(values, torch.Tensor) or values.dtype != _E4M3 or values.dim() != 2 or not values.is_cuda:
            _refuse("Fp8Rows: values have to be a (rows, cols) torch.float8_e4m3fn tensor on the GPU")
        if not isinstance(scale, torch.Tensor) or scale.dtype not in (_E8M0, torch.float32) or scale.dim() != 2 or scale.device != values.device:
            _refuse("Fp8Rows: scale has to be a 2-d torch.float8_e8m0fnu or torch.float32 tensor on the values' device")
        block_rows = _whole(block_rows, "block_rows")
        if block_rows not in (1, BLOCK):
            _refuse("Fp8Rows: block_rows is 1 or %d, got %r", BLOCK, block_rows)
        rows, cols = values.shape
        want = (-(-rows // block_rows), -(-cols // BLOCK))
        if not 1 <= cols <= _MAX_COLS or tuple(scale.shape) != want:
            _refuse("Fp8Rows: scale is %s, expected %s for %d x %d values in %d x %d blocks", tuple(scale.shape), want, rows, cols, block_rows, BLOCK)
        _no_grad(scale, "scale")
        _no_grad(values, "values")
        _no_tangent(scale, values)
        if rows and not (cols % 16 == 0 and values.stride(1) == 1 and (rows == 1 or values.stride(0) % 16 == 0 and values.stride(0) >= cols) and values.data_ptr() % 16 == 0):
            values = _padded(values, _pitch(cols))
        if rows and scale.dtype == _E8M0 and not _whole_dwords(scale):
            scale = _padded(scale, -(-want[1] // 4) * 4)
        elif rows and scale.dtype == torch.float32 and not ((scale.stride(1) == 1 or want[1] == 1) and (want[0] == 1 or scale.stride(0) >= want[1])):
            scale = scale.contiguous()
        self._set(values, scale, block_rows)

    def _set(self, values, scale, block_rows):
        rows, cols = values.shape
        kb = -(-cols // BLOCK)
        self._values, self._scale, self.rows, self.cols, self.block_rows, self.device = values, scale, rows, cols, block_rows, values.device
        e8m0 = scale.dtype == _E8M0
        ld = values.stride(0) if rows > 1 else _pitch(cols)
        sld = scale.stride(0) if scale.shape[0] > 1 else (-(-kb // 4) * 4 if e8m0 else kb)
        self._c = Fp8(values.data_ptr(), scale.data_ptr(), rows, ld, sld, cols, block_rows, 1 if e8m0 else 0, 0)
        self._store = None

    # values and scale of operands that the kernels made live in one buffer and become tensors when somebody looks
    @property
    def values(self):
        if self._values is None:
            self._values = self._store.view(_E4M3).as_strided((self.rows, self.cols), (self._c.ld, 1))
        return self._values

    @property
    def scale(self):
        if self._scale is None:
            self._scale = self._store.view(_E8M0).as_strided((-(-self.rows // self.block_rows), -(-self.cols // BLOCK)), (self._c.scale_ld, 1), self.rows * self._c.ld)
        return self._scale

    @staticmethod
    def empty(rows, cols, device, block_rows=1):
        """Uninitialised rows with e8m0 scales, for `out=` of the operators that write 8-bit rows."""
        rows, cols, block_rows = _whole(rows, "rows"), _whole(cols, "cols"), _whole(block_rows, "block_rows")
        if block_rows != 1 and block_rows != BLOCK:
            _refuse("Fp8Rows: block_rows is 1 or %d, got %r", BLOCK, block_rows)
        if rows < 0 or not 1 <= cols <= _MAX_COLS:
            _refuse("Fp8Rows: %d x %d values", rows, cols)
        ld, sld = _pitch(cols), -(-cols // (4 * BLOCK)) * 4
        nbytes = rows * ld
        self = Fp8Rows.__new__(Fp8Rows)
        self._store = store = torch.empty(nbytes + -(-rows // block_rows) * sld, dtype=torch.uint8, device=device)
        self._values = self._scale = None
        self.rows, self.cols, self.block_rows, self.device = rows, cols, block_rows, store.device
        ptr = store.data_ptr()
        self._c = Fp8(ptr, ptr + nbytes, rows, ld, sld, cols, block_rows, 1, 0)
        return self

    def dequantize(self, dtype=torch.float32):
        """The (rows, cols) values the blocks stand for, in plain torch operations (for inspection and tests)."""
        s = self.scale.contiguous()
        if s.dtype != torch.float32:                               # 2^(b - 127) is the exponent field, but for the ends of the range
            b = s.view(torch.uint8).to(torch.int32)
            s = torch.where(b == 0, 0x400000, torch.where(b == 255, 0x7fc00000, b << 23)).to(torch.int32).view(torch.float32)
        s = s.repeat_interleave(self.block_rows, 0)[:self.rows].repeat_interleave(BLOCK, 1)[:, :self.cols]
        return (self.values.float() * s).to(dtype)


def _pitch(cols):
    """Bytes between rows of 8-bit values: whole 128-byte lines per block of K (a block that straddles two lines costs the product up to
    1.9x: 1362 x 553 x 5993 44 us at a pitch of 6000, 25 us at 6016); short rows stay close together."""
    return -(-cols // 16) * 16 if cols <= BLOCK else -(-cols // BLOCK) * BLOCK


def _whole_dwords(scale):
    """Whether e8m0 scales can be read four at a time where they lie (the bytes behind a row's last scale are read and not used)."""
    rows, kb = scale.shape
    ld, step = scale.stride()
    if step != 1 and kb > 1 or rows > 1 and (ld % 4 or ld < kb) or scale.data_ptr() % 4:
        return False
    return scale.untyped_storage().nbytes() - scale.storage_offset() >= (rows - 1) * ld * (rows > 1) + -(-kb // 4) * 4


def _padded(x, pitch):
    """A copy of 8-bit rows in a buffer with `pitch` bytes between rows, zeros behind the last column."""
    store = torch.zeros(x.shape[0], pitch, dtype=torch.uint8, device=x.device)
    store[:, :x.shape[1]] = x.contiguous().view(torch.uint8)
    return store.view(x.dtype)[:, :x.shape[1]]


def _fp8_out(out, rows, cols, device, block_rows):
    if out is None:
        return Fp8Rows.empty(rows, cols, device, block_rows)
    if not isinstance(out, Fp8Rows) or out.rows != rows or out.cols != cols or out.block_rows != block_rows or not out._c.scale_e8m0:
        _refuse("row_ops: out has to be Fp8Rows.empty(%d, %d, device, block_rows=%d)", rows, cols, block_rows)
    if out.device != device:
        _refuse("row_ops: out is on %s, the input on %s", out.device, device)
    return out


_norm_workspace = functools.lru_cache(1024)(lib.lssvc_group_norm_workspace_bytes)       # (a foreign call takes 1 us)


def _group_norm(x, groups, weight, bias, eps, act, slope, images, out, fp8):
    dev = x.device if isinstance(x, (T, torch.Tensor)) else None
    xr = _rows(x, "x")
    if groups.__class__ is not int:
        groups = _whole(groups, "groups")
    if images is not None and images.__class__ is not int:
        images = _whole(images, "images")
    if eps.__class__ is not float or slope.__class__ is not float:
        eps, slope = _number(eps, "eps"), _number(slope, "slope")
    if _elsewhere(dev, x, weight, bias, out):
        with torch.cuda.device(dev):
            return _group_norm(x, groups, weight, bias, eps, act, slope, images, out, fp8)
    if images is None:
        images = 1 if isinstance(x, T) or x.dim() == 2 else x.shape[0]
    elif not isinstance(x, T) and x.dim() == 4 and images != x.shape[0]:
        _refuse("group_norm: images=%d, but x has %d", images, x.shape[0])
    rows, cols = xr.rows, xr.cols
    if rows == 0:
        images = 1
    if not 0 < groups <= cols or not 0 < images <= max(rows, 1):
        _refuse("group_norm: %d rows x %d channels are not %r images, %r groups", rows, cols, images, groups)
    code = _act_code(act)
    wp = None if weight is None else _vector(weight, "weight", cols, dev)
    bp = None if bias is None else _vector(bias, "bias", cols, dev)
    if fp8:
        out = _fp8_out(out, rows, cols, dev, 1)
        yr, y8 = None, out._c
    else:
        y8 = None
        if out is None and not isinstance(x, T) and x.dim() == 2:
            out = torch.empty_like(x) if xr.ld == cols else x.new_empty((rows, cols))
            yr = Rows(out.data_ptr(), rows, cols, cols, xr.dtype)
        else:
            if out is None:
                out = T.empty(x.H, x.W, cols, dev) if isinstance(x, T) else torch.empty_like(x)
            yr = _rows(out, "out")
            if out.device != dev:
                _refuse("row_ops: out is on %s, the input on %s", out.device, dev)
    need = _norm_workspace(rows, images, cols, groups, xr.dtype, fp8)
    ws = torch.empty(need, dtype=torch.uint8, device=dev) if need else None
    check(lib.lssvc_group_norm(xr, images, groups, wp, bp, eps, code, slope, yr, y8, ws.data_ptr() if need else None, need, _raw_stream(dev.index)))
    return out


def group_norm(x, groups, weight=None, bias=None, *, eps=1e-5, act=None, slope=0.01, images=None, out=None):
    """act(group_norm(x)): statistics over the rows of each of `images` images and the C / groups channels of a group, sums in 64 bits (values
    up to 1e38, of any offset); weight / bias: C fp32 values. images: for 2-d rows and T (default 1); a 4-d tensor brings its own. out: rows of
    x's shape and type, x itself allowed. act: None, 'lrelu' (slope), 'relu', 'silu'."""
    return _group_norm(x, groups, weight, bias, eps, act, slope, images, out, False)


def group_norm_fp8(x, groups, weight=None, bias=None, *, eps=1e-5, act=None, slope=0.01, images=None, out=None):
    """quantize_fp8(act(group_norm(x))) in the pass that normalises: the fp32 result goes into 1 x 128 blocks and is not written itself."""
    return _group_norm(x, groups, weight, bias, eps, act, slope, images, out, True)


def quantize_fp8(x, block_rows=1, out=None):
    """x as 8-bit blocks: block_rows=1 (1 x 128) for activations, 128 (128 x 128) for weights. Of each block the scale is the smallest
    power of two s >= 2^-126 with max |x| <= 448 s (1 for a block of zeros), values are e4m3(x / s) to nearest even. A value that is not
    finite becomes NaN and does not move the scale."""
    xr = _rows(x, "x")
    dev = x.device
    if _elsewhere(dev, x, out):
        with torch.cuda.device(dev):
            return quantize_fp8(x, block_rows, out)
    out = _fp8_out(out, xr.rows, xr.cols, dev, block_rows)
    check(lib.lssvc_quantize_fp8(xr, out._c, _raw_stream(dev.index)))
    return out


def matmul_fp8(a, w, bias=None, *, act=None, slope=0.01, residual=None, out=None, dtype=None):
    """act(a @ w.T + bias) + residual. a: Fp8Rows (M, K) of 1 x 128 blocks; w: Fp8Rows (N, K) of 128 x 128 blocks; both with e8m0 or both
    with fp32 scales. Sums in fp32, one rounding to the output's type. bias: N fp32 values. residual, out: M rows of N channels
    (residual may be out). dtype: the output's type; by default that of out or residual, or bf16.

    What is summed: fp32 results, the products themselves. 16-bit results, what the 8-bit matrix instruction makes of them: of each 8 columns
    (8 i ... 8 i + 7) it cuts every product, toward zero, at 2^-13 of the power of two of the largest one. That is 1.5e-5 of the result in the
    2-norm for normally distributed operands, 2.4e-5 where channels differ in spread, 7e-5 where one of each 8 is 64 times the others; at
    worst 7 * 2^-13 of the largest product of every 8, which shows where those cancel. dtype=torch.float32 has none of it, at half the rate.

    Scales: a block's two are multiplied with each other in fp32 where they are fp32, and for fp32 results; outside fp32's range that product is
    inf or 0, though block times scales may not be."""
    if not isinstance(a, Fp8Rows) or not isinstance(w, Fp8Rows):
        _refuse("matmul_fp8: operands are Fp8Rows (quantize_fp8, group_norm_fp8)")
    dev = a.device
    if _elsewhere(dev, a, w, bias, residual, out):
        with torch.cuda.device(dev):
            return matmul_fp8(a, w, bias, act=act, slope=slope, residual=residual, out=out, dtype=dtype)
    m, n = a.rows, w.rows
    code = _act_code(act)
    if slope.__class__ is not float:
        slope = _number(slope, "slope")
    bp = None if bias is None else _vector(bias, "bias", n, dev)
    rr = None if residual is None else _rows(residual, "residual")
    if out is None:
        if dtype is None:
            dtype = torch.bfloat16 if rr is None else torch.float32 if isinstance(residual, T) else residual.dtype
        dt = _DTYPE.get(dtype) if isinstance(dtype, torch.dtype) else None
        if dt is None:
            _refuse("matmul_fp8: type %s (fp32, fp16 or bf16 expected)", dtype)
        if rr is None or (not isinstance(residual, T) and residual.dim() == 2):
            out = torch.empty((m, n), dtype=dtype, device=dev)
            yr = Rows(out.data_ptr(), m, n, n, dt)
        else:
            out = T.empty(residual.H, residual.W, rr.cols, dev) if isinstance(residual, T) else torch.empty_like(residual)
            yr = _rows(out, "out")
    else:
        yr = _rows(out, "out")
    if dtype is not None and not (isinstance(dtype, torch.dtype) and _DTYPE.get(dtype) == yr.dtype):
        _refuse("matmul_fp8: dtype %s is not the output's", dtype)
    if w.device != dev or residual is not None and residual.device != dev or out.device != dev:
        _refuse("matmul_fp8: operands on several devices")
    check(lib.lssvc_matmul_fp8(a._c, w._c, bp, code, slope, rr, yr, _raw_stream(dev.index)))
    return out
