"""The row operators on the GPU against their definitions in 64 bits (tests/row_ops_ref.py), at the sizes, pitches, types and values
where they can go wrong. Tolerances are the error bounds derived there."""
import pytest
import torch

from row_ops_ref import HALF_STEP, act64, dequantize64, group_norm64, matmul64, quantize64

pytestmark = pytest.mark.gpu
F32, F16, BF16 = torch.float32, torch.float16, torch.bfloat16
DEV = "cuda:0"


@pytest.fixture(scope="module")
def ops():
    from lssvc_amd import row_ops
    return row_ops


def gen(seed):
    return torch.Generator().manual_seed(seed)


def features(g, rows, c, offset=0.5, dtype=F32):
    x = torch.randn(rows, c, generator=g) * torch.exp(0.5 * torch.randn(1, c, generator=g)) + offset * torch.randn(1, c, generator=g)
    return x.to(dtype)


def wide_rows(x, pad, fill=float("nan")):
    """x on the GPU as a slice of a buffer that is `pad` channels wider; the rest holds `fill`."""
    if pad == 0:
        return x.to(DEV)
    buf = torch.full((x.shape[0], x.shape[1] + pad), fill, dtype=x.dtype, device=DEV)
    buf[:, pad // 2:pad // 2 + x.shape[1]] = x.to(DEV)
    return buf[:, pad // 2:pad // 2 + x.shape[1]]


def within(got, want, tol, what=""):
    got = got.detach().cpu().double()
    assert torch.equal(torch.isnan(got), torch.isnan(want)), what + ": NaN in other places"
    bad = ((got - want).abs() > tol) & ~torch.isnan(want)
    assert not bad.any(), "%s: %d of %d values off, worst %.3g of the bound" % (
        what, int(bad.sum()), bad.numel(), float(((got - want).abs() / tol)[~torch.isnan(want)].max()))


# ---- group norm ---------------------------------------------------------------------------------------------------------------
NORM_CASES = [
    # images, rows of an image, C, groups: one row, one channel, channels below / beside multiples of 8, resident and split forms,
    # groups wider than a slice, as many groups as channels
    (1, 1, 1, 1), (1, 1, 8, 2), (2, 3, 3, 1), (1, 5, 7, 7), (3, 4, 9, 3), (1, 64, 16, 4), (2, 100, 20, 5), (1, 540, 64, 8), (5, 17, 48, 8),
    (1, 1000, 33, 11), (1, 2160, 12, 12), (2, 2160, 96, 3), (1, 333, 1000, 8), (1, 9, 5000, 2), (1, 3, 8200, 2), (1, 700, 4104, 1),
    (1, 20000, 24, 3), (1, 5000, 1027, 1027), (1, 4000, 2060, 1), (1, 6000, 2049, 3), (1, 3000, 1030, 103), (2, 5000, 100, 5), (1, 9000, 130, 1), (1, 40000, 8, 8), (1, 70000, 3, 1), (130, 40, 64, 4), (3000, 1, 40, 4), (700, 2, 6, 2),
]


@pytest.mark.parametrize("dtype", [F32, F16, BF16], ids=["f32", "f16", "bf16"])
@pytest.mark.parametrize("images,rows,c,groups", NORM_CASES)
def test_group_norm(ops, images, rows, c, groups, dtype):
    g = gen(rows * 31 + c)
    act = [None, "relu", "lrelu", "silu"][(rows + c) % 4]
    x = features(g, images * rows, c, dtype=dtype)
    w, b = (1 + 0.2 * torch.randn(c, generator=g), 0.3 * torch.randn(c, generator=g)) if (rows + groups) % 3 else (None, None)
    want, tol = group_norm64(x, images, groups, w, b, 1e-5, act)
    tol = tol + HALF_STEP[dtype] * (want.abs() + tol) + (2.0 ** -25 if dtype == F16 else 2.0 ** -140)
    dw, db = (None, None) if w is None else (w.to(DEV), b.to(DEV))
    for pad in (0, 5, 16):
        xd = wide_rows(x, pad)
        y = ops.group_norm(xd, groups, dw, db, act=act, images=images)
        assert y.shape == x.shape and y.dtype == dtype
        within(y, want, tol, "pad %d" % pad)
        out = wide_rows(torch.zeros_like(x), pad, fill=7.0)
        whole = out._base if out._base is not None else out
        assert ops.group_norm(xd, groups, dw, db, act=act, images=images, out=out) is out
        assert torch.equal(out, y)
        if pad:
            assert (whole[:, :pad // 2] == 7).all() and (whole[:, pad // 2 + c:] == 7).all()      # what lies beside the slice stays
        assert ops.group_norm(xd, groups, dw, db, act=act, images=images, out=xd) is xd            # in place
        assert torch.equal(xd, y)


@pytest.mark.parametrize("dtype", [F32, F16, BF16], ids=["f32", "f16", "bf16"])
@pytest.mark.parametrize("images,rows,c,groups", NORM_CASES)
def test_group_norm_fp8(ops, images, rows, c, groups, dtype):
    g = gen(rows * 37 + c)
    act = [None, "relu", "lrelu", "silu"][(rows + 3 * c) % 4]
    x = features(g, images * rows, c, dtype=dtype)
    w, b = 1 + 0.2 * torch.randn(c, generator=g), 0.3 * torch.randn(c, generator=g)
    want, tol = group_norm64(x, images, groups, w, b, 1e-5, act)
    for pad in (0, 5):
        q = ops.group_norm_fp8(wide_rows(x, pad), groups, w.to(DEV), b.to(DEV), act=act, images=images)
        check_fp8(q, want, tol)


def check_fp8(q, want, tol):
    """8-bit rows of a result that is itself known within `tol`: every scale is the smallest one for some value of the block's maximum
    within its tolerance, every value within half a step (2^-4 of it, or 2^-10 scales below the smallest normal) and the tolerance."""
    rows, cols = want.shape
    assert q.rows == rows and q.cols == cols and q.values.shape == want.shape
    cb = -(-cols // 128)
    s = torch.exp2(q.scale.contiguous().view(torch.uint8).cpu().double() - 127)
    assert s.shape == (rows, cb)
    pad = lambda t: torch.nn.functional.pad(t, (0, cb * 128 - cols)).view(rows, cb, 128).amax(2)
    hi, lo = pad(want.abs() + tol), pad((want.abs() - tol).clamp(min=0))
    zero = hi == 0
    assert (s[zero] == 1).all()
    assert (lo <= 448 * s).all()
    assert ((hi > 224 * s) | (s == 2.0 ** -126) | (lo == 0)).all()
    got = dequantize64(q.values, q.scale, 1)
    each = s[:, torch.arange(cols) // 128]
    bound = tol * (1 + 2.0 ** -3) + torch.maximum(2.0 ** -4 * want.abs(), 2.0 ** -10 * each)
    assert ((got - want).abs() <= bound).all(), float(((got - want).abs() / bound).max())
    assert not behind(q).any()


def behind(q):
    """The bytes of each row from the last column to the next multiple of 16."""
    ld = q.values.stride(0)
    assert ld % 16 == 0 and q.values.data_ptr() % 16 == 0
    return q.values.as_strided((q.rows, -(-q.cols // 16) * 16), (ld, 1)).view(torch.uint8)[:, q.cols:]


@pytest.mark.parametrize("offset", [100.0, 3000.0])
@pytest.mark.parametrize("rows", [500, 30000])
def test_group_norm_keeps_the_digits_of_a_small_spread(ops, offset, rows):
    """A map whose offset is far larger than its spread: E[x^2] - E[x]^2 in fp32 would lose everything."""
    g = gen(3)
    x = torch.randn(rows, 32, generator=g) + offset
    x[0] = 50 * offset                                # the first row (the pivot) is an outlier, too
    want, tol = group_norm64(x, 1, 4, None, None, 1e-5, None)
    within(ops.group_norm(x.to(DEV), 4), want, tol + 2.0 ** -24 * want.abs())


@pytest.mark.parametrize("rows", [40, 30000])
def test_group_norm_not_finite_values_stay_in_their_group(ops, rows):
    x = torch.randn(2 * rows, 32, generator=gen(5))
    x[3, 9], x[rows + 7, 30] = float("nan"), float("inf")
    want, tol = group_norm64(x.nan_to_num(0.0, 0.0, 0.0), 2, 4, None, None, 1e-5, "silu")
    want = want.view(2, rows, 4, 8)
    want[0, :, 1], want[1, :, 3] = float("nan"), float("nan")
    y = ops.group_norm(x.to(DEV), 4, act="silu", images=2)
    within(y, want.view(2 * rows, 32), tol + 1e-6)
    q = ops.group_norm_fp8(x.to(DEV), 4, act="silu", images=2)
    assert torch.equal(torch.isnan(q.values.float()).cpu(), torch.isnan(want.view(2 * rows, 32)))
    assert not (q.scale.contiguous().view(torch.uint8) == 255).any()


def test_group_norm_constant_groups_give_the_bias(ops):
    b = torch.randn(24, generator=gen(1)).to(DEV)
    for rows in (6, 50000):
        y = ops.group_norm(torch.full((rows, 24), 3.25, device=DEV), 3, None, b)
        assert torch.equal(y, b.expand(rows, 24))


@pytest.mark.parametrize("rows,c,groups", [(50, 40, 5), (2000, 33, 11), (30000, 96, 4), (20000, 260, 130)])
def test_group_norm_with_one_of_weight_and_bias(ops, rows, c, groups):
    g = gen(c)
    x, v = features(g, rows, c), 0.5 + torch.rand(c, generator=g)
    for w, b in ((v, None), (None, v)):
        want, tol = group_norm64(x, 1, groups, w, b, 1e-5, "relu")
        dw, db = (None if t is None else t.to(DEV) for t in (w, b))
        within(ops.group_norm(x.to(DEV), groups, dw, db, act="relu"), want, tol + 2.0 ** -24 * want.abs())
        check_fp8(ops.group_norm_fp8(x.to(DEV), groups, dw, db, act="relu"), want, tol)


def test_group_norm_kinds_of_rows(ops):
    from lssvc_amd.hip_ops import T
    g = gen(8)
    x = torch.randn(3, 20, 6, 10, generator=g)
    rows = x.permute(0, 2, 3, 1).reshape(180, 20)
    want, tol = group_norm64(rows, 3, 5, None, None, 1e-5, "lrelu")
    xd = x.to(DEV).to(memory_format=torch.channels_last)
    y = ops.group_norm(xd, 5, act="lrelu")
    assert y.shape == x.shape and y.is_contiguous(memory_format=torch.channels_last)
    within(y.permute(0, 2, 3, 1).reshape(180, 20), want, tol + 2.0 ** -24 * want.abs())
    wide = torch.zeros(3, 32, 6, 10, device=DEV).to(memory_format=torch.channels_last)
    wide[:, 4:24] = xd
    assert torch.equal(ops.group_norm(wide[:, 4:24], 5, act="lrelu"), y)          # a channel slice
    t = T.from_nchw(xd[:1].contiguous(memory_format=torch.channels_last))
    z = ops.group_norm(t, 5, act="lrelu")
    assert isinstance(z, T) and torch.equal(z.to_nchw(), y[:1])
    with pytest.raises(ops.LssvcHipError):
        ops.group_norm(x.to(DEV), 5)                                             # NCHW memory
    with pytest.raises(ops.LssvcHipError):
        ops.group_norm(xd, 5, images=2)


@pytest.mark.parametrize("shape", [(2, 20, 1, 10), (2, 20, 6, 1), (3, 20, 1, 1), (1, 20, 1, 1), (2, 1, 4, 5), (0, 20, 3, 3), (2, 20, 0, 3)])
def test_maps_of_few_pixels_and_slices_of_them(ops, shape):
    """Shapes whose strides leave open which memory format they are in."""
    n, c, h, w = shape
    wide = torch.randn(n, c + 12, h, w, generator=gen(c + h)).to(DEV).to(memory_format=torch.channels_last)
    x = wide[:, 4:4 + c]
    rows = x.permute(0, 2, 3, 1).reshape(-1, c)
    y = ops.group_norm(x, 1, images=None)
    q = ops.quantize_fp8(x)
    z = ops.matmul_fp8(q, ops.quantize_fp8(torch.eye(c, device=DEV), 128), residual=x)
    assert y.shape == x.shape == z.shape and (q.rows, q.cols) == (n * h * w, c)
    if rows.shape[0]:
        want, tol = group_norm64(rows.cpu(), n, 1, None, None, 1e-5, None)
        within(y.permute(0, 2, 3, 1).reshape(-1, c), want, tol + 2.0 ** -24 * want.abs())
        assert torch.equal(q.values.contiguous().cpu().double(), quantize64(rows.cpu(), 1)[0])
        assert torch.equal(z.permute(0, 2, 3, 1).reshape(-1, c), q.dequantize() + rows)      # (one product and 0: exact but for the last sum)


# ---- quantiser ----------------------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("dtype", [F32, F16, BF16], ids=["f32", "f16", "bf16"])
@pytest.mark.parametrize("block_rows", [1, 128])
@pytest.mark.parametrize("rows,cols", [(1, 1), (1, 128), (3, 16), (2, 17), (17, 127), (5, 129), (130, 300), (129, 128), (128, 1000), (260, 40)])
def test_quantize_is_exact(ops, rows, cols, block_rows, dtype):
    g = gen(rows + 1000 * cols)
    x = (torch.randn(rows, cols, generator=g) * torch.exp(3 * torch.randn(rows, 1, generator=g))).to(dtype)
    x[rows // 2, cols // 2:] = 0
    want, e = quantize64(x, block_rows)
    for pad in (0, 3):
        q = ops.quantize_fp8(wide_rows(x, pad), block_rows)
        assert q.values.dtype == torch.float8_e4m3fn and q.scale.dtype == torch.float8_e8m0fnu and q.block_rows == block_rows
        assert torch.equal(q.scale.contiguous().view(torch.uint8).cpu().double() - 127, e)
        assert torch.equal(q.values.contiguous().cpu().double(), want)
        assert not behind(q).any()
        assert torch.equal(q.dequantize().cpu().double(), dequantize64(q.values, q.scale, block_rows))


@pytest.mark.parametrize("block_rows", [1, 128])
def test_quantize_every_rounding(ops, block_rows):
    """All finite bf16 values of a binade range around e4m3's, each in a block whose maximum is 448: every tie, every subnormal."""
    bits = torch.arange(0, 65536, dtype=torch.int32)
    v = (bits << 16).view(F32)
    v = v[torch.isfinite(v) & (v.abs() <= 448) & (v.abs() >= 2.0 ** -14)]
    n = -(-v.numel() // 127)
    x = torch.zeros(n, 128)
    x[:, 1:] = torch.nn.functional.pad(v, (0, n * 127 - v.numel())).view(n, 127)
    x[:, 0] = 448
    want, e = quantize64(x, block_rows)
    assert (e == 0).all()
    q = ops.quantize_fp8(x.to(DEV), block_rows)
    assert torch.equal(q.values.cpu().double(), want)
    assert torch.equal(torch.signbit(q.values.float().cpu()), torch.signbit(x))


def test_quantize_special_values(ops):
    x = torch.zeros(8, 256)
    x[0, :4] = torch.tensor([float("inf"), -float("inf"), float("nan"), 1.0])       # the scale is the finite maximum's
    x[1, 0] = float("nan")                                                          # nothing finite but zeros
    x[2, 0] = 3.4028234663852886e38                                                 # the largest fp32 value
    x[3, 0], x[3, 1] = 1e-45, -1.1754943508222875e-38                               # subnormals: the smallest scale
    x[4, 0] = 448.0
    x[5, 0] = 448.0000305175781                                                     # one step more: the next scale
    x[6, :] = -0.0
    want, e = quantize64(x, 1)
    q = ops.quantize_fp8(x.to(DEV))
    assert torch.equal(q.scale.contiguous().view(torch.uint8).cpu().double() - 127, e)
    got = q.values.cpu().double()
    assert torch.equal(torch.isnan(got), torch.isnan(want))
    assert torch.equal(got.nan_to_num(0.0), want.nan_to_num(0.0))
    assert e[4, 0] == 0 and e[5, 0] == 1 and e[3, 0] == -126 and e[1, 0] == 0


# ---- product ------------------------------------------------------------------------------------------------------------------
def operands(ops, g, m, n, k, kind):
    a = ops.quantize_fp8(features(g, m, k).to(DEV))
    w = ops.quantize_fp8((torch.randn(n, k, generator=g) / k ** 0.5).to(DEV), 128)
    if kind == "any":
        rescale = lambda q, br: ops.Fp8Rows(q.values, (torch.exp2(q.scale.contiguous().view(torch.uint8).float() - 127)
                                                       * (0.6 + 0.8 * torch.rand(tuple(q.scale.shape), generator=g).to(DEV))), br)
        a, w = rescale(a, 1), rescale(w, 128)
    return a, w, dequantize64(a.values, a.scale, 1), dequantize64(w.values, w.scale, 128)


MATMUL_CASES = [
    (1, 1, 1), (1, 16, 16), (2, 5, 17), (1, 100, 128), (3, 129, 129), (15, 64, 300), (16, 200, 1000), (17, 77, 515), (31, 300, 2000), (32, 16, 4100),
    (33, 1, 64), (33, 70, 127), (64, 64, 128), (65, 257, 640), (100, 1000, 96), (128, 130, 1030), (200, 200, 200), (257, 511, 384), (400, 1000, 130),
    (1500, 1300, 150), (2100, 2200, 90), (5000, 300, 257), (3300, 4000, 260),
    (2, 5, 100003), (70, 130, 50000), (1, 200001, 20), (20001, 1, 130),                                               # long, wide, tall
    # each tiling in its own range (the choice is by estimated time), the last block of K whole and cut, 1 - 4 blocks behind a multiple of 4;
    # the results' type follows from the sum of the sizes
    (96, 2644, 3401), (139, 1781, 3991), (146, 1487, 3934), (49, 4027, 4173), (400, 400, 1024),                       # 16 x 64
    (352, 2870, 3597), (399, 2394, 3862), (341, 2756, 4189), (2330, 430, 4149),                                       # 32 x 64
    (3850, 253, 4129), (3896, 220, 4174), (4139, 173, 4162), (3970, 205, 406),                                         # 64 x 64
    (3942, 4108, 269), (997, 4056, 1149), (3551, 1142, 1102), (4423, 820, 1152),                                      # 128 x 128
    (3111, 3974, 1037), (4885, 2486, 1043), (3230, 3886, 1028), (4662, 2565, 946),                                    # 256 x 256
    (3223, 3835, 1019), (3255, 3819, 920), (2841, 4265, 731), (4416, 2712, 464),                                      # 192 x 256
]


@pytest.mark.parametrize("kind", ["pow2", "any"])
@pytest.mark.parametrize("m,n,k", MATMUL_CASES)
def test_matmul_fp8(ops, m, n, k, kind):
    g = gen(m + 7 * n + 11 * k)
    a, w, a64, w64 = operands(ops, g, m, n, k, kind)
    pick = m + n + k
    dtype = [F32, F16, BF16][pick % 3]
    act = [None, "relu", "lrelu", "silu"][pick % 4]
    bias = 0.3 * torch.randn(n, generator=g) if pick % 5 else None
    res = torch.randn(m, n, generator=g).to(dtype) if pick % 2 else None
    want, tol = matmul64(a64, w64, bias, act, res, dtype)
    bd = None if bias is None else bias.to(DEV)
    rd = None if res is None else wide_rows(res, 3)
    y = ops.matmul_fp8(a, w, bd, act=act, residual=rd, dtype=dtype)
    assert y.shape == (m, n) and y.dtype == dtype
    within(y, want, tol)
    out = wide_rows(torch.zeros(m, n, dtype=dtype), 5, fill=7.0)
    ops.matmul_fp8(a, w, bd, act=act, residual=rd, out=out)
    assert torch.equal(out, y)
    whole = out._base
    assert (whole[:, :2] == 7).all() and (whole[:, 2 + n:] == 7).all()
    if res is not None:
        assert ops.matmul_fp8(a, w, bd, act=act, residual=rd, out=rd) is rd          # onto the residual
        assert torch.equal(rd, y)


@pytest.mark.parametrize("dtype", [F32, F16, BF16], ids=["f32", "f16", "bf16"])
@pytest.mark.parametrize("act", [None, "relu", "lrelu", "silu"])
@pytest.mark.parametrize("m", [7, 150])
def test_matmul_fp8_epilogues(ops, m, act, dtype):
    g = gen(m)
    a, w, a64, w64 = operands(ops, g, m, 90, 200, "pow2")
    bias, res = torch.randn(90, generator=g), torch.randn(m, 90, generator=g).to(dtype)
    want, tol = matmul64(a64, w64, bias, act, res, dtype, slope=0.2)
    within(ops.matmul_fp8(a, w, bias.to(DEV), act=act, slope=0.2, residual=res.to(DEV)), want, tol)


@pytest.mark.parametrize("dtype", [F32, BF16], ids=["f32", "bf16"])
@pytest.mark.parametrize("m,n", [(40, 70), (700, 600), (3000, 3000)])
def test_matmul_fp8_operands_at_any_pitch(ops, m, n, dtype):
    """Slices of wider tensors, read in place: pitches that are no multiple of a line, values behind the last column that are not zero."""
    g = gen(m + n)
    for k in (144, 560):
        wide = lambda rows: (8 * torch.randn(rows, k + 48, generator=g)).to(torch.float8_e4m3fn).to(DEV)[:, 16:16 + k]
        scales = lambda rows: (0.5 + torch.rand(rows, -(-k // 128) + 3, generator=g)).to(DEV)[:, 1:1 + -(-k // 128)]
        av, wv, sa, sw = wide(m), wide(n), scales(m), scales(-(-n // 128))
        a, w = ops.Fp8Rows(av, sa), ops.Fp8Rows(wv, sw, 128)
        assert a.values.data_ptr() == av.data_ptr() and w.scale.data_ptr() == sw.data_ptr()
        want, tol = matmul64(dequantize64(av, sa, 1), dequantize64(wv, sw, 128), None, "relu", None, dtype)
        within(ops.matmul_fp8(a, w, act="relu", dtype=dtype), want, tol)


@pytest.mark.parametrize("dtype", [F32, BF16], ids=["f32", "bf16"])
@pytest.mark.parametrize("m", [20, 1000])
def test_matmul_fp8_ends_of_the_scales(ops, m, dtype):
    """The smallest and the largest power of two, whose product is an ordinary one, and the byte that stands for NaN."""
    g = gen(m)
    a, w = ops.quantize_fp8(torch.randn(m, 256, generator=g).to(DEV)), ops.quantize_fp8(torch.randn(300, 256, generator=g).to(DEV), 128)
    sa, sw = torch.full((m, 2), 127, dtype=torch.uint8, device=DEV), torch.full((3, 2), 127, dtype=torch.uint8, device=DEV)
    sa[:, 0], sw[:, 0] = 0, 254
    sa[:, 1], sw[:, 1] = 254, 0
    a, w = ops.Fp8Rows(a.values, sa.view(torch.float8_e8m0fnu)), ops.Fp8Rows(w.values, sw.view(torch.float8_e8m0fnu), 128)
    want, tol = matmul64(a.values.cpu().double(), w.values.cpu().double(), None, None, None, dtype)
    within(ops.matmul_fp8(a, w, dtype=dtype), want, tol)
    sa[:], sw[:] = 127, 127
    sa[5, 1], sw[1, 0] = 255, 255
    a, w = ops.Fp8Rows(a.values, sa.view(torch.float8_e8m0fnu)), ops.Fp8Rows(w.values, sw.view(torch.float8_e8m0fnu), 128)
    want[5], want[:, 128:256] = float("nan"), float("nan")
    within(ops.matmul_fp8(a, w, dtype=dtype), want, tol)


def test_matmul_fp8_blocks_of_very_different_scales(ops):
    """Every block of K has its own power of two, 2^-60 ... 2^60: a wrong scale byte is visible at once."""
    g = gen(2)
    for m in (5, 300):
        x, wt = torch.randn(m, 1500, generator=g), torch.randn(200, 1500, generator=g)
        e = torch.randint(-60, 61, (12,), generator=g)[torch.arange(1500) // 128]
        x, wt = x * torch.exp2(e.float()), wt * torch.exp2(-e.float())
        a, w = ops.quantize_fp8(x.to(DEV)), ops.quantize_fp8(wt.to(DEV), 128)
        a64, w64 = dequantize64(a.values, a.scale, 1), dequantize64(w.values, w.scale, 128)
        want, tol = matmul64(a64, w64, None, None, None, F32)
        within(ops.matmul_fp8(a, w, dtype=F32), want, tol)


def test_matmul_fp8_nan_stays_in_its_row(ops):
    for m in (20, 200):
        x = torch.randn(m, 260, generator=gen(4))
        x[3, 259] = float("nan")
        a, w = ops.quantize_fp8(x.to(DEV)), ops.quantize_fp8(torch.randn(100, 260, generator=gen(5)).to(DEV), 128)
        y = ops.matmul_fp8(a, w, dtype=F32).cpu()
        assert torch.isnan(y[3]).all() and torch.isfinite(y[torch.arange(m) != 3]).all()


# ---- together -----------------------------------------------------------------------------------------------------------------
def test_norm_product_chain(ops):
    """A pointwise block as it is used: norm + silu -> 8 bits -> widening product + lrelu -> 8 bits -> product + skip, on a channels-last map."""
    g = gen(6)
    n, c, h, w = 2, 96, 18, 30
    x = torch.randn(n, c, h, w, generator=g)
    gamma, beta = 1 + 0.1 * torch.randn(c, generator=g), 0.1 * torch.randn(c, generator=g)
    w1, b1 = torch.randn(4 * c, c, generator=g) / c ** 0.5, 0.1 * torch.randn(4 * c, generator=g)
    w2, b2 = torch.randn(c, 4 * c, generator=g) / (4 * c) ** 0.5, 0.1 * torch.randn(c, generator=g)
    xd = x.to(DEV).to(memory_format=torch.channels_last)
    q1, q2 = ops.quantize_fp8(w1.to(DEV), 128), ops.quantize_fp8(w2.to(DEV), 128)
    q = ops.group_norm_fp8(xd, 8, gamma.to(DEV), beta.to(DEV), act="silu")
    hidden = ops.matmul_fp8(q, q1, b1.to(DEV), act="lrelu", slope=0.1)
    qh = ops.quantize_fp8(hidden)
    y = ops.matmul_fp8(qh, q2, b2.to(DEV), residual=xd)
    assert y.shape == x.shape and y.dtype == F32 and y.is_contiguous(memory_format=torch.channels_last)
    rows = x.permute(0, 2, 3, 1).reshape(-1, c)
    norm, tol = group_norm64(rows, n, 8, gamma, beta, 1e-5, "silu")
    check_fp8(q, norm, tol)
    want, tol = matmul64(dequantize64(q.values, q.scale, 1), dequantize64(q1.values, q1.scale, 128), b1, "lrelu", None, BF16, slope=0.1)
    within(hidden, want, tol)
    v, e = quantize64(hidden.cpu(), 1)
    assert torch.equal(qh.values.contiguous().cpu().double(), v)
    want, tol = matmul64(dequantize64(qh.values, qh.scale, 1), dequantize64(q2.values, q2.scale, 128), b2, None, rows, F32)
    within(y.permute(0, 2, 3, 1).reshape(-1, c), want, tol)
    # against the block in full precision: 8-bit operands are off by at most 2^-4 each, 2^-4 / sqrt(3) on average, independent of each other
    f1 = act64(norm @ w1.double().t() + b1, "lrelu", 0.1)
    full = f1 @ w2.double().t() + b2 + rows.double()
    err = (y.permute(0, 2, 3, 1).reshape(-1, c).cpu().double() - full).norm() / (full - rows.double()).norm()
    assert err < 2.0 ** -4


def test_views_of_the_engine(ops):
    """hip_ops.T in and out: a slice of a wider buffer as the product's residual and target."""
    from lssvc_amd.hip_ops import T
    g = gen(15)
    x, wide = torch.randn(1, 24, 9, 14, generator=g), torch.randn(1, 40, 9, 14, generator=g)
    t, s = T.from_nchw(x.to(DEV).contiguous(memory_format=torch.channels_last)), T.from_nchw(wide.to(DEV).contiguous(memory_format=torch.channels_last))
    part = s.slice(8, 32)
    q, w = ops.quantize_fp8(t), ops.quantize_fp8(torch.randn(24, 24, generator=g).to(DEV), 128)
    rows, res = x.permute(0, 2, 3, 1).reshape(-1, 24), wide.permute(0, 2, 3, 1).reshape(-1, 40)
    assert torch.equal(q.values.contiguous().cpu().double(), quantize64(rows, 1)[0])
    want, tol = matmul64(dequantize64(q.values, q.scale, 1), dequantize64(w.values, w.scale, 128), None, "relu", res[:, 8:32].contiguous(), F32)
    y = ops.matmul_fp8(q, w, act="relu", residual=part)
    assert isinstance(y, T) and (y.H, y.W, y.C) == (9, 14, 24)
    within(y.to_nchw()[0].permute(1, 2, 0).reshape(-1, 24), want, tol)
    ops.matmul_fp8(q, w, act="relu", residual=part, out=part)
    after = s.to_nchw()[0].permute(1, 2, 0).reshape(-1, 40)
    within(after[:, 8:32], want, tol)
    assert torch.equal(after[:, :8].cpu(), res[:, :8]) and torch.equal(after[:, 32:].cpu(), res[:, 32:])


# ---- calls --------------------------------------------------------------------------------------------------------------------
def block(ops, s):
    q = ops.group_norm_fp8(s["x"], 4, s["g"], s["b"], act="silu")
    return ops.matmul_fp8(q, s["w"], s["bias"], act="lrelu", residual=s["x"]), ops.group_norm(s["x"], 4, s["g"], s["b"])


def block_state(ops, rows, seed):
    g = gen(seed)
    return {"x": torch.randn(rows, 64, generator=g).to(DEV), "g": torch.randn(64, generator=g).to(DEV), "b": torch.randn(64, generator=g).to(DEV),
            "w": ops.quantize_fp8(torch.randn(64, 64, generator=g).to(DEV), 128), "bias": torch.randn(64, generator=g).to(DEV)}


@pytest.mark.parametrize("rows", [20, 4000, 60000])
def test_captured_calls_replay(ops, rows):
    """Two graphs of the same calls on states of their own, replayed in turn with eager work between: every replay is the eager result."""
    states = [block_state(ops, rows, 1), block_state(ops, rows, 2)]
    eager = [block(ops, s) for s in states]
    torch.cuda.synchronize()
    graphs = []
    for s in states:
        gr = torch.cuda.CUDAGraph()
        with torch.cuda.graph(gr):
            out = block(ops, s)
        graphs.append((gr, out))
    for _ in range(3):
        for (gr, out), want in zip(graphs, eager):
            for o in out:
                o.zero_()
            gr.replay()
            again = block(ops, states[0])
            torch.cuda.synchronize()
            assert all(torch.equal(o, w) for o, w in zip(out, want))
            assert all(torch.equal(o, w) for o, w in zip(again, eager[0]))
    s0 = states[0]["x"].clone()
    states[0]["x"].copy_(states[1]["x"])                        # new inputs in the captured buffers
    want = block(ops, states[0])
    graphs[0][0].replay()
    torch.cuda.synchronize()
    assert all(torch.equal(o, w) for o, w in zip(graphs[0][1], want))
    states[0]["x"].copy_(s0)


def test_calls_on_two_streams_at_once(ops):
    states = [block_state(ops, 30000, k) for k in range(2)]
    want = [block(ops, s) for s in states]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in states]
    got = [[], []]
    for _ in range(4):
        for k, st in enumerate(streams):
            with torch.cuda.stream(st):
                got[k].append(block(ops, states[k]))
    torch.cuda.synchronize()
    for k in range(2):
        for r in got[k]:
            assert all(torch.equal(o, w) for o, w in zip(r, want[k]))


def test_calls_from_two_threads(ops):
    """Every thread on a stream of its own, maps whose slices take different amounts of LDS."""
    import threading
    states = [[torch.randn(rows, 64, generator=gen(rows)).to(DEV) for rows in sizes] for sizes in ((300, 2400), (1200, 1900))]
    want = [[ops.group_norm(x, 8, act="silu") for x in s] for s in states]
    torch.cuda.synchronize()
    wrong = []

    def work(k):
        with torch.cuda.stream(torch.cuda.Stream()):
            for _ in range(50):
                got = [ops.group_norm(x, 8, act="silu") for x in states[k]]
            torch.cuda.current_stream().synchronize()
            wrong.extend(k for a, b in zip(got, want[k]) if not torch.equal(a, b))
    threads = [threading.Thread(target=work, args=(k,)) for k in range(2)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert wrong == []


def test_the_same_call_twice_gives_the_same_bits(ops):
    s = block_state(ops, 50000, 9)
    first = block(ops, s)
    for _ in range(3):
        assert all(torch.equal(a, b) for a, b in zip(block(ops, s), first))


def test_offsets_beyond_32_bits(ops):
    """More than 2^31 values in and out: the rows at the end are what they are in a call of their own."""
    g, images, rows, c = gen(7), 270, 65536, 128
    last = features(g, rows, c, dtype=BF16)
    x = torch.empty(images * rows, c, dtype=BF16, device=DEV)
    x.view(images, rows, c)[:] = last.to(DEV)
    x[:-rows].mul_(-2)
    y = ops.group_norm(x, 8, act="silu", images=images)
    want, tol = group_norm64(last, 1, 8, None, None, 1e-5, "silu")
    within(y[-rows:], want, tol + HALF_STEP[BF16] * (want.abs() + tol) + 2.0 ** -140)
    del y
    q = ops.group_norm_fp8(x, 8, act="silu", images=images)
    own = ops.Fp8Rows(q.values[-rows:], q.scale[-rows:])
    check_fp8(own, want, tol)
    del q, own
    a, tail = ops.quantize_fp8(x), ops.quantize_fp8(x[-500:])
    assert torch.equal(a.values[-500:].float(), tail.values.float()) and torch.equal(a.scale[-500:].float(), tail.scale.float())
    w = ops.quantize_fp8(torch.randn(130, c, generator=g).to(DEV), 128)
    y = ops.matmul_fp8(a, w)
    want, tol = matmul64(dequantize64(tail.values, tail.scale, 1), dequantize64(w.values, w.scale, 128), None, None, None, BF16)
    within(y[-500:], want, tol)
    del y, a
    v = x.view(128, -1)                                                   # one block of rows, its columns 2^24 values wide
    w = ops.quantize_fp8(v, 128)
    want, e = quantize64(v[:, -256:].cpu(), 128)
    assert torch.equal(w.values[:, -256:].contiguous().cpu().double(), want)
    assert torch.equal(w.scale[:, -2:].contiguous().view(torch.uint8).cpu().double() - 127, e)


def test_no_rows(ops):
    x = torch.empty(0, 48, device=DEV)
    assert ops.group_norm(x, 3).shape == (0, 48)
    q = ops.group_norm_fp8(x, 3)
    assert (q.rows, q.cols) == (0, 48)
    q = ops.quantize_fp8(x)
    w = ops.quantize_fp8(torch.randn(10, 48, device=DEV), 128)
    assert ops.matmul_fp8(q, w).shape == (0, 10)
    assert ops.quantize_fp8(x, 128).scale.shape == (0, 1)


def test_operands_from_a_checkpoint(ops):
    """Values and scales that came from elsewhere: odd columns, sliced and unaligned storage are copied once, others are used in place."""
    g = gen(12)
    vals = (torch.randn(40, 90, generator=g) * 8).to(torch.float8_e4m3fn).to(DEV)
    scale = (torch.rand(40, 1, generator=g) + 0.5).to(DEV)
    a = ops.Fp8Rows(vals, scale)
    assert a.values.data_ptr() != vals.data_ptr() and torch.equal(a.values.float(), vals.float())
    wv = (torch.randn(30, 96, generator=g) * 8).to(torch.float8_e4m3fn).to(DEV)
    w = ops.Fp8Rows(wv[:, :90], (torch.rand(1, 1, generator=g) + 0.5).to(DEV), 128)
    want, tol = matmul64(dequantize64(vals, scale, 1), dequantize64(wv[:, :90], w.scale, 128), None, None, None, F32)
    within(ops.matmul_fp8(a, w, dtype=F32), want, tol)
    aligned = ops.Fp8Rows(wv, torch.ones(30, 1, device=DEV))
    assert aligned.values.data_ptr() == wv.data_ptr()


def test_refusals_on_the_gpu(ops):
    E = ops.LssvcHipError
    x = torch.randn(32, 64, device=DEV)
    q, w = ops.quantize_fp8(x), ops.quantize_fp8(torch.randn(48, 64, device=DEV), 128)
    f = ops.Fp8Rows(w.values, torch.ones(1, 1, device=DEV), 128)
    for call in (
            lambda: ops.group_norm(x, 5), lambda: ops.group_norm(x, 0), lambda: ops.group_norm(x, 4, images=3), lambda: ops.group_norm(x, 4, act="gelu"),
            lambda: ops.group_norm(x, 4, torch.ones(63, device=DEV)), lambda: ops.group_norm(x, 4, torch.ones(64)), lambda: ops.group_norm(x, 4, eps=-1.0),
            lambda: ops.group_norm(x.t(), 4), lambda: ops.group_norm(x.double(), 4), lambda: ops.group_norm(x.cpu(), 4), lambda: ops.group_norm(x, 4, out=x[:16]),
            lambda: ops.group_norm(x, 4, out=x.half()), lambda: ops.group_norm(x.clone().requires_grad_(), 4), lambda: ops.group_norm(x[None], 4),
            lambda: ops.group_norm(x[:31], 4, out=x[1:]),                                 # overlaps in part
            lambda: ops.group_norm_fp8(x, 4, out=w), lambda: ops.quantize_fp8(x, 64), lambda: ops.quantize_fp8(x, out=w),
            lambda: ops.matmul_fp8(q, q), lambda: ops.matmul_fp8(w, w), lambda: ops.matmul_fp8(q, f), lambda: ops.matmul_fp8(x, w),
            lambda: ops.matmul_fp8(q, ops.quantize_fp8(torch.randn(48, 80, device=DEV), 128)), lambda: ops.matmul_fp8(q, w, torch.zeros(47, device=DEV)),
            lambda: ops.matmul_fp8(q, w, residual=torch.zeros(32, 47, device=DEV)), lambda: ops.matmul_fp8(q, w, residual=torch.zeros(32, 48, device=DEV), dtype=F16),
            lambda: ops.matmul_fp8(q, w, out=torch.zeros(31, 48, device=DEV)), lambda: ops.matmul_fp8(q, w, dtype=torch.float64),
            lambda: ops.matmul_fp8(q, w, out=torch.zeros(32, 48, device=DEV), dtype=F16),
            lambda: ops.group_norm(x, 4 + (1 << 32)), lambda: ops.group_norm(x, 4, images=1 + (1 << 32)),      # not their low 32 bits
            lambda: ops.group_norm(x, 4, torch.ones(32, 64, device=DEV)[0], out=x[:, :64].t()),
            lambda: ops.matmul_fp8(q, ops.quantize_fp8(torch.empty(0, 64, device=DEV), 128)),
            lambda: ops.Fp8Rows(q.values, q.scale, 128), lambda: ops.Fp8Rows(q.values, q.scale, 7), lambda: ops.Fp8Rows(x, q.scale),
    ):
        with pytest.raises(E):
            call()
    y = x[:31]
    out = torch.empty(31, 64, device=DEV)
    assert ops.group_norm(y, 4, out=out) is out                                           # and the next call works


def test_workspace_is_checked(ops):
    from lssvc_amd import _lib
    x = torch.randn(60000, 64, device=DEV)
    y = torch.empty_like(x)
    r, o = ops._rows(x, "x"), ops._rows(y, "y")
    need = _lib.lib.lssvc_group_norm_workspace_bytes(60000, 1, 64, 4, _lib.F32, 0)
    assert need > 0
    ws = torch.empty(need, dtype=torch.uint8, device=DEV)
    call = lambda p, n: _lib.lib.lssvc_group_norm(r, 1, 4, None, None, 1e-5, 0, 0.0, o, None, p, n, torch.cuda.current_stream().cuda_stream)
    assert call(None, 0) != 0 and b"workspace" in _lib.lib.lssvc_last_error()
    assert call(ws.data_ptr(), need - 1) != 0
    assert call(ws.data_ptr(), need) == 0
    torch.cuda.synchronize()
