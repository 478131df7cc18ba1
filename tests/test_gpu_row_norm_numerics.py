"""Group norm against 64 bits as closely as its arithmetic allows: large, small and offset values, and every form within a few half steps of
fp32, so that an error of the statistics cannot hide behind the bound of a sum in 32 bits."""
import pytest
import torch

from row_ops_ref import EPS32, HALF_STEP, act64, act_error
from test_gpu_row_ops import BF16, DEV, F16, F32, NORM_CASES, check_fp8, features, gen, ops, wide_rows, within   # noqa: F401 (ops: fixture)

pytestmark = pytest.mark.gpu


def norm_tight(x, images, groups, weight, bias, eps, act):
    """-> (y, allowed error) of statistics in 64 bits and one evaluation per value in fp32:
      d = x - hi(mean)            one half step of |d|, |d| <= |x - mean| + half a step of |mean|
      a = rstd * w                rstd rounded, the product rounded: two half steps
      b' = bias - low(mean) * a   one half step of |b'|, |b'| <= |bias| + half a step of |mean| a
      d * a + b'                  one half step of the result
    and what 64-bit sums of at most 1024 additions in a chain leave of mean and variance: 2^-43 of the mean in magnitudes, 2^-43 (1 + mean^2 / var)
    of the variance, half of that of rstd."""
    rows, c = x.shape
    v = x.double().view(images, rows // images, groups, c // groups)
    mu = v.mean(dim=(1, 3), keepdim=True)
    rstd = 1 / ((v - mu).square().mean(dim=(1, 3), keepdim=True) + eps).sqrt()
    flat = lambda t: t.expand_as(v).reshape(rows, c)
    w = torch.ones(c, dtype=torch.float64) if weight is None else weight.double()
    b = torch.zeros(c, dtype=torch.float64) if bias is None else bias.double()
    n = ((v - mu) * rstd).reshape(rows, c)
    z = n * w + b
    far = flat(mu.abs() * rstd)                                            # |mean| in units of the spread
    dz = EPS32 * (3 * (n * w).abs() + b.abs() + z.abs() + 4 * EPS32 * far * w.abs()) * (1 + 2.0 ** -20) + 2.0 ** -43 * ((1 + far) * w.abs() + (1 + far * far) * (n * w).abs())
    return act64(z, act), act_error(z, dz, act)


# one, two and more groups in a thread's channels (4 or 8), their sums entered in pairs or in turns, maps on the chip and larger ones
GROUP_CASES = [(1, 600, 64, 16), (1, 600, 60, 20), (1, 600, 56, 8), (2, 600, 72, 12), (1, 600, 64, 64), (2, 600, 62, 31), (1, 600, 63, 21), (1, 4000, 24, 24), (1, 3500, 16, 16),
               (1, 3300, 32, 16), (2, 440, 128, 128), (1, 190, 128, 64), (1, 300, 120, 24), (1, 20000, 64, 16), (1, 20000, 60, 20), (2, 20000, 56, 8), (1, 20000, 64, 64), (2, 20000, 62, 31),
               (1, 20000, 63, 21), (1, 20000, 66, 11), (1, 9000, 2100, 300)]


@pytest.mark.parametrize("images,rows,c,groups", [s for s in NORM_CASES if s[0] * s[1] * s[2] > 100] + GROUP_CASES)
def test_every_form_within_a_few_half_steps(ops, images, rows, c, groups):      # noqa: F811
    g = gen(rows * 41 + c)
    act = [None, "relu", "lrelu"][(rows + c) % 3]
    x = features(g, images * rows, c)
    w, b = (1 + 0.2 * torch.randn(c, generator=g), 0.3 * torch.randn(c, generator=g)) if (rows + groups) % 3 else (None, None)
    dw, db = (None, None) if w is None else (w.to(DEV), b.to(DEV))
    want, tol = norm_tight(x, images, groups, w, b, 1e-5, act)
    within(ops.group_norm(x.to(DEV), groups, dw, db, act=act, images=images), want, tol)
    check_fp8(ops.group_norm_fp8(wide_rows(x, 5), groups, dw, db, act=act, images=images), want, tol)


def rounded_once(got, want, tol):
    """Every value is what some number within `tol` of `want` rounds to (the ends one fp32 step further out: 64 bits go to 16 by way of 32)."""
    inf = torch.tensor(float("inf"))
    low, high = torch.nextafter((want - tol).float(), -inf).to(got.dtype), torch.nextafter((want + tol).float(), inf).to(got.dtype)
    got = got.cpu()
    bad = ~((got >= low) & (got <= high))
    assert not bad.any(), "%d of %d values" % (int(bad.sum()), bad.numel())


@pytest.mark.parametrize("dtype", [F16, BF16], ids=["f16", "bf16"])
@pytest.mark.parametrize("images,rows,c,groups", [(3, 1961, 100, 5), (2, 1000, 96, 3), (1, 34560, 64, 8), (2, 9000, 100, 5), (1, 20000, 257, 1), (2, 3000, 1030, 103)] + GROUP_CASES)
def test_16_bit_results_are_rounded_once(ops, images, rows, c, groups, dtype):  # noqa: F811
    """A bound of half a step of 16 bits hides an error of the statistics; which way a value rounds does not."""
    x = features(gen(rows + c), images * rows, c, dtype=dtype)
    want, tol = norm_tight(x, images, groups, None, None, 1e-5, None)
    rounded_once(ops.group_norm(x.to(DEV), groups, images=images), want, tol)


@pytest.mark.parametrize("spread,offset,eps", [(1e20, 0, 1e-5), (1e17, 1e20, 1e-5), (1e30, 0, 0.0), (1e37, 0, 1e-5), (1e37, -3e37, 0.0), (1e-18, 0, 0.0), (1e-25, 1e-24, 0.0), (1e-30, 0, 0.0)])
@pytest.mark.parametrize("dtype", [F32, BF16], ids=["f32", "bf16"])
@pytest.mark.parametrize("images,rows,c,groups", [(2, 300, 64, 4), (1, 60000, 64, 4), (2, 200, 100, 5), (1, 30000, 100, 5), (1, 50000, 3, 1)])
def test_values_whose_squares_leave_fp32(ops, images, rows, c, groups, dtype, spread, offset, eps):      # noqa: F811
    """Finite values have finite results whatever their size, in the form for small maps and in the one for large maps."""
    g = gen(rows + c)
    x = (spread * torch.randn(images * rows, c, generator=g, dtype=torch.float64) + offset).to(dtype)
    w, b = 1 + 0.2 * torch.randn(c, generator=g), 0.3 * torch.randn(c, generator=g)
    want, tol = norm_tight(x, images, groups, w, b, eps, "relu")
    xd, wd, bd = x.to(DEV), w.to(DEV), b.to(DEV)
    y = ops.group_norm(xd, groups, wd, bd, eps=eps, act="relu", images=images)
    within(y, want, tol + HALF_STEP[dtype] * (want.abs() + tol))
    check_fp8(ops.group_norm_fp8(xd, groups, wd, bd, eps=eps, act="relu", images=images), want, tol)


@pytest.mark.parametrize("rows", [500, 30000])
@pytest.mark.parametrize("c,groups", [(32, 4), (100, 5)])
@pytest.mark.parametrize("offset", [100.0, 3000.0, 1e5])
def test_an_offset_costs_no_digits(ops, offset, rows, c, groups):               # noqa: F811
    x = torch.randn(rows, c, generator=gen(3)) + offset
    want, tol = norm_tight(x, 1, groups, None, None, 1e-5, None)
    within(ops.group_norm(x.to(DEV), groups), want, tol)


def test_a_block_at_the_border_of_two_scales(ops):                              # noqa: F811
    """Maxima of 448 * 2^e itself, and a step to either side, exact in fp32: the scale is the definition's."""
    x = torch.zeros(6, 128)
    x[:, ::2], x[:, 1::2] = 1.0, -1.0                                           # mean 0, variance 1 in every row: y = weight * x
    w = torch.full((128,), 0.5)
    for e in (-3, 0, 5):
        for step, scale in ((-1, e), (0, e), (1, e + 1)):
            top = torch.tensor(448.0 * 2.0 ** e)
            top = top if step == 0 else torch.nextafter(top, torch.tensor(float("inf") if step > 0 else 0.0))
            w[7] = top
            q = ops.group_norm_fp8(x.to(DEV), 1, w.to(DEV), None, eps=0.0, images=6)
            assert (q.scale.contiguous().view(torch.uint8).cpu().int() - 127 == scale).all(), (e, step)
