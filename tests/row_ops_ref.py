"""The row operators from their definitions, in 64 bits on the CPU, with the error that each result may have."""
import torch

EPS32 = 2.0 ** -24                        # half a step of fp32, relative
HALF_STEP = {torch.float32: 2.0 ** -24, torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}


def act64(z, act, slope=0.01):
    if act == "relu":
        return torch.where(z < 0, torch.zeros_like(z), z)
    if act == "lrelu":
        return torch.where(z >= 0, z, slope * z)
    if act == "silu":
        return z / (1 + torch.exp(-z))
    return z


def act_error(z, dz, act):
    """What an error dz of z becomes behind the activation, the activation's own rounding included: slopes are at most 1.1 (silu),
    silu's exp and reciprocal are good to a few units and exp's argument error is |z| half steps."""
    y = act64(z, act)
    own = EPS32 * (8 + z.abs()) * y.abs() if act == "silu" else EPS32 * y.abs()
    return 1.1 * dz + own


def group_norm64(x, images, groups, weight, bias, eps, act, slope=0.01):
    """x (rows, C), weight / bias (C) or None -> (y, allowed error of an fp32 evaluation)."""
    rows, c = x.shape
    v = x.double().view(images, rows // images, groups, c // groups)
    mu = v.mean(dim=(1, 3), keepdim=True)
    rstd = 1 / ((v - mu).square().mean(dim=(1, 3), keepdim=True) + eps).sqrt()
    w = torch.ones(c, dtype=torch.float64) if weight is None else weight.double()
    b = torch.zeros(c, dtype=torch.float64) if bias is None else bias.double()
    n = ((v - mu) * rstd).reshape(rows, c)
    z = n * w + b
    # the variance is a sum in chains of at most 256 additions: half of 256 half steps on rstd, the same on the mean in units of the
    # spread; the mean itself is an fp32 number: 2 half steps of it
    dz = EPS32 * (256 * (n.abs() + 1) * w.abs() + 2 * (mu.abs() * rstd).expand_as(v).reshape(rows, c) * w.abs() + 2 * b.abs() + 4 * z.abs())
    return act64(z, act, slope), act_error(z, dz, act)


def quantize64(x, block_rows):
    """-> (values as numbers, exponents) of the block quantiser: the smallest power of two s >= 2^-126 with max |x| <= 448 s."""
    rows, cols = x.shape
    x = x.double()
    rb, cb = -(-rows // block_rows), -(-cols // 128)
    full = torch.zeros(rb * block_rows, cb * 128, dtype=torch.float64)
    full[:rows, :cols] = torch.where(torch.isfinite(x), x.abs(), torch.zeros_like(x))
    amax = full.view(rb, block_rows, cb, 128).amax(dim=(1, 3))
    e = torch.zeros_like(amax)
    for i in range(rb):
        for j in range(cb):
            a = amax[i, j].item()
            if a > 0:
                k = -126
                while a > 448 * 2.0 ** k:
                    k += 1
                e[i, j] = k
    s = (2.0 ** e)[torch.arange(rows) // block_rows][:, torch.arange(cols) // 128]
    v = x / s
    step = torch.exp2(torch.floor(torch.log2(v.abs().nan_to_num(1.0, 1.0, 1.0).clamp(min=2.0 ** -6))) - 3)
    q = torch.round(v / step) * step                                       # torch.round: ties to even
    return torch.where(torch.isfinite(v), q, torch.full_like(q, float("nan"))), e


def dequantize64(values, scale, block_rows):
    """(rows, cols) float8 values and their block scales -> the numbers they stand for."""
    rows, cols = values.shape
    s = scale.contiguous().cpu()
    s = s.double() if s.dtype == torch.float32 else torch.exp2(s.view(torch.uint8).double() - 127)
    return values.contiguous().cpu().double() * s[torch.arange(rows) // block_rows][:, torch.arange(cols) // 128]


def matmul64(a, w, bias, act, residual, dtype, slope=0.01):
    """a (M, K), w (N, K) as numbers -> (y, allowed error): sums in fp32 in any order err by at most their length in half steps of the sum
    of magnitudes (K products that are exact, one scale factor each, one addition each). For 16-bit results the matrix instruction may
    drop, of each 8 products, what lies 13 binary places below the largest one's exponent: up to 7 * 2^-13 of the magnitudes."""
    k = a.shape[1]
    z = a @ w.t()
    dz = (EPS32 * (k + 8) + (0 if dtype == torch.float32 else 7 * 2.0 ** -13)) * (a.abs() @ w.abs().t())
    if bias is not None:
        z = z + bias.double()
        dz = dz + EPS32 * z.abs()
    y, dy = act64(z, act, slope), act_error(z, dz, act)
    if residual is not None:
        y = y + residual.double()
        dy = dy + EPS32 * y.abs()
    tiny = 2.0 ** -25 if dtype == torch.float16 else 2.0 ** -140          # half of the smallest step near zero
    return y, dy + HALF_STEP[dtype] * (y.abs() + dy) + tiny
