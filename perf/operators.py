"""Measured cases of the row operators: group norm with an activation (also straight into 8 bits), the block quantiser, and the
matrix product of 8-bit operands with a scale for each block of 128.

`own` chooses between the plain form (elementary torch operations in 32 bits) and the framework's kernels
(lssvc_amd.row_ops). Cases are plain dicts: see listed() for what each stands for.
"""
import math

import torch

own = False

DEV = "cuda:0"
TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
E4M3, E8M0 = torch.float8_e4m3fn, torch.float8_e8m0fnu      # 8-bit values; 8-bit scales that are powers of two
BLOCK = 128


# ---- cases ----------------------------------------------------------------------------------------------------------------
def _norm(op, images, h, w, c, groups, dtype, act, pad=0):
    # pad: the map is a channel slice of a buffer that is `pad` channels wider (channel concatenation and chunking make such views)
    return {"op": op, "images": images, "h": h, "w": w, "c": c, "groups": groups, "dtype": dtype, "act": act, "pad": pad}


def _quant(rows, cols, block_rows, dtype):
    return {"op": "quantize", "rows": rows, "cols": cols, "block_rows": block_rows, "dtype": dtype}


def _matmul(m, n, k, scales, dtype, act, bias, residual):
    return {"op": "matmul", "m": m, "n": n, "k": k, "scales": scales, "dtype": dtype, "act": act, "bias": bias, "residual": residual}


def listed():
    return [
        # the hyper-latent of a 1080p frame: one small map, latency is everything
        dict(_norm("norm", 1, 18, 30, 64, 8, "f32", "silu"), name="norm hyper-latent 18x30x64 f32"),
        # a batch of odd maps that live in a wider buffer (channel concatenation), odd group width
        dict(_norm("norm", 3, 37, 53, 100, 5, "f16", "lrelu", 12), name="norm 3x37x53x100 f16 slice"),
        # a full-resolution feature map of a 1080p frame: HBM-bound
        dict(_norm("norm", 1, 1152, 1920, 48, 8, "f32", "silu"), name="norm 1152x1920x48 f32"),
        # a 1/8-resolution feature map on its way into an 8-bit product
        dict(_norm("norm_fp8", 1, 144, 240, 256, 32, "bf16", "silu"), name="norm to fp8 144x240x256 bf16"),
        # small ragged maps on their way into an 8-bit product
        dict(_norm("norm_fp8", 2, 45, 77, 200, 8, "f16", "none"), name="norm to fp8 2x45x77x200 f16"),
        # the activations of a 1/8-resolution map, one scale for each pixel's 128 channels
        dict(_quant(34560, 768, 1, "bf16"), name="quantize 34560x768 bf16"),
        # a weight of odd sizes, one scale for each 128 x 128 block
        dict(_quant(1000, 5000, 128, "f32"), name="quantize weight 1000x5000 f32"),
        # one token through a square layer: the weight's bytes are the bound
        dict(_matmul(1, 4096, 4096, "pow2", "bf16", "none", True, False), name="matmul 1x4096x4096"),
        # a few tokens, odd widths, scales that are no powers of two
        dict(_matmul(24, 5000, 1000, "any", "f16", "silu", True, False), name="matmul 24x5000x1000 any scales"),
        # the widening product of a ConvFFN on a 36x60 map, fp32 out with a skip
        dict(_matmul(2160, 768, 192, "pow2", "f32", "lrelu", True, True), name="matmul 2160x768x192 f32 skip"),
        # a long batch with ragged sizes and checkpoint scales
        dict(_matmul(4000, 2500, 4096, "any", "bf16", "none", False, True), name="matmul 4000x2500x4096 any scales"),
        # the largest: bound by the matrix units
        dict(_matmul(8192, 8192, 8192, "pow2", "bf16", "silu", True, False), name="matmul 8192x8192x8192"),
    ]


def _log(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["norm", "norm", "norm_fp8", "quantize", "matmul", "matmul", "matmul"])
    dtype = rng.choice(["f32", "f16", "bf16"])
    if op in ("norm", "norm_fp8"):
        groups = rng.choice([1, 2, 4, 5, 8, 16, 32])
        c = groups * _log(rng, 1 if groups >= 8 else 8, 1024 // groups)
        images = rng.choice([1, 1, 1, 2, 3, 8])
        most = 1152 * 1920 * 48 // (images * c)                      # no more values than the largest listed map
        h = _log(rng, 4, min(1152, max(4, most // 4)))
        w = _log(rng, 4, min(1920, max(4, most // h)))
        return _norm(op, images, h, w, c, groups, dtype, rng.choice(["none", "relu", "lrelu", "silu"]), rng.choice([0, 0, 4, 16, 3]))
    if op == "quantize":
        return _quant(_log(rng, 1, 40000), _log(rng, 16, 8192) if rng.random() < 0.7 else 16 * _log(rng, 4, 64), rng.choice([1, 1, 128]), dtype)
    return _matmul(_log(rng, 1, 8192), _log(rng, 64, 8192), _log(rng, 64, 8192), rng.choice(["pow2", "pow2", "any"]), dtype,
                   rng.choice(["none", "relu", "lrelu", "silu"]), rng.random() < 0.6, rng.random() < 0.3)


# ---- inputs ---------------------------------------------------------------------------------------------------------------
def _gen(seed):
    g = torch.Generator(device=DEV)
    g.manual_seed(int(seed))
    return g


def _randn(g, *shape):
    return torch.randn(*shape, generator=g, device=DEV)


def _features(g, rows, cols):
    """Feature-map values: every channel has its own offset and spread, a few are far larger than the rest."""
    spread = torch.exp(0.7 * _randn(g, 1, cols))
    offset = 0.5 * _randn(g, 1, cols)
    return _randn(g, rows, cols).mul_(spread).add_(offset)


def _up(v, to):
    return (v + to - 1) // to * to


def _in_storage(values, cols, to):
    """8-bit values (rows, cols) in rows whose pitch is the next multiple of `to` bytes, zeros behind the last column."""
    store = torch.zeros(values.shape[0], _up(cols, to), dtype=torch.uint8, device=DEV)
    store[:, :cols] = values.view(torch.uint8)
    return store.view(values.dtype)[:, :cols]


def prepare(case, seed):
    g = _gen(seed)
    s = {"case": case}
    if case["op"] in ("norm", "norm_fp8"):
        rows, c = case["images"] * case["h"] * case["w"], case["c"]
        wide = _features(g, rows, c + case["pad"]).to(TYPES[case["dtype"]])
        s["x"] = wide[:, :c]
        s["weight"], s["bias"] = 1 + 0.2 * _randn(g, c), 0.2 * _randn(g, c)
    elif case["op"] == "quantize":
        s["x"] = _features(g, case["rows"], case["cols"]).to(TYPES[case["dtype"]])
    else:
        m, n, k = case["m"], case["n"], case["k"]
        qa, sa = _plain_quantize(_features(g, m, k), 1)
        qw, sw = _plain_quantize(_randn(g, n, k) / math.sqrt(k), BLOCK)
        if case["scales"] == "any":                                # scales of a checkpoint: fp32, no powers of two
            sa = _plain_scale(sa) * (0.6 + 0.8 * torch.rand(sa.shape, generator=g, device=DEV))
            sw = _plain_scale(sw) * (0.6 + 0.8 * torch.rand(sw.shape, generator=g, device=DEV))
        else:
            sa, sw = _in_storage(sa, sa.shape[1], 4), _in_storage(sw, sw.shape[1], 4)
        s["qa"], s["sa"], s["qw"], s["sw"] = _in_storage(qa, k, 16), sa, _in_storage(qw, k, 16), sw
        s["bias"] = 0.2 * _randn(g, n) if case["bias"] else None
        s["residual"] = _randn(g, m, n).to(TYPES[case["dtype"]]) if case["residual"] else None
        if own:
            from lssvc_amd.row_ops import Fp8Rows
            s["a"] = Fp8Rows(s["qa"], s["sa"])
            s["w"] = Fp8Rows(s["qw"], s["sw"], block_rows=BLOCK)
    return s


# ---- the plain forms ------------------------------------------------------------------------------------------------------
def _plain_act(y, act):
    if act == "relu":
        return y.clamp(min=0)
    if act == "lrelu":
        return torch.where(y >= 0, y, 0.01 * y)
    if act == "silu":
        return y / (1 + torch.exp(-y))
    return y


def _plain_norm(x, case, weight, bias):
    images, rows, groups = case["images"], case["h"] * case["w"], case["groups"]
    v = x.float().reshape(images, rows, groups, case["c"] // groups)
    v = v - v.mean(dim=(1, 3), keepdim=True)
    v = v * torch.rsqrt(v.square().mean(dim=(1, 3), keepdim=True) + 1e-5)
    return _plain_act(v.reshape(images * rows, case["c"]) * weight + bias, case["act"])


def _plain_quantize(x, block_rows):
    rows, cols = x.shape
    br, bc = (rows + block_rows - 1) // block_rows, (cols + BLOCK - 1) // BLOCK
    v = torch.zeros(br * block_rows, bc * BLOCK, dtype=torch.float32, device=x.device)
    v[:rows, :cols] = x
    v = v.view(br, block_rows, bc, BLOCK)
    amax = torch.where(torch.isfinite(v), v.abs(), 0).amax(dim=(1, 3), keepdim=True)
    mantissa, exponent = torch.frexp(amax)                          # amax = mantissa * 2^exponent, 448 = 0.875 * 2^9
    e = torch.where(amax > 0, (exponent - torch.where(mantissa <= 0.875, 9, 8)).clamp(min=-126), 0)
    scale = (e + 127).to(torch.uint8).view(E8M0)                    # 2^e
    q = (v / _plain_scale(scale)).to(E4M3).view(br * block_rows, bc * BLOCK)
    return q[:rows, :cols], scale.reshape(br, bc)


def _plain_scale(scale):
    """Scales in 32 bits: a power of two's 8 bits are the exponent field of the fp32 number."""
    return scale if scale.dtype == torch.float32 else (scale.view(torch.uint8).to(torch.int32) << 23).view(torch.float32)


def _plain_dequantize(q, scale, block_rows, rows, cols):
    full = _plain_scale(scale).repeat_interleave(block_rows, 0)[:rows].repeat_interleave(BLOCK, 1)[:, :cols]
    return q.float() * full


def _plain(s, case):
    if case["op"] == "norm":
        return {"y": _plain_norm(s["x"], case, s["weight"], s["bias"]).to(s["x"].dtype)}
    if case["op"] == "norm_fp8":
        q, scale = _plain_quantize(_plain_norm(s["x"], case, s["weight"], s["bias"]), 1)
        return {"values": q, "scale": scale}
    if case["op"] == "quantize":
        q, scale = _plain_quantize(s["x"], case["block_rows"])
        return {"values": q, "scale": scale}
    a = _plain_dequantize(s["qa"], s["sa"], 1, case["m"], case["k"])
    w = _plain_dequantize(s["qw"], s["sw"], BLOCK, case["n"], case["k"])
    y = a @ w.t()
    if s["bias"] is not None:
        y = y + s["bias"]
    y = _plain_act(y, case["act"])
    if s["residual"] is not None:
        y = y + s["residual"].float()
    return {"y": y.to(TYPES[case["dtype"]])}


# ---- the framework's calls ------------------------------------------------------------------------------------------------
def _act(case):
    return None if case["act"] == "none" else case["act"]


def _own(s, case):
    from lssvc_amd import row_ops
    if case["op"] == "norm":
        return {"y": row_ops.group_norm(s["x"], case["groups"], s["weight"], s["bias"], act=_act(case), images=case["images"])}
    if case["op"] == "norm_fp8":
        q = row_ops.group_norm_fp8(s["x"], case["groups"], s["weight"], s["bias"], act=_act(case), images=case["images"])
        return {"values": q.values, "scale": q.scale}
    if case["op"] == "quantize":
        q = row_ops.quantize_fp8(s["x"], block_rows=case["block_rows"])
        return {"values": q.values, "scale": q.scale}
    return {"y": row_ops.matmul_fp8(s["a"], s["w"], s["bias"], act=_act(case), residual=s["residual"], dtype=TYPES[case["dtype"]])}


def run(state):
    return _own(state, state["case"]) if own else _plain(state, state["case"])


# ---- work -----------------------------------------------------------------------------------------------------------------
def work(case):
    size = 4 if case["dtype"] == "f32" else 2
    if case["op"] in ("norm", "norm_fp8"):
        rows, c = case["images"] * case["h"] * case["w"], case["c"]
        out = rows * c * size if case["op"] == "norm" else rows * (c + (c + BLOCK - 1) // BLOCK)
        return {"bytes": rows * c * size + 8 * c + out, "flops": 8 * rows * c}
    if case["op"] == "quantize":
        rows, cols = case["rows"], case["cols"]
        blocks = ((rows + case["block_rows"] - 1) // case["block_rows"]) * ((cols + BLOCK - 1) // BLOCK)
        return {"bytes": rows * cols * (size + 1) + blocks, "flops": 3 * rows * cols}
    m, n, k = case["m"], case["n"], case["k"]
    kb = (k + BLOCK - 1) // BLOCK
    scales = (1 if case["scales"] == "pow2" else 4) * kb * (m + (n + BLOCK - 1) // BLOCK)
    return {"bytes": m * k + n * k + scales + m * n * size * (2 if case["residual"] else 1) + (4 * n if case["bias"] else 0), "flops": 2 * m * n * k}


# ---- the definitions, in 64 bits ------------------------------------------------------------------------------------------
def _exact_act(y, act):
    if act == "relu":
        return torch.relu(y)
    if act == "lrelu":
        return torch.maximum(y, y * 0.01)
    if act == "silu":
        return y * torch.sigmoid(y)
    return y


def _exact_norm(s, case):
    n, g = case["images"], case["groups"]
    x = s["x"].double().view(n, -1, g, case["c"] // g).transpose(1, 2).reshape(n, g, -1)
    var, mean = torch.var_mean(x, dim=2, correction=0, keepdim=True)
    x = ((x - mean) / (var + 1e-5).sqrt()).view(n, g, -1, case["c"] // g).transpose(1, 2).reshape(n, -1, case["c"])
    return _exact_act(x * s["weight"].double() + s["bias"].double(), case["act"]).view(-1, case["c"])


def _exact_e4m3(v):
    """v rounded to the nearest value of e4m3 (3 mantissa bits, smallest normal 2^-6), ties to even."""
    step = torch.exp2(torch.floor(torch.log2(v.abs().clamp(min=2.0 ** -6))).clamp(min=-6) - 3)
    return torch.round(v / step) * step


def _exact_quantize(x, block_rows):
    rows, cols = x.shape
    amax = torch.nn.functional.pad(x.abs(), (0, -cols % BLOCK, 0, -rows % block_rows))
    amax = amax.unflatten(1, (-1, BLOCK)).amax(2).unflatten(0, (-1, block_rows)).amax(1)
    e = torch.ceil(torch.log2(amax.clamp(min=1e-300) / 448))
    e = torch.where(amax > 448 * torch.exp2(e), e + 1, torch.where(amax <= 448 * torch.exp2(e - 1), e - 1, e)).clamp(min=-126)
    scale = torch.where(amax > 0, torch.exp2(e), 1.0)
    r, c = torch.arange(rows, device=x.device) // block_rows, torch.arange(cols, device=x.device) // BLOCK
    return _exact_e4m3(x / scale[r][:, c]), scale


def _exact_scale(scale):
    return scale.double() if scale.dtype == torch.float32 else torch.exp2(scale.contiguous().view(torch.uint8).double() - 127)


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "norm":
        return {"y": _exact_norm(s, case)}
    if case["op"] == "norm_fp8":
        q, scale = _exact_quantize(_exact_norm(s, case), 1)
        return {"values": q, "scale": scale}
    if case["op"] == "quantize":
        q, scale = _exact_quantize(s["x"].double(), case["block_rows"])
        return {"values": q, "scale": scale}
    m, n, k = case["m"], case["n"], case["k"]
    y = torch.zeros(m, n, dtype=torch.float64, device=DEV)
    at = torch.arange(n, device=DEV) // BLOCK
    for b in range((k + BLOCK - 1) // BLOCK):
        part = slice(b * BLOCK, min(k, (b + 1) * BLOCK))
        p = s["qa"][:, part].double() @ s["qw"][:, part].double().t()
        y += p * _exact_scale(s["sa"][:, b])[:, None] * _exact_scale(s["sw"][:, b])[at][None, :]
    if s["bias"] is not None:
        y += s["bias"].double()
    y = _exact_act(y, case["act"])
    return {"y": y + s["residual"].double() if s["residual"] is not None else y}
