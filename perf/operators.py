"""The operators that a DP-trained block runs around its clipped layers, and what they are timed on.

Three operators, all of which keep the samples of a batch apart (no statistic, mask or scale of one sample depends on
another), which per-sample clipping needs:

  group_norm  group normalisation over channels-last input with the activation behind it and, optionally, the dropout
              behind that; the backward gives dx and the per-sample-clipped, averaged dgamma and dbeta
  dropout     dropout from a counter-based generator (and the residual sum behind it): no mask is stored, the
              backward draws it again
  fp8_linear  a layer's forward product and input gradient in 8-bit floating point (e4m3) with one scale for each
              block of 128: 1 x 128 along the contraction for activations and gradients, 128 x 128 for the weight;
              quantising all three is part of the pass

`run` computes them in elementary torch operations, or, where `own` is true, through `flashdp4review_b200.core`.
"""
import math

import torch

own = False

_DTYPES = {"fp32": torch.float32, "bf16": torch.bfloat16, "fp16": torch.float16}
_EPS = 1e-5
_CLAMP = 1.0
_M32 = 0xFFFFFFFF


# ---- cases -------------------------------------------------------------------------------------------
def _group_norm(name, b, t, c, groups, dtype, act, p):
    return {"name": name, "op": "group_norm", "b": b, "t": t, "c": c, "groups": groups, "dtype": dtype, "act": act, "p": p}


def _dropout(name, b, t, d, dtype, p, residual):
    return {"name": name, "op": "dropout", "b": b, "t": t, "d": d, "dtype": dtype, "p": p, "residual": residual}


def _fp8_linear(name, rows, k, n, dtype, bias):
    return {"name": name, "op": "fp8_linear", "rows": rows, "k": k, "n": n, "dtype": dtype, "bias": bias}


def listed():
    return [
        # the last stage of a small convolutional classifier, 8 x 8 positions: launches and host time
        _group_norm("group_norm_fp32_b4_t64_c128", 4, 64, 128, 32, "fp32", "none", 0.0),
        # the first stage of an image-to-image network, 64 x 64 positions, groups of ten channels
        _group_norm("group_norm_silu_bf16_b16_t4096_c320", 16, 4096, 320, 32, "bf16", "silu", 0.0),
        # the repository's LayerNorm configuration as a group norm, with the activation and dropout of an MLP
        _group_norm("group_norm_gelu_drop_bf16_b16_t1024_c1024", 16, 1024, 1024, 32, "bf16", "gelu_tanh", 0.1),
        # 37 x 37 positions and channels that no vector divides
        _group_norm("group_norm_gelu_fp16_b3_t1369_c90", 3, 1369, 90, 6, "fp16", "gelu", 0.0),
        # large images in the default dtype
        _group_norm("group_norm_silu_fp32_b8_t16384_c256", 8, 16384, 256, 16, "fp32", "silu", 0.0),
        # the repository's small single-layer configuration: launches and host time
        _dropout("dropout_fp32_b4_t128_d768", 4, 128, 768, "fp32", 0.1, False),
        # the residual branch of a GPT-2-medium block, micro-batch 16
        _dropout("dropout_add_bf16_b16_t1024_d1024", 16, 1024, 1024, "bf16", 0.1, True),
        # the hidden activations of an MLP of the same width, micro-batch 32
        _dropout("dropout_bf16_b32_t1024_d4096", 32, 1024, 4096, "bf16", 0.1, False),
        # the repository's small single-layer configuration in the default dtype
        _fp8_linear("fp8_linear_fp32_512_768x768", 512, 768, 768, "fp32", True),
        # padded image patches with a class token, widths that no block divides
        _fp8_linear("fp8_linear_fp16_2364_999x1000", 2364, 999, 1000, "fp16", True),
        # GPT-2-medium's MLP, micro-batch 16
        _fp8_linear("fp8_linear_bf16_16384_1024x4096", 16384, 1024, 4096, "bf16", True),
        # the up-projection of the Llama-2-7B-shaped decoder, micro-batch 4
        _fp8_linear("fp8_linear_bf16_8192_4096x11008", 8192, 4096, 11008, "bf16", False),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _width(rng, lo, hi):
    """Mostly multiples of 64, some of 8 only, now and then any number."""
    n = _log_int(rng, lo, hi)
    return max(lo, n // (step := rng.choice([64, 64, 64, 8, 8, 1])) * step)


def draw(rng):
    op = rng.choice(["group_norm", "group_norm", "dropout", "fp8_linear", "fp8_linear"])
    dtype = rng.choice(["fp32", "bf16", "bf16", "fp16"])
    if op == "group_norm":
        groups = rng.choice([1, 4, 8, 16, 32, 32, 6])
        c = max(1, _log_int(rng, 32, 2048) // groups) * groups
        b = _log_int(rng, 1, 64)
        # (a group of a few numbers is all cancellation: sixteen at least)
        t = max(min(_log_int(rng, 1, 16384), 33_000_000 // (b * c)), -(-16 * groups // c))
        case = _group_norm(None, b, t, c, groups, dtype, rng.choice(["none", "silu", "silu", "gelu", "gelu_tanh"]), rng.choice([0.0, 0.0, 0.1, 0.5]))
    elif op == "dropout":
        b, d = _log_int(rng, 1, 64), _width(rng, 16, 8192)
        t = min(_log_int(rng, 1, 4096), max(1, 100_000_000 // (b * d)))
        case = _dropout(None, b, t, d, dtype, rng.choice([0.05, 0.1, 0.1, 0.3, 0.5]), rng.random() < 0.5)
    else:
        rows, k, n = _log_int(rng, 1, 32768), _width(rng, 64, 11008), _width(rng, 64, 11008)
        rows = max(1, min(rows, int(3.6e11 / (k * n)), 150_000_000 // (k + n)))
        case = _fp8_linear(None, rows, k, n, dtype, rng.random() < 0.5)
    del case["name"]
    return case


# ---- inputs ------------------------------------------------------------------------------------------
def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    dtype = _DTYPES[case["dtype"]]

    def normal(*shape, scale=1.0, mean=0.0):
        return torch.randn(*shape, device="cuda", generator=gen) * scale + mean

    s = {"case": case, "seed": seed * 0x9E3779B97F4A7C15 & 0xFFFFFFFFFFFFFFFF}
    if case["op"] == "group_norm":
        b, t, c = case["b"], case["t"], case["c"]
        # what a convolution or projection leaves: channels of their own mean and spread
        s["x"] = (normal(b, t, c) * normal(c, scale=0.2, mean=1.5).abs() + normal(c, scale=0.5)).to(dtype)
        # mean-reduced losses give samples gradients of very different size
        s["dy"] = (normal(b, t, c, scale=1e-2) * torch.exp(normal(b, 1, 1))).to(dtype)
        s["weight"], s["bias"] = normal(c, scale=0.1, mean=1.0), normal(c, scale=0.1)
        s["clip"] = 1e-2 * math.sqrt(t * c)              # about the norm of a sample's dgamma: some are clipped, some are not
    elif case["op"] == "dropout":
        shape = (case["b"], case["t"], case["d"])
        s["x"], s["dy"] = normal(*shape).to(dtype), normal(*shape, scale=1e-2).to(dtype)
        s["residual"] = normal(*shape).to(dtype) if case["residual"] else None
    else:
        rows, k, n = case["rows"], case["k"], case["n"]
        s["x"] = (normal(rows, k) * torch.exp(0.5 * normal(1, k))).to(dtype)       # some features run larger than others
        s["g"] = (normal(rows, n, scale=1e-3) * torch.exp(normal(rows, 1))).to(dtype)
        s["weight"] = normal(n, k, scale=0.02).to(dtype)
        s["bias"] = normal(n, scale=0.02).to(dtype) if case["bias"] else None
    return s


# ---- the keep-mask -----------------------------------------------------------------------------------
def _mulhilo(m, x):
    prod = m * x                                          # wraps in 64 bits, whose two halves are still the product's
    return (prod >> 32) & _M32, prod & _M32


def _philox(c0, c1, c2, c3, k0, k1):
    """Philox4x32-10 on 32-bit words held in int64."""
    for _ in range(10):
        hi0, lo0 = _mulhilo(0xD2511F53, c0)
        hi1, lo1 = _mulhilo(0xCD9E8D57, c2)
        c0, c1, c2, c3 = hi1 ^ c1 ^ k0, lo1, hi0 ^ c3 ^ k1, lo0
        k0, k1 = (k0 + 0x9E3779B9) & _M32, (k1 + 0xBB67AE85) & _M32
    return c0, c1, c2, c3


def _halves(words):
    """The eight 16-bit numbers of a draw, low halves first."""
    w = torch.stack(words, dim=1)
    return torch.stack((w & 0xFFFF, w >> 16), dim=2).reshape(-1, 8)


def _keep(shape, device, p, seed):
    """Element i belongs to draw i // 8 of its stream; it is dropped where its 32 bits -- 16 of the draw, and below
    them 16 of a second one -- are less than p * 2^32."""
    n = math.prod(shape)
    group = torch.arange((n + 7) // 8, device=device)
    lo, hi = group & _M32, group >> 32
    zero = torch.zeros_like(group)
    k0, k1 = seed & _M32, (seed >> 32) ^ 0x44524F50
    top = _halves(_philox(lo, hi, zero + 1, zero + 1, k0, k1))
    low = _halves(_philox(lo, hi | 0x80000000, zero + 1, zero + 1, k0, k1))
    return ((top << 16 | low) >= round(p * 2 ** 32)).reshape(-1)[:n].reshape(shape)


# ---- plain forms -------------------------------------------------------------------------------------
def _act(z, act):
    """The activation and its derivative."""
    if act == "none":
        return z, torch.ones_like(z)
    if act == "silu":
        s = torch.sigmoid(z)
        return z * s, s * (1 + z * (1 - s))
    if act == "gelu":
        phi = 0.5 * (1 + torch.erf(z * math.sqrt(0.5)))
        return z * phi, phi + z * torch.exp(-0.5 * z * z) * (1 / math.sqrt(2 * math.pi))
    k = math.sqrt(2 / math.pi)
    h = torch.tanh(k * (z + 0.044715 * z * z * z))
    return 0.5 * z * (1 + h), 0.5 * (1 + h) + 0.5 * z * (1 - h * h) * k * (1 + 3 * 0.044715 * z * z)


def _clipped(per_sample, clip):
    norm = per_sample.double().square().sum(1).sqrt().float()
    factor = torch.clamp(clip / (norm + 1e-10), max=_CLAMP)
    return (per_sample * factor[:, None]).sum(0) / per_sample.shape[0]


def _plain_group_norm(s):
    case, dtype = s["case"], s["x"].dtype
    b, t, c, g, p = case["b"], case["t"], case["c"], case["groups"], case["p"]
    x, dy = s["x"].float(), s["dy"].float()
    keep = _keep(x.shape, x.device, p, s["seed"]) if p > 0 else None
    by_group = x.view(b, t, g, c // g)
    mean = by_group.mean((1, 3), dtype=torch.float64, keepdim=True)
    var = (by_group - mean).square().mean((1, 3), keepdim=True)
    rstd = (1 / (var + _EPS).sqrt()).float()
    xhat = ((by_group - mean).float() * rstd).view(b, t, c)
    rows = rstd.expand(b, 1, g, c // g).reshape(b, 1, c)
    a, slope = _act(xhat * s["weight"] + s["bias"], case["act"])
    y = a
    if keep is not None:
        y, dy = torch.where(keep, a * (1 / (1 - p)), 0.0), torch.where(keep, dy * (1 / (1 - p)), 0.0)
    gz = dy * slope
    dbeta, dgamma = gz.sum(1, dtype=torch.float64).float(), (gz * xhat).sum(1, dtype=torch.float64).float()
    n = t * c // g
    s1 = ((dbeta * s["weight"]).view(b, 1, g, -1).sum(3, keepdim=True) / n).expand(b, 1, g, c // g).reshape(b, 1, c)
    s2 = ((dgamma * s["weight"]).view(b, 1, g, -1).sum(3, keepdim=True) / n).expand(b, 1, g, c // g).reshape(b, 1, c)
    dx = rows * (gz * s["weight"] - s1 - xhat * s2)
    return {"y": y.to(dtype), "dx": dx.to(dtype), "dgamma": _clipped(dgamma, s["clip"]), "dbeta": _clipped(dbeta, s["clip"])}


def _plain_dropout(s):
    case, x = s["case"], s["x"]
    p = case["p"]
    keep = _keep(x.shape, x.device, p, s["seed"])
    y = torch.where(keep, x.float() * (1 / (1 - p)), 0.0)
    if s["residual"] is not None:
        y = y + s["residual"].float()
    return {"y": y.to(x.dtype), "dx": torch.where(keep, s["dy"].float() * (1 / (1 - p)), 0.0).to(x.dtype)}


def _power_scale(amax):
    """The smallest power of two that brings `amax` to at most 448, e4m3's largest number; 1 for a block of zeros."""
    m, e = torch.frexp(amax)
    return torch.where(amax > 0, torch.ldexp(torch.ones_like(amax), (e - torch.where(m <= 0.875, 9, 8)).clamp(min=-126)), torch.ones_like(amax))


def _blocked(a, rows):
    """`a` in whole blocks of rows x 128, zeros past its end: (row blocks, rows, column blocks, 128)."""
    r, c = a.shape
    a = torch.nn.functional.pad(a, (0, -c % 128, 0, -r % rows))
    return a.view(a.shape[0] // rows, rows, a.shape[1] // 128, 128)


def _dequantised(a, rows):
    """The values that `a` [., .] stands for in e4m3 with one scale for each block of rows x 128."""
    blocks = _blocked(a.float(), rows)
    scale = _power_scale(blocks.abs().amax((1, 3), keepdim=True))
    return ((blocks / scale).to(torch.float8_e4m3fn).float() * scale).reshape(blocks.shape[0] * rows, -1)[: a.shape[0], : a.shape[1]]


def _plain_fp8_linear(s):
    dtype = s["x"].dtype
    w = _dequantised(s["weight"], 128)
    y = _dequantised(s["x"], 1) @ w.t()
    if s["bias"] is not None:
        y = y + s["bias"].float()
    return {"y": y.to(dtype), "dx": (_dequantised(s["g"], 1) @ w).to(dtype)}


# ---- one pass ----------------------------------------------------------------------------------------
def _own(s):
    from flashdp4review_b200 import core

    case, x = s["case"], s["x"]
    if case["op"] == "fp8_linear":
        w8 = core.fp8_quantize_weight(s["weight"])
        return {"y": core.fp8_linear_forward(x, w8, s["bias"]), "dx": core.fp8_linear_input_grad(s["g"], w8)}
    spec = core.DropoutSpec(p=case["p"], seed=s["seed"], stream_id=1, step=1) if case["p"] > 0 else None
    if case["op"] == "dropout":
        return {"y": core.dropout(x, spec, residual=s["residual"]), "dx": core.dropout_backward(s["dy"], spec)}
    act = None if case["act"] == "none" else case["act"]
    y, stats = core.group_norm_forward(x, s["weight"], s["bias"], case["groups"], _EPS, activation=act, dropout=spec)
    dx, dgamma, dbeta = core.dp_group_norm_backward(
        s["dy"], x, s["weight"], s["bias"], stats["mean"], stats["rstd"], case["groups"], s["clip"], _CLAMP,
        activation=act, dropout=spec)
    return {"y": y, "dx": dx, "dgamma": dgamma, "dbeta": dbeta}


def run(s):
    if own:
        return _own(s)
    return {"group_norm": _plain_group_norm, "dropout": _plain_dropout, "fp8_linear": _plain_fp8_linear}[s["case"]["op"]](s)


# ---- what a pass cannot do without -------------------------------------------------------------------
def work(case):
    """Inputs read once, outputs written once; the multiply-adds of the products, and for the others the arithmetic of an
    element (the generator's included)."""
    elt = 4 if case["dtype"] == "fp32" else 2
    if case["op"] == "fp8_linear":
        rows, k, n = case["rows"], case["k"], case["n"]
        # x, g, weight and bias in; y and dx out
        return {"bytes": float(elt * (2 * rows * k + 2 * rows * n + k * n + (n if case["bias"] else 0))), "flops": 4.0 * rows * k * n}
    if case["op"] == "dropout":
        n = case["b"] * case["t"] * case["d"]
        return {"bytes": float(elt * n * (5 if case["residual"] else 4)), "flops": 30.0 * n}
    n = case["b"] * case["t"] * case["c"]
    # x and dy in, y and dx out; the forward ends before the gradient exists, so x is an input of both
    return {"bytes": float(elt * 5 * n + 16 * case["c"]), "flops": (40.0 if case["p"] == 0 else 60.0) * n}


# ---- from the definitions, in 64 bits ----------------------------------------------------------------
def _exact_e4m3(v):
    """Round to nearest even on e4m3's grid: three bits behind the leading one, which does not go below 2^-6."""
    _, e = torch.frexp(v)
    step = torch.ldexp(torch.ones_like(v), (e - 1).clamp(min=-6) - 3)
    return torch.round(v / step) * step


def _exact_blocks(a, down):
    """a [r, c] through e4m3, blocks of down x 128."""
    a = a.double()
    r, c = a.shape
    row_block = torch.arange(r, device=a.device) // down
    col_block = torch.arange(c, device=a.device) // 128
    wide = torch.zeros(r, int(col_block[-1]) + 1, dtype=torch.float64, device=a.device)
    wide.scatter_reduce_(1, col_block.expand(r, c), a.abs(), "amax")
    top = torch.zeros(int(row_block[-1]) + 1, wide.shape[1], dtype=torch.float64, device=a.device)
    top.scatter_reduce_(0, row_block[:, None].expand_as(wide), wide, "amax")
    exponent = torch.ceil(torch.log2((top / 448).clamp(min=2.0 ** -126)))
    # (a logarithm may miss the border of a power of two by its last bit)
    exponent = exponent - ((top <= 448 * torch.exp2(exponent - 1)) & (exponent > -126)).double()
    exponent = exponent + (top > 448 * torch.exp2(exponent)).double()
    scale = torch.exp2(exponent)[row_block][:, col_block]
    return _exact_e4m3(a / scale) * scale


def _exact_keep(case, s, shape):
    """The draw, word by word with 16-bit limbs in place of a wide product."""
    n = math.prod(shape)
    index = torch.arange(n, device="cuda")
    draw_no, place = index.div(8, rounding_mode="floor"), index.remainder(8)
    words = torch.zeros(2, 4, (n + 7) // 8, dtype=torch.int64, device="cuda")
    for second in (0, 1):
        numbers = torch.arange((n + 7) // 8, device="cuda")
        c = [numbers.remainder(1 << 32), numbers.div(1 << 32, rounding_mode="floor") + second * (1 << 31),
             torch.ones_like(numbers), torch.ones_like(numbers)]
        key = [s["seed"] % (1 << 32), (s["seed"] // (1 << 32)) ^ 0x44524F50]
        for turn in range(10):
            out = []
            for m, v in ((0xD2511F53, c[0]), (0xCD9E8D57, c[2])):
                low, high = v.remainder(1 << 16), v.div(1 << 16, rounding_mode="floor")
                first, then = low * m, high * m
                total_low = first + then.remainder(1 << 16) * (1 << 16)
                out.append((total_low.div(1 << 32, rounding_mode="floor") + then.div(1 << 16, rounding_mode="floor"), total_low.remainder(1 << 32)))
            (h0, l0), (h1, l1) = out
            c = [h1 ^ c[1] ^ ((key[0] + turn * 0x9E3779B9) % (1 << 32)), l1, h0 ^ c[3] ^ ((key[1] + turn * 0xBB67AE85) % (1 << 32)), l0]
        words[second] = torch.stack(c)
    which, shift = place.div(2, rounding_mode="floor"), 16 * place.remainder(2)
    top = torch.bitwise_right_shift(words[0][which, draw_no], shift).remainder(1 << 16)
    low = torch.bitwise_right_shift(words[1][which, draw_no], shift).remainder(1 << 16)
    return (top * (1 << 16) + low >= round(case["p"] * (1 << 32))).view(shape)


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "fp8_linear":
        x, g, w = _exact_blocks(s["x"], 1), _exact_blocks(s["g"], 1), _exact_blocks(s["weight"], 128)
        y = torch.einsum("rk,nk->rn", x, w)
        return {"y": y if s["bias"] is None else y + s["bias"].double(), "dx": torch.einsum("rn,nk->rk", g, w)}
    p = case["p"]
    kept = _exact_keep(case, s, s["x"].shape).double() / (1 - p) if p > 0 else 1.0
    x, dy = s["x"].double(), s["dy"].double()
    if case["op"] == "dropout":
        return {"y": x * kept if s["residual"] is None else x * kept + s["residual"].double(), "dx": dy * kept}
    b, t, c, g = case["b"], case["t"], case["c"], case["groups"]
    gamma, beta = s["weight"].double(), s["bias"].double()
    grouped = x.transpose(1, 2).reshape(b, g, -1)
    spread = torch.sqrt(grouped.var(2, unbiased=False, keepdim=True) + _EPS)
    xhat = ((grouped - grouped.mean(2, keepdim=True)) / spread).reshape(b, c, t)
    z = xhat * gamma[:, None] + beta[:, None]
    if case["act"] == "silu":
        a, slope = z / (1 + torch.exp(-z)), (1 + torch.exp(-z) * (1 + z)) / (1 + torch.exp(-z)) ** 2
    elif case["act"] == "gelu":
        cdf = torch.special.ndtr(z)
        a, slope = z * cdf, cdf + z * torch.exp(-z * z / 2) / math.sqrt(2 * math.pi)
    elif case["act"] == "gelu_tanh":
        # (1 + tanh u) / 2 = 1 / (1 + exp(-2 u))
        u = math.sqrt(2 / math.pi) * (z + 0.044715 * z ** 3)
        half = torch.sigmoid(2 * u)
        a, slope = z * half, half + z * 2 * half * (1 - half) * math.sqrt(2 / math.pi) * (1 + 0.134145 * z ** 2)
    else:
        a, slope = z, torch.ones_like(z)
    kept = kept.transpose(1, 2) if p > 0 else kept
    gz = dy.transpose(1, 2) * kept * slope
    per_beta, per_gamma = gz.sum(2), (gz * xhat).sum(2)
    gx = (gz * gamma[:, None]).reshape(b, g, -1)
    hat = xhat.reshape(b, g, -1)
    dx = (gx - gx.mean(2, keepdim=True) - hat * (gx * hat).mean(2, keepdim=True)) / spread
    out = {"y": (a * kept).transpose(1, 2), "dx": dx.reshape(b, c, t).transpose(1, 2)}
    for name, grads in (("dgamma", per_gamma), ("dbeta", per_beta)):
        length = torch.linalg.vector_norm(grads, dim=1, keepdim=True)
        out[name] = (grads * torch.clamp(s["clip"] / (length + 1e-10), max=_CLAMP)).mean(0)
    return out
