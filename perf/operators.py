"""What the MXFP4 and layer-norm operators are measured on: cases, inputs, the operators in elementary torch operations, the calls
a user makes of the framework, and the same results from the definitions in 64 bits.

  quantise   hk.quantize(x, E2M1) and hk.dequantize of its result: MXFP4 codes with one E8M0 scale per 32 elements, and the values they stand for
  product    hk.gemm / hk.gemm_scaled with E2M1 weights: C = A @ B^T (bf16), activations in E2M1, E2M3, E3M2, E4M3 or E5M2
  norm       hk.layer_norm (result in x's type) or hk.layer_norm_quantize (result as an MX operand), with mean and rstd
  norm_grad  hk.layer_norm_backward: dx, and the weight's and the bias's gradients summed over the rows
"""
import math

import torch

own = False

# element formats: the framework's code, bits, mantissa bits, exponent bias, exponent of the largest binade, largest value
FORMATS = {
    "e2m3": (0, 6, 3, 1, 2, 7.5),
    "e3m2": (1, 6, 2, 3, 4, 28.0),
    "e4m3": (2, 8, 3, 7, 8, 448.0),
    "e5m2": (3, 8, 2, 15, 15, 57344.0),
    "e2m1": (4, 4, 1, 1, 2, 6.0),
}
TYPES = {"bf16": torch.bfloat16, "fp32": torch.float32}
EPS = 1e-5


def listed():
    return [
        # a decode step's activations of 16 sequences on their way into a product: latency
        {"name": "quantise_step", "op": "quantise", "rows": 16, "K": 8192, "dtype": "bf16"},
        # a weight matrix quantised from its fp32 master copy, as after every optimiser step of quantised training
        {"name": "quantise_weights", "op": "quantise", "rows": 8192, "K": 8192, "dtype": "fp32"},
        # one token against a feed-forward weight, 4-bit weights and 8-bit activations: the weight stream is the work
        {"name": "decode_1_w4a8", "op": "product", "M": 1, "N": 28672, "K": 8192, "a": "e4m3", "epilogue": False},
        # 16 sequences, 4-bit on both sides
        {"name": "decode_16_w4a4", "op": "product", "M": 16, "N": 28672, "K": 8192, "a": "e2m1", "epilogue": False},
        # a ragged batch: rows, columns and scale rows off every tile and vector size, with channel scales and a bias
        {"name": "ragged_w4a4", "op": "product", "M": 1111, "N": 2050, "K": 1920, "a": "e2m1", "epilogue": True},
        # a prompt through the feed-forward up-projection, 6-bit activations
        {"name": "prompt_w4a6", "op": "product", "M": 4096, "N": 14336, "K": 8192, "a": "e2m3", "epilogue": False},
        # the square product of the framework's benchmark, 4-bit on both sides
        {"name": "square_w4a4", "op": "product", "M": 8192, "N": 8192, "K": 8192, "a": "e2m1", "epilogue": False},
        # the norm of a decode step
        {"name": "norm_step", "op": "norm", "rows": 16, "H": 8192, "dtype": "bf16", "to": "same"},
        # fp32 residual stream of an odd width (rows start off every vector boundary)
        {"name": "norm_odd", "op": "norm", "rows": 1500, "H": 1001, "dtype": "fp32", "to": "same"},
        # the norm in front of a projection of a long prompt, its result handed on as a 6-bit operand
        {"name": "norm_to_e2m3", "op": "norm", "rows": 16384, "H": 8192, "dtype": "bf16", "to": "e2m3"},
        # the gradient in a training step of 16384 tokens
        {"name": "norm_grad", "op": "norm_grad", "rows": 16384, "H": 8192, "dtype": "bf16"},
        # the gradient of a small odd layer
        {"name": "norm_grad_odd", "op": "norm_grad", "rows": 300, "H": 1001, "dtype": "fp32"},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["quantise", "product", "product", "norm", "norm_grad"])
    if op == "quantise":
        K = 32 * _log(rng, 1, 512)
        return {"op": op, "rows": _log(rng, 1, max(1, min(65536, 2**26 // K))), "K": K, "dtype": rng.choice(["bf16", "fp32"])}
    if op == "product":
        K = 128 * _log(rng, 1, 64)
        N = _log(rng, 16, 28672)
        return {"op": op, "M": _log(rng, 1, max(1, min(8192, 2**39 // (N * K), 2**26 // N))), "N": N, "K": K,
                "a": rng.choice(["e2m1", "e2m1", "e4m3", "e5m2", "e2m3", "e3m2"]), "epilogue": rng.random() < 0.3}
    to = rng.choice(["same", "same", "e2m3", "e3m2", "e4m3", "e5m2"]) if op == "norm" else "same"
    H = 32 * _log(rng, 1, 512) if to != "same" else _log(rng, 2, 16384)
    case = {"op": op, "rows": _log(rng, 1, max(1, min(65536, 2**27 // H))), "H": H, "dtype": rng.choice(["bf16", "bf16", "fp32"])}
    return dict(case, to=to) if op == "norm" else case


# ---------------------------------------------------------------------------------- the number format in elementary operations
def _quantised(x, fmt):
    """fp32 [rows, K] -> (magnitudes on the format's grid, signs, scale exponents), blocks of 32 along K."""
    _, _, mant, bias, emax, top = FORMATS[fmt]
    b = x.reshape(-1, 32)
    amax = b.abs().amax(1, keepdim=True)
    e = (torch.frexp(amax)[1] - 1 - emax).clamp(-127, 127)
    e = torch.where(amax > 0, e, torch.full_like(e, -127))
    mag = torch.ldexp(b.abs(), -e).clamp(max=top)
    step_e = (torch.frexp(mag)[1] - 1).clamp(min=1 - bias) - mant
    return torch.ldexp(torch.round(torch.ldexp(mag, -step_e)), step_e), b < 0, e


def _values(x, fmt):
    grid, neg, e = _quantised(x, fmt)
    return torch.ldexp(torch.where(neg, -grid, grid), e).reshape(x.shape)


def _magnitudes(fmt, device):
    """What the codes 0, 1, 2, ... without the sign bit stand for."""
    _, bits, mant, bias, _, _ = FORMATS[fmt]
    code = torch.arange(1 << (bits - 1), device=device)
    e, m = code >> mant, (code & ((1 << mant) - 1)).float()
    sub, norm = torch.ldexp(m, torch.full_like(code, 1 - bias - mant)), torch.ldexp(m + (1 << mant), e - bias - mant)
    return torch.where(e > 0, norm, sub)


def _packed(x, fmt):
    """fp32 [rows, K] -> operand bytes and E8M0 scale bytes."""
    bits = FORMATS[fmt][1]
    grid, neg, e = _quantised(x, fmt)
    code = torch.bucketize(grid, _magnitudes(fmt, x.device)) | (neg.long() << (bits - 1))
    code = code.to(torch.int32).reshape(x.shape[0], -1)
    if bits == 8:
        out = code
    elif bits == 4:
        out = code[:, 0::2] | (code[:, 1::2] << 4)
    else:
        w = code[:, 0::4] | (code[:, 1::4] << 6) | (code[:, 2::4] << 12) | (code[:, 3::4] << 18)
        out = torch.stack([w & 255, (w >> 8) & 255, w >> 16], -1).reshape(x.shape[0], -1)
    return out.to(torch.uint8).contiguous(), (e + 127).to(torch.uint8).reshape(x.shape[0], -1).contiguous()


def _unpacked(packed, fmt):
    bits = FORMATS[fmt][1]
    if bits == 8:
        return packed.to(torch.int32)
    if bits == 4:
        return torch.stack([packed & 15, packed >> 4], -1).reshape(packed.shape[0], -1).to(torch.int32)
    t = packed.to(torch.int32)
    w = t[:, 0::3] | (t[:, 1::3] << 8) | (t[:, 2::3] << 16)
    return torch.stack([w & 63, (w >> 6) & 63, (w >> 12) & 63, w >> 18], -1).reshape(packed.shape[0], -1)


def _decoded(packed, scales, fmt):
    bits = FORMATS[fmt][1]
    mag = _magnitudes(fmt, packed.device)
    v = torch.cat([mag, -mag])[_unpacked(packed, fmt)]
    return torch.ldexp(v.reshape(-1, 32), scales.reshape(-1, 1).to(torch.int32) - 127).reshape(v.shape)


# ---------------------------------------------------------------------------------- inputs
def _normal(g, *shape):
    return torch.randn(*shape, generator=g, device="cuda")


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(int(seed))
    s = {"case": case}
    if case["op"] == "quantise":
        # values whose blocks differ in size, as rows and channels of weights and activations do
        x = _normal(g, case["rows"], case["K"]).reshape(-1, 32)
        x = x * torch.exp(1.5 * _normal(g, x.shape[0], 1))
        s["x"] = x.reshape(case["rows"], case["K"]).to(TYPES[case["dtype"]])
    elif case["op"] == "product":
        M, N, K = case["M"], case["N"], case["K"]
        x = _normal(g, M, K)
        outlier = torch.rand(K, generator=g, device="cuda") < 1e-3      # channels far above the others
        s["A"], s["scale_A"] = _packed(torch.where(outlier, 50 * x, x), case["a"])
        s["B"], s["scale_B"] = _packed(0.02 * _normal(g, N, K), "e2m1")
        if case["epilogue"]:
            s["row"] = torch.exp(0.3 * _normal(g, M))
            s["col"] = torch.exp(0.3 * _normal(g, N))
            s["bias"] = _normal(g, N)
    else:
        rows, H, t = case["rows"], case["H"], TYPES[case["dtype"]]
        # a residual stream: rows with means and sizes of their own
        x = _normal(g, rows, H) * torch.exp(0.5 * _normal(g, rows, 1)) + _normal(g, rows, 1)
        s["x"] = x.to(t)
        s["weight"] = (1 + 0.2 * _normal(g, H)).to(t)
        s["bias"] = (0.2 * _normal(g, H)).to(t)
        if case["op"] == "norm_grad":
            s["dy"] = (0.1 * _normal(g, rows, H)).to(t)
            s["mean"], s["rstd"] = _stats(s["x"].float())
    return s


# ---------------------------------------------------------------------------------- the operators
def _stats(x):
    mean = x.mean(1)
    d = x - mean[:, None]
    return mean, 1 / torch.sqrt((d * d).mean(1) + EPS)


def run(s):
    case = s["case"]
    if own:
        import hipkittensp_b200 as hk

        if case["op"] == "quantise":
            packed, scales = hk.quantize(s["x"], hk.E2M1)
            return hk.dequantize(packed, scales, hk.E2M1, dtype=s["x"].dtype)
        if case["op"] == "product":
            fmt = FORMATS[case["a"]][0]
            if case["epilogue"]:
                return hk.gemm_scaled(s["A"], s["scale_A"], s["B"], s["scale_B"], s["row"], s["col"], s["bias"], fmt=fmt, fmt_b=hk.E2M1)
            return hk.gemm(s["A"], s["scale_A"], s["B"], s["scale_B"], fmt=fmt, fmt_b=hk.E2M1)
        if case["op"] == "norm_grad":
            dx, dweight, dbias = hk.layer_norm_backward(s["dy"], s["x"], s["mean"], s["rstd"], s["weight"])
            return {"dx": dx, "dweight": dweight, "dbias": dbias}
        if case["to"] == "same":
            y, mean, rstd = hk.layer_norm(s["x"], s["weight"], s["bias"], eps=EPS)
        else:
            fmt = FORMATS[case["to"]][0]
            packed, scales, mean, rstd = hk.layer_norm_quantize(s["x"], s["weight"], s["bias"], eps=EPS, fmt=fmt)
            y = hk.dequantize(packed, scales, fmt, dtype=torch.bfloat16)
        return {"y": y, "mean": mean, "rstd": rstd}

    if case["op"] == "quantise":
        return _values(s["x"].float(), "e2m1").to(s["x"].dtype)
    if case["op"] == "product":
        c = _decoded(s["A"], s["scale_A"], case["a"]) @ _decoded(s["B"], s["scale_B"], "e2m1").t()
        if case["epilogue"]:
            c = c * s["col"] * s["row"][:, None] + s["bias"]
        return c.to(torch.bfloat16)
    x, w = s["x"].float(), s["weight"].float()
    if case["op"] == "norm_grad":
        dy = s["dy"].float()
        xhat = (x - s["mean"][:, None]) * s["rstd"][:, None]
        wdy = dy * w
        dx = (wdy - wdy.mean(1, keepdim=True) - xhat * (wdy * xhat).mean(1, keepdim=True)) * s["rstd"][:, None]
        return {"dx": dx.to(s["x"].dtype), "dweight": (dy * xhat).sum(0), "dbias": dy.sum(0)}
    mean, rstd = _stats(x)
    y = (x - mean[:, None]) * rstd[:, None] * w + s["bias"].float()
    y = y.to(s["x"].dtype) if case["to"] == "same" else _values(y, case["to"]).to(torch.bfloat16)
    return {"y": y, "mean": mean, "rstd": rstd}


def work(case):
    if case["op"] == "quantise":
        n, t = case["rows"] * case["K"], TYPES[case["dtype"]].itemsize
        return {"bytes": n * (2 * t + 17 / 32), "flops": 4 * n}
    if case["op"] == "product":
        M, N, K = case["M"], case["N"], case["K"]
        operands = M * K * (FORMATS[case["a"]][1] / 8 + 1 / 32) + N * K * 17 / 32
        return {"bytes": operands + 2 * M * N + (4 * (M + 2 * N) if case["epilogue"] else 0), "flops": 2 * M * N * K}
    n, t = case["rows"] * case["H"], TYPES[case["dtype"]].itemsize
    if case["op"] == "norm_grad":
        return {"bytes": 3 * n * t + 8 * case["rows"] + case["H"] * (t + 8), "flops": 14 * n}
    result = t if case["to"] == "same" else FORMATS[case["to"]][1] / 8 + 1 / 32 + 2      # the codes and scales, and the values read back
    return {"bytes": n * (t + result) + 8 * case["rows"] + 2 * case["H"] * t, "flops": 8 * n}


# ---------------------------------------------------------------------------------- the definitions in 64 bits
def _grid64(fmt, device):
    """All non-negative values of a format, ascending, from its definition: k * 2^(lowest - mant) below 2^lowest, then binade by binade."""
    _, _, mant, bias, emax, top = FORMATS[fmt]
    lowest = 1 - bias
    v = [k * 2.0 ** (lowest - mant) for k in range(1 << mant)]
    for e in range(lowest, emax + 1):
        v += [(1 + k / (1 << mant)) * 2.0**e for k in range(1 << mant)]
    return torch.tensor([x for x in v if x <= top], dtype=torch.float64, device=device)


def _nearest64(x, fmt):
    """The MX value nearest to each element of a float64 [rows, K], ties to the even code."""
    emax = FORMATS[fmt][4]
    grid = _grid64(fmt, x.device)
    b = x.reshape(-1, 32)
    amax = b.abs().amax(1, keepdim=True)
    e = (torch.frexp(amax)[1] - 1 - emax).clamp(-127, 127)      # (log2 of an exact power of two may come out just below it)
    scale = torch.ldexp(torch.ones_like(amax), torch.where(amax > 0, e, torch.full_like(e, -127)))
    m = b.abs() / scale
    hi = torch.searchsorted(grid, m).clamp(1, grid.numel() - 1)
    lo = hi - 1
    below, above = m - grid[lo], grid[hi] - m
    pick = torch.where((above < below) | ((above == below) & (hi % 2 == 0)), hi, lo)
    return (torch.sign(b) * grid[pick] * scale).reshape(x.shape)


def _operand64(packed, scales, fmt):
    """Operand bytes -> the values in 64 bits: the K codes of a row are K * bits bits, lowest first."""
    bits, mant, bias = FORMATS[fmt][1:4]
    rows = packed.shape[0]
    stream = (packed[:, :, None] >> torch.arange(8, dtype=torch.uint8, device=packed.device)) & 1
    stream = stream.reshape(rows, -1, bits).double()
    weight = 2.0 ** torch.arange(bits, dtype=torch.float64, device=packed.device)
    m = (stream[..., :mant] * weight[:mant]).sum(-1)
    e = (stream[..., mant:bits - 1] * weight[: bits - 1 - mant]).sum(-1)
    v = torch.where(e > 0, (1 + m / (1 << mant)) * torch.exp2(e - bias), m * 2.0 ** (1 - bias - mant))
    v = v * (1 - 2 * stream[..., bits - 1])
    return v * torch.exp2(scales.double() - 127).repeat_interleave(32, 1)


def _operand64_in_parts(packed, scales, fmt):
    step = max(1, 2**24 // (packed.shape[1] * 8))
    return torch.cat([_operand64(packed[i:i + step], scales[i:i + step], fmt) for i in range(0, packed.shape[0], step)])


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "quantise":
        return _nearest64(s["x"].double(), "e2m1")
    if case["op"] == "product":
        c = _operand64_in_parts(s["A"], s["scale_A"], case["a"]) @ _operand64_in_parts(s["B"], s["scale_B"], "e2m1").t()
        if case["epilogue"]:
            c = s["row"].double()[:, None] * c * s["col"].double()[None, :] + s["bias"].double()[None, :]
        return c
    x, w = s["x"].double(), s["weight"].double()
    rows, H = x.shape
    if case["op"] == "norm_grad":
        # the gradient of sum(dy * y) by the chain rule through y = w * xhat + b, xhat = (x - mean) * rstd
        dy, rstd = s["dy"].double(), s["rstd"].double()[:, None]
        xhat = (x - s["mean"].double()[:, None]) * rstd
        dxhat = w * dy
        dx = rstd / H * (H * dxhat - dxhat.sum(1, keepdim=True) - xhat * torch.einsum("rh,rh->r", dxhat, xhat)[:, None])
        return {"dx": dx, "dweight": torch.einsum("rh,rh->h", dy, xhat), "dbias": torch.ones(rows, dtype=torch.float64, device=x.device) @ dy}
    mean = x.sum(1) / H
    var = (x * x).sum(1) / H - mean * mean
    y = (x - mean[:, None]) / torch.sqrt(var + EPS)[:, None] * w + s["bias"].double()
    return {"y": y if case["to"] == "same" else _nearest64(y, case["to"]), "mean": mean, "rstd": torch.rsqrt(var + EPS)}
