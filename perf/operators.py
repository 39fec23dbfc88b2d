"""Cases of the microscaled operators: quantisation, dequantisation, product and RMS norm.

A microscaled matrix holds 8- or 4-bit elements and one scale for each block of
consecutive elements of a row:

  mxfp8   e4m3 elements, blocks of 32, scale 2^e (e8m0)
  mxfp4   e2m1 elements, blocks of 32, scale 2^e (e8m0)
  nvfp4   e2m1 elements, blocks of 16, scale e4m3, and one fp32 scale for the tensor

The element bytes are rows of ceil(cols / 32) * 32 elements (two 4-bit elements in a
byte, the first in the low half); the scale bytes are tiles of 128 rows x 4 blocks, in
which row r, block c is byte (r % 32) * 16 + (r / 32) * 4 + c. Padding is zero.

Each kind of case here:
  quantize   a matrix to mxfp8 elements and scales
  roundtrip  quantisation, then dequantisation: the values that the bits stand for
  gemm       C = A . B^T of two microscaled matrices
  norm       h = x + residual, RMS norm of h times the weight, to mxfp8; returns h too
  norm_gemm  the norm's output straight into a product with microscaled weights
  step       the three products of a linear layer's training step, on operands that the
             step quantises itself (along either axis)
"""
import importlib.util
import math
import sys
from pathlib import Path

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}
BLOCK = {"mxfp8": 32, "mxfp4": 32, "nvfp4": 16}
EPS = 1e-6


def _pkg():
    if "hopper_lab_b200" not in sys.modules:
        path = Path(__file__).resolve().parents[1] / "hopper-lab_b200" / "__init__.py"
        spec = importlib.util.spec_from_file_location("hopper_lab_b200", path)
        mod = importlib.util.module_from_spec(spec)
        sys.modules["hopper_lab_b200"] = mod
        spec.loader.exec_module(mod)
    return sys.modules["hopper_lab_b200"]


def listed():
    return [
        # one token's activations on their way into an 8-bit product: launch latency
        {"name": "quantize_token", "kind": "quantize", "fmt": "mxfp8", "dtype": "bf16", "rows": 1, "cols": 4096,
         "transpose": False},
        # a prompt's activations, or a weight matrix: bandwidth
        {"name": "quantize_matrix", "kind": "quantize", "fmt": "mxfp8", "dtype": "bf16", "rows": 8192, "cols": 8192,
         "transpose": False},
        # odd sizes, the tensor's scale found on the way: calibration and error studies
        {"name": "roundtrip_ragged", "kind": "roundtrip", "fmt": "nvfp4", "dtype": "f16", "rows": 1001, "cols": 5003,
         "transpose": False},
        # fp32 master weights quantised along their other axis, for a backward product
        {"name": "roundtrip_transposed", "kind": "roundtrip", "fmt": "mxfp4", "dtype": "f32", "rows": 4096,
         "cols": 8192, "transpose": True},
        # the repository's headline GEMM size, in 4 bits
        {"name": "gemm_square", "kind": "gemm", "fmt": "nvfp4", "dtype": "bf16", "M": 8192, "N": 8192, "K": 8192},
        # an 8-bit product of a middle size
        {"name": "gemm_8bit", "kind": "gemm", "fmt": "mxfp8", "dtype": "f16", "M": 4096, "N": 4096, "K": 4096},
        # a batch of odd length against odd weights
        {"name": "gemm_ragged", "kind": "gemm", "fmt": "mxfp4", "dtype": "bf16", "M": 777, "N": 5001, "K": 2200},
        # one token against a large weight matrix: decoding, bound by reading the weights
        {"name": "gemm_token", "kind": "gemm", "fmt": "nvfp4", "dtype": "bf16", "M": 1, "N": 8192, "K": 8192},
        # one token of the residual stream before a projection
        {"name": "norm_token", "kind": "norm", "fmt": "mxfp8", "dtype": "bf16", "rows": 1, "cols": 8192,
         "residual": True},
        # a prompt's residual stream
        {"name": "norm_matrix", "kind": "norm", "fmt": "mxfp8", "dtype": "bf16", "rows": 8192, "cols": 8192,
         "residual": True},
        # a decoding batch through norm and projection, in 4 bits
        {"name": "norm_gemm_batch", "kind": "norm_gemm", "fmt": "nvfp4", "dtype": "bf16", "M": 24, "N": 16384,
         "K": 4096},
        # forward and both backward products of a linear layer
        {"name": "linear_step", "kind": "step", "fmt": "mxfp8", "dtype": "bf16", "M": 4096, "N": 8192, "K": 4096},
    ]


def _log_uniform(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["quantize", "roundtrip", "gemm", "gemm", "norm", "norm_gemm", "step"])
    dtype = rng.choice(["bf16", "bf16", "f16", "f32"])
    fmt = rng.choice(["mxfp8", "mxfp4", "nvfp4"])
    if kind in ("quantize", "roundtrip"):
        return {"kind": kind, "fmt": "mxfp8" if kind == "quantize" else fmt, "dtype": dtype,
                "rows": _log_uniform(rng, 1, 8192), "cols": _log_uniform(rng, 17, 8192),
                "transpose": rng.random() < 0.4}
    if kind == "norm":
        return {"kind": kind, "fmt": "mxfp8", "dtype": dtype, "rows": _log_uniform(rng, 1, 8192),
                "cols": _log_uniform(rng, 64, 8192), "residual": rng.random() < 0.7}
    low = {"bf16": "bf16", "f16": "f16", "f32": "bf16"}[dtype]
    if kind == "norm_gemm":
        return {"kind": kind, "fmt": fmt, "dtype": low, "M": _log_uniform(rng, 1, 256),
                "N": _log_uniform(rng, 256, 16384), "K": _log_uniform(rng, 256, 8192)}
    if kind == "step":
        return {"kind": kind, "fmt": fmt, "dtype": low, "M": _log_uniform(rng, 64, 4096),
                "N": _log_uniform(rng, 128, 8192), "K": _log_uniform(rng, 128, 4096)}
    return {"kind": kind, "fmt": fmt, "dtype": low, "M": _log_uniform(rng, 1, 8192),
            "N": _log_uniform(rng, 64, 8192), "K": _log_uniform(rng, 64, 8192)}


# ------------------------------------------------------------------------- plain form
def _round_e2m1(v):
    """To the nearest of 0, 0.5, 1, 1.5, 2, 3, 4, 6; ties to the even significand."""
    a = v.abs()
    m = 0.5 * ((a > 0.25).float() + (a >= 0.75).float() + (a > 1.25).float() + (a >= 1.75).float())
    m = m + (a > 2.5).float() + (a >= 3.5).float() + 2.0 * (a > 5.0).float()
    return torch.where(v < 0, -m, m)


def _blocks(x, fmt):
    """(rows, padded columns / block, block) in 32 bits, padded with zeros to 32 columns."""
    x = x.float()
    pad = -x.shape[1] % 32
    if pad:
        x = torch.cat([x, x.new_zeros(x.shape[0], pad)], 1)
    return x.reshape(x.shape[0], -1, BLOCK[fmt])


def _tensor_scale(x):
    """amax / (6 * 448), the largest element times the largest block scale."""
    amax = x.float().abs().amax()
    return torch.where(amax > 0, (amax / 2688.0).clamp_min(2.0 ** -126), torch.ones_like(amax)).reshape(1)


def _quantize(x, fmt, tensor_scale=None):
    """Element values (rows, blocks, block) and block scales (rows, blocks), in 32 bits."""
    v = _blocks(x, fmt)
    if fmt == "nvfp4":
        if tensor_scale is not None:
            v = v * (1.0 / tensor_scale)
        s = (v.abs().amax(-1) / 6.0).clamp_max(448.0).to(torch.float8_e4m3fn).float()
        s1 = s.unsqueeze(-1)
        q = _round_e2m1(torch.where(s1 > 0, v / torch.where(s1 > 0, s1, 1.0), 0.0))
        return q, s
    # the smallest power of two that brings the largest element within the format's range
    emax, most = (8, 0.875) if fmt == "mxfp8" else (2, 0.75)
    mant, exp = torch.frexp(v.abs().amax(-1))
    e = exp - 1 - emax + (mant > most).to(exp.dtype)
    e = torch.where(mant > 0, e.clamp_min(-127), -127).double()
    v = v * torch.exp2(-e).float().unsqueeze(-1)
    q = v.to(torch.float8_e4m3fn).float() if fmt == "mxfp8" else _round_e2m1(v)
    return q, torch.exp2(e)


def _dequantize(q, s, tensor_scale, cols, dtype):
    v = q * s.float().unsqueeze(-1)
    if tensor_scale is not None:
        v = v * tensor_scale
    return v.reshape(q.shape[0], -1)[:, :cols].to(dtype)


def _tiles(s):
    """(rows, blocks) to tiles of 128 x 4, padded with zero bytes."""
    rows, n = s.shape
    s = torch.nn.functional.pad(s, (0, -n % 4, 0, -rows % 128))
    s = s.reshape(s.shape[0] // 128, 4, 32, s.shape[1] // 4, 4)
    return s.permute(0, 3, 2, 1, 4).reshape(s.shape[0], s.shape[3], 32, 16).contiguous()


def _untile(t, rows, n):
    t = t.reshape(t.shape[0], t.shape[1], 32, 4, 4).permute(0, 3, 2, 1, 4)
    return t.reshape(t.shape[0] * 128, -1)[:rows, :n]


def _scale_bytes(s, fmt):
    if fmt == "nvfp4":
        return s.to(torch.float8_e4m3fn).view(torch.uint8)
    return (torch.log2(s) + 127).to(torch.uint8)


def _pack(q, fmt):
    q = q.reshape(q.shape[0], -1)
    if fmt == "mxfp8":
        return q.to(torch.float8_e4m3fn).view(torch.uint8)
    steps = torch.tensor([0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0], device=q.device)
    code = torch.bucketize(q.abs(), steps).to(torch.uint8) | ((q < 0).to(torch.uint8) << 3)
    return code[:, 0::2] | (code[:, 1::2] << 4)


def _unpack(data, fmt):
    if fmt == "mxfp8":
        return data.view(torch.float8_e4m3fn).float()
    lut = torch.tensor([0, 0.5, 1, 1.5, 2, 3, 4, 6, -0.0, -0.5, -1, -1.5, -2, -3, -4, -6], device=data.device)
    return lut[torch.stack([data & 15, data >> 4], -1).long()].reshape(data.shape[0], -1)


def _decode(m):
    """A microscaled operand's values in 32 bits, without the tensor's scale."""
    q = _unpack(m["data"], m["fmt"])
    n = q.shape[1] // BLOCK[m["fmt"]]
    s = _untile(m["scales"], q.shape[0], n)
    s = s.view(torch.float8_e4m3fn).float() if m["fmt"] == "nvfp4" else torch.exp2(s.double() - 127).float()
    return (q.reshape(q.shape[0], n, -1) * s.unsqueeze(-1)).reshape(q.shape[0], -1)


def _scaled(v, *scales):
    for s in scales:
        if s is not None:
            v = v * s
    return v


def _norm(x, weight, residual):
    h = x.float() if residual is None else x.float() + residual.float()
    y = h * torch.rsqrt(h.square().mean(-1, keepdim=True) + EPS) * weight.float()
    return y, h


def _coded(q, s):
    """mxfp8 elements and scale tiles as 8-bit tensors, whose values the bytes stand for."""
    return {"elements": q.reshape(q.shape[0], -1).to(torch.float8_e4m3fn),
            "scales": _tiles(_scale_bytes(s, "mxfp8")).view(torch.float8_e8m0fnu)}


# ------------------------------------------------------------------------------ inputs
def _normal(gen, rows, cols, dtype, spread=1.0):
    """Normal values with a few columns ten times as large, as activations have them."""
    x = torch.randn(rows, cols, generator=gen, device="cuda") * spread
    big = torch.randint(0, cols, (max(1, cols // 256),), generator=gen, device="cuda")
    x[:, big] *= 10.0
    return x.to(dtype)


def _operand(gen, rows, cols, fmt, spread):
    x = _normal(gen, rows, cols, torch.float32, spread)
    ts = _tensor_scale(x) if fmt == "nvfp4" else None
    q, s = _quantize(x, fmt, ts)
    return {"fmt": fmt, "rows": rows, "cols": cols, "data": _pack(q, fmt), "scales": _tiles(_scale_bytes(s, fmt)),
            "tensor_scale": ts}


def _handle(m):
    return _pkg().MxTensor(m["data"], m["scales"], m["fmt"], m["rows"], m["cols"], m["tensor_scale"])


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    kind, fmt, dtype = case["kind"], case["fmt"], DTYPES[case["dtype"]]
    s = {"case": case}
    if kind in ("quantize", "roundtrip"):
        s["x"] = _normal(gen, case["rows"], case["cols"], dtype)
    elif kind == "norm":
        s["x"] = _normal(gen, case["rows"], case["cols"], dtype)
        s["residual"] = _normal(gen, case["rows"], case["cols"], dtype) if case["residual"] else None
        s["weight"] = (1.0 + 0.1 * torch.randn(case["cols"], generator=gen, device="cuda")).to(dtype)
    elif kind == "gemm":
        s["a"] = _operand(gen, case["M"], case["K"], fmt, 1.0)
        s["b"] = _operand(gen, case["N"], case["K"], fmt, case["K"] ** -0.5)
    elif kind == "norm_gemm":
        s["x"] = _normal(gen, case["M"], case["K"], dtype)
        s["residual"] = _normal(gen, case["M"], case["K"], dtype)
        s["weight"] = (1.0 + 0.1 * torch.randn(case["K"], generator=gen, device="cuda")).to(dtype)
        s["b"] = _operand(gen, case["N"], case["K"], fmt, case["K"] ** -0.5)
    else:
        s["x"] = _normal(gen, case["M"], case["K"], dtype)
        s["w"] = _normal(gen, case["N"], case["K"], dtype, case["K"] ** -0.5)
        s["dy"] = _normal(gen, case["M"], case["N"], dtype, 1e-3)
    if own:
        for k in ("a", "b"):
            if k in s:
                s[k] = _handle(s[k])
    return s


# -------------------------------------------------------------------------------- runs
def _run_own(s):
    p, case = _pkg(), s["case"]
    kind, fmt, dtype = case["kind"], case["fmt"], case["dtype"]
    if kind == "quantize":
        t = p.quantize_mx(s["x"], fmt, transpose=case["transpose"])
        return {"elements": t.data.view(torch.float8_e4m3fn), "scales": t.scales.view(torch.float8_e8m0fnu)}
    if kind == "roundtrip":
        return p.dequantize_mx(p.quantize_mx(s["x"], fmt, transpose=case["transpose"]), out_dtype=dtype)
    if kind == "norm":
        t, h = p.rms_norm_mx(s["x"], s["weight"], s["residual"], eps=EPS, fmt=fmt)
        return {"elements": t.data.view(torch.float8_e4m3fn), "scales": t.scales.view(torch.float8_e8m0fnu), "h": h}
    if kind == "gemm":
        return p.gemm_mx(s["a"], s["b"], out_dtype=dtype)
    if kind == "norm_gemm":
        t, h = p.rms_norm_mx(s["x"], s["weight"], s["residual"], eps=EPS, fmt=fmt)
        return {"c": p.gemm_mx(t, s["b"], out_dtype=dtype), "h": h}
    x, w, dy = s["x"], s["w"], s["dy"]
    y = p.gemm_mx(p.quantize_mx(x, fmt), p.quantize_mx(w, fmt), out_dtype=dtype)
    dx = p.gemm_mx(p.quantize_mx(dy, fmt), p.quantize_mx(w, fmt, transpose=True), out_dtype=dtype)
    dw = p.gemm_mx(p.quantize_mx(dy, fmt, transpose=True), p.quantize_mx(x, fmt, transpose=True), out_dtype=dtype)
    return {"y": y, "dx": dx, "dw": dw}


def _quantized(x, fmt):
    """The values in 32 bits that x's quantisation stands for, the tensor's scale included."""
    ts = _tensor_scale(x) if fmt == "nvfp4" else None
    q, s = _quantize(x, fmt, ts)
    return _dequantize(q, s, ts, x.shape[1], torch.float32)


def run(s):
    if own:
        return _run_own(s)
    case = s["case"]
    kind, fmt, dtype = case["kind"], case["fmt"], DTYPES[case["dtype"]]
    if kind == "quantize":
        return _coded(*_quantize(s["x"].t() if case["transpose"] else s["x"], fmt))
    if kind == "roundtrip":
        return _quantized(s["x"].t() if case["transpose"] else s["x"], fmt).to(dtype)
    if kind == "norm":
        y, h = _norm(s["x"], s["weight"], s["residual"])
        return {**_coded(*_quantize(y, fmt)), "h": None if s["residual"] is None else h.to(dtype)}
    if kind == "gemm":
        a, b = s["a"], s["b"]
        return _scaled(_decode(a) @ _decode(b).t(), a["tensor_scale"], b["tensor_scale"]).to(dtype)
    if kind == "norm_gemm":
        y, h = _norm(s["x"], s["weight"], s["residual"])
        a = _dequantize(*_quantize(y, fmt), None, case["K"], torch.float32)
        c = a @ _decode(s["b"])[:, :case["K"]].t()
        return {"c": _scaled(c, s["b"]["tensor_scale"]).to(dtype), "h": h.to(dtype)}
    x, w, dy = s["x"], s["w"], s["dy"]
    return {"y": (_quantized(x, fmt) @ _quantized(w, fmt).t()).to(dtype),
            "dx": (_quantized(dy, fmt) @ _quantized(w.t(), fmt).t()).to(dtype),
            "dw": (_quantized(dy.t(), fmt) @ _quantized(x.t(), fmt).t()).to(dtype)}


# -------------------------------------------------------------------------------- work
def _mx_bytes(rows, cols, fmt):
    bits = 8 if fmt == "mxfp8" else 4
    return rows * cols * (bits / 8 + 1 / BLOCK[fmt])


def work(case):
    kind, fmt, e = case["kind"], case["fmt"], DTYPES[case["dtype"]].itemsize
    if kind == "quantize":
        n = case["rows"] * case["cols"]
        return {"bytes": n * e + _mx_bytes(case["rows"], case["cols"], fmt), "flops": 3 * n}
    if kind == "roundtrip":
        n = case["rows"] * case["cols"]
        return {"bytes": 2 * n * e + 2 * _mx_bytes(case["rows"], case["cols"], fmt), "flops": 5 * n}
    if kind == "norm":
        n = case["rows"] * case["cols"]
        streams = 3 if case["residual"] else 1
        return {"bytes": n * e * streams + case["cols"] * e + _mx_bytes(case["rows"], case["cols"], fmt),
                "flops": 7 * n}
    M, N, K = case["M"], case["N"], case["K"]
    flops = 2 * M * N * K
    if kind == "gemm":
        return {"bytes": _mx_bytes(M, K, fmt) + _mx_bytes(N, K, fmt) + M * N * e, "flops": flops}
    if kind == "norm_gemm":
        return {"bytes": 3 * M * K * e + K * e + 2 * _mx_bytes(M, K, fmt) + _mx_bytes(N, K, fmt) + M * N * e,
                "flops": flops}
    quantized = _mx_bytes(M, K, fmt) + _mx_bytes(N, K, fmt) + _mx_bytes(M, N, fmt)
    return {"bytes": 2 * (M * K + N * K + M * N) * e + 4 * quantized, "flops": 3 * flops}


# ------------------------------------------------------------------ definition, 64 bits
def _exact_quantize(x, fmt, tensor_scale=None):
    """Element values and block scales in 64 bits; x (rows, cols) is already 64 bits."""
    rows, cols = x.shape
    full = torch.zeros(rows, -(-cols // 32) * 32, dtype=torch.float64, device=x.device)
    full[:, :cols] = x
    v = full.view(rows, -1, BLOCK[fmt])

    def grid(t, bits, low, top):
        # nearest multiple of the value's own step, ties to even, saturated
        _, e = torch.frexp(t)
        step = torch.exp2((e - 1).clamp_min(low).double() - bits)
        return (torch.round(t / step) * step).clamp(-top, top)

    def element(t):
        return grid(t, 3, -6, 448.0) if fmt == "mxfp8" else grid(t, 1, 0, 6.0)

    amax = v.abs().amax(-1)
    if fmt == "nvfp4":
        if tensor_scale is not None:
            # the operator scales by the fp32 reciprocal and holds the product in fp32
            r = (1.0 / tensor_scale.double()).float().double()
            v = (v * r).float().double()
            amax = v.abs().amax(-1)
        s = grid(amax / 6.0, 3, -6, 448.0)
        live = s > 0
        t = v / torch.where(live, s, torch.ones_like(s)).unsqueeze(-1)
        return element(t) * live.unsqueeze(-1), s
    most = 448.0 if fmt == "mxfp8" else 6.0
    e = torch.ceil(torch.log2(amax / most)).clamp_min(-127.0)
    # log2 may round across a power of two: settle by the inequality itself
    e = torch.where(amax > most * torch.exp2(e), e + 1, e)
    e = torch.where((e > -127) & (amax <= most * torch.exp2(e - 1)), e - 1, e)
    return element(v * torch.exp2(-e).unsqueeze(-1)), torch.exp2(e)


def _exact_tiles(s):
    rows, n = s.shape
    groups = -(-n // 4)
    out = torch.full((-(-rows // 128), groups, 32, 16), 2.0 ** -127, dtype=torch.float64, device=s.device)
    r = torch.arange(rows, device=s.device)[:, None]
    c = torch.arange(n, device=s.device)[None, :]
    out[r // 128, c // 4, r % 32, (r % 128) // 32 * 4 + c % 4] = s
    return out


def _exact_values(x, fmt):
    ts = None
    if fmt == "nvfp4":
        amax = x.abs().amax()
        ts = (amax.float() / 2688.0 if amax > 0 else torch.ones_like(amax).float())
    q, s = _exact_quantize(x, fmt, ts)
    v = (q * s.unsqueeze(-1)).reshape(x.shape[0], -1)[:, :x.shape[1]]
    return v if ts is None else v * ts.double()


def _exact_decode(m):
    data, fmt = m["data"], m["fmt"]
    if fmt == "mxfp8":
        b = data.long()
        e, f = (b >> 3) & 15, (b & 7).double()
        v = torch.where(e > 0, (8 + f) * torch.exp2(e.double() - 10), f * 2.0 ** -9)
        v = torch.where(b >= 128, -v, v)
    else:
        b = torch.empty(data.shape[0], data.shape[1] * 2, dtype=torch.int64, device=data.device)
        b[:, 0::2], b[:, 1::2] = (data % 16).long(), (data // 16).long()
        e, f = (b >> 1) & 3, (b & 1).double()
        v = torch.where(e > 0, (2 + f) * torch.exp2(e.double() - 2), 0.5 * f)
        v = torch.where(b >= 8, -v, v)
    r = torch.arange(v.shape[0], device=v.device)[:, None]
    c = torch.arange(v.shape[1] // BLOCK[fmt], device=v.device)[None, :]
    b = m["scales"][r // 128, c // 4, r % 32, (r % 128) // 32 * 4 + c % 4].long()
    if fmt == "nvfp4":
        e, f = b >> 3, (b & 7).double()
        s = torch.where(e > 0, (8 + f) * torch.exp2(e.double() - 10), f * 2.0 ** -9)
    else:
        s = torch.exp2(b.double() - 127)
    v = v * s.repeat_interleave(BLOCK[fmt], 1)
    return v if m["tensor_scale"] is None else v * m["tensor_scale"].double()


def _exact_norm(s):
    h = s["x"].double()
    if s["residual"] is not None:
        h = h + s["residual"].double()
    rms = (h.pow(2).sum(1, keepdim=True) / h.shape[1] + EPS).sqrt()
    return h / rms * s["weight"].double(), h


def exact(case, seed):
    s = prepare(case, seed)
    kind, fmt = case["kind"], case["fmt"]
    if kind in ("quantize", "roundtrip"):
        x = s["x"].double()
        x = x.t().contiguous() if case["transpose"] else x
        if kind == "roundtrip":
            return _exact_values(x, fmt)
        q, sc = _exact_quantize(x, fmt)
        return {"elements": q.reshape(x.shape[0], -1), "scales": _exact_tiles(sc)}
    if kind == "norm":
        y, h = _exact_norm(s)
        q, sc = _exact_quantize(y, fmt)
        return {"elements": q.reshape(y.shape[0], -1), "scales": _exact_tiles(sc),
                "h": None if s["residual"] is None else h}
    if kind == "gemm":
        return _exact_decode(s["a"]) @ _exact_decode(s["b"]).t()
    if kind == "norm_gemm":
        y, h = _exact_norm(s)
        q, sc = _exact_quantize(y, fmt)
        a = (q * sc.unsqueeze(-1)).reshape(y.shape[0], -1)
        return {"c": a @ _exact_decode(s["b"]).t(), "h": h}
    x, w, dy = s["x"].double(), s["w"].double(), s["dy"].double()
    return {"y": _exact_values(x, fmt) @ _exact_values(w, fmt).t(),
            "dx": _exact_values(dy, fmt) @ _exact_values(w.t().contiguous(), fmt).t(),
            "dw": _exact_values(dy.t().contiguous(), fmt) @ _exact_values(x.t().contiguous(), fmt).t()}
