"""Plain 64-bit forms of the microscaled operators, shared by their tests.

A matrix is handled as (values of the elements, values of the block scales); `scale_tiles`
and `element_bytes` lay them out as include/b200gemm.h describes.
"""
from __future__ import annotations

import numpy as np

BLOCK = {"mxfp8": 32, "mxfp4": 32, "nvfp4": 16}
E2M1 = np.array([0, 0.5, 1, 1.5, 2, 3, 4, 6], dtype=np.float64)


def _e4m3_table():
    b = np.arange(127)
    e, f = b >> 3, b & 7
    return np.where(e > 0, (8 + f) * 2.0 ** (e - 10.0), f * 2.0 ** -9)


E4M3 = _e4m3_table()  # codes 0 ... 126


def nearest(v, table):
    """Code of the nearest table entry to |v|, ties to the even code, saturating. Table codes
    alternate in their lowest significand bit, so the even code is the even significand."""
    a = np.abs(v)
    hi = np.clip(np.searchsorted(table, a), 1, len(table) - 1)
    lo = hi - 1
    up, down = table[hi] - a, a - table[lo]
    code = np.where(up < down, hi, np.where(up > down, lo, np.where(hi % 2 == 0, hi, lo)))
    return np.where(a >= table[-1], len(table) - 1, code)


def pad_cols(x):
    return np.pad(x, ((0, 0), (0, -x.shape[1] % 32)))


def mx_exponent(amax, fmt):
    """Smallest e >= -127 with amax <= max * 2^e."""
    top = 448.0 if fmt == "mxfp8" else 6.0
    e = np.full(amax.shape, -127)
    with np.errstate(divide="ignore"):
        guess = np.floor(np.log2(np.where(amax > 0, amax, 1e-300) / top)).astype(int)
    for d in (-1, 0, 1, 2):
        g = np.maximum(guess + d, -127)
        e = np.where((amax > top * 2.0 ** e) & (g > e), g, e)
    return e


def found_scale(amax):
    """Tensor scale that the quantiser finds for a largest finite magnitude."""
    return np.float32(amax) * (np.float32(1) / np.float32(2688))


def quantize(x, fmt, tensor_scale=None):
    """(element codes, scale bytes), each (rows, n); x is 64-bit and holds the input exactly.
    Element codes carry the sign in their top bit; -0 is not told from 0."""
    x = pad_cols(np.asarray(x, dtype=np.float64))
    rows = x.shape[0]
    if fmt == "nvfp4" and tensor_scale is not None:
        with np.errstate(over="ignore", invalid="ignore"):
            r = np.float64(np.float32(1.0) / np.float32(tensor_scale))
            x = np.float64(np.float32(x * r))  # the operator holds u in fp32
    v = x.reshape(rows, -1, BLOCK[fmt])
    bad = ~np.isfinite(v).all(-1)
    vf = np.where(bad[..., None], 0.0, v)
    amax = np.abs(vf).max(-1)
    table, sign = (E4M3, 128) if fmt == "mxfp8" else (E2M1, 8)
    if fmt == "nvfp4":
        with np.errstate(over="ignore"):  # the definition's product, held in fp32
            byte = nearest(np.float64(np.float32(amax) * (np.float32(1) / np.float32(6))), E4M3)
        s = E4M3[byte]
        q = np.where(s[..., None] > 0, vf / np.where(s > 0, s, 1.0)[..., None], 0.0)
        byte = np.where(bad, 0x7F, byte)
    else:
        e = mx_exponent(amax, fmt)
        q = vf * 2.0 ** -e[..., None].astype(np.float64)
        byte = np.where(bad, 0xFF, e + 127)
    code = nearest(q, table)
    code = np.where((q < 0) & (code > 0), code + sign, code)
    return code.reshape(rows, -1).astype(np.uint8), byte.astype(np.uint8), bad


def element_values(code, fmt):
    if fmt == "mxfp8":
        t = np.append(E4M3, np.nan)
        return np.where(code >= 128, -1.0, 1.0) * t[code & 127]
    return np.where(code >= 8, -1.0, 1.0) * E2M1[code & 7]


def scale_values(byte, fmt):
    if fmt == "nvfp4":
        return np.append(E4M3, np.nan)[byte & 127]
    return np.where(byte == 255, np.nan, 2.0 ** (byte.astype(np.float64) - 127))


def values(code, byte, fmt, cols, tensor_scale=None):
    v = element_values(code, fmt).reshape(code.shape[0], -1, BLOCK[fmt]) * scale_values(byte, fmt)[..., None]
    v = v.reshape(code.shape[0], -1)[:, :cols]
    return v if tensor_scale is None else v * np.float64(np.float32(tensor_scale))


def element_bytes(code, fmt):
    if fmt == "mxfp8":
        return code
    return (code[:, 0::2] | (code[:, 1::2] << 4)).astype(np.uint8)


def element_codes(data, fmt):
    if fmt == "mxfp8":
        return data
    return np.stack([data & 15, data >> 4], -1).reshape(data.shape[0], -1)


def scale_tiles(byte):
    rows, n = byte.shape
    out = np.zeros((-(-rows // 128), -(-n // 4), 32, 16), dtype=np.uint8)
    r, c = np.arange(rows)[:, None], np.arange(n)[None, :]
    out[r // 128, c // 4, r % 32, r % 128 // 32 * 4 + c % 4] = byte
    return out


def scale_bytes(tiles, rows, n):
    r, c = np.arange(rows)[:, None], np.arange(n)[None, :]
    return tiles[r // 128, c // 4, r % 32, r % 128 // 32 * 4 + c % 4]


def unsigned_zero(code, fmt):
    """Codes with -0 turned into 0."""
    return np.where(code == (128 if fmt == "mxfp8" else 8), 0, code)


def random_operand(rng, rows, cols, fmt, exact=False):
    """(codes, scale bytes) with random elements. `exact`: integers up to 6 (4 bits) or 8 times
    block scales of 1, 2 or 4 (1, 1.5, 2, 3 for nvfp4), whose products and sums are multiples
    of 1/4 and stay far below 2^22, so that fp32 holds every partial sum exactly."""
    kp = -(-cols // 32) * 32
    n = kp // BLOCK[fmt]
    if exact:
        ints = np.array([0, 1, 2, 3, 4, 6], dtype=np.float64)
        val = rng.choice(ints, size=(rows, kp)) * rng.choice([-1.0, 1.0], size=(rows, kp))
        if fmt == "nvfp4":
            byte = nearest(rng.choice([1.0, 1.5, 2.0, 3.0], size=(rows, n)), E4M3)
        else:
            byte = 127 + rng.integers(0, 3, size=(rows, n))
    else:
        val = rng.standard_normal((rows, kp)) * (100.0 if fmt == "mxfp8" else 2.5)
        byte = (nearest(np.abs(rng.standard_normal((rows, n))) + 0.05, E4M3) if fmt == "nvfp4"
                else 127 + rng.integers(-6, 4, size=(rows, n)))
    code = nearest(val, E4M3 if fmt == "mxfp8" else E2M1)
    code = np.where((val < 0) & (code > 0), code + (128 if fmt == "mxfp8" else 8), code)
    code[:, cols:] = 0
    return code.astype(np.uint8), byte.astype(np.uint8)
