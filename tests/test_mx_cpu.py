"""Microscaled operators without a GPU: sizes, struct layouts, refusals (all of them before any
device work), and the plain forms of mx_check.py against values worked out by hand."""
import ctypes as C
import subprocess
from pathlib import Path

import numpy as np
import pytest

import mx_check as X

ROOT = Path(__file__).resolve().parents[1]


# ----------------------------------------------------------------------- plain forms
def test_plain_e2m1_and_e4m3_rounding():
    v = np.array([0.25, 0.26, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0, 5.01, 7.0])
    np.testing.assert_array_equal(X.E2M1[X.nearest(v, X.E2M1)], [0, 0.5, 1, 1, 2, 2, 4, 4, 6, 6])
    assert X.E4M3[-1] == 448 and X.E4M3[1] == 2.0 ** -9 and X.E4M3[8] == 2.0 ** -6 and X.E4M3[0x38] == 1.0
    import torch

    r = np.random.default_rng(0).standard_normal(4000) * np.exp2(np.arange(4000) % 22 - 12.0)
    r = np.clip(np.float32(r), -448, 448)
    want = torch.from_numpy(r).to(torch.float8_e4m3fn).float().abs().numpy()
    np.testing.assert_array_equal(X.E4M3[X.nearest(r.astype(np.float64), X.E4M3)], want)


def test_plain_scales():
    amax = np.array([6.0, 6.001, 3.0, 448.0, 0.0, 1e-45])
    np.testing.assert_array_equal(X.mx_exponent(amax, "mxfp4"), [0, 1, -1, 7, -127, -127])
    np.testing.assert_array_equal(X.mx_exponent(np.array([448.0, 449.0, 1.75, 1.76]), "mxfp8"), [0, 1, -8, -7])


@pytest.mark.parametrize("fmt", list(X.BLOCK))
def test_plain_quantisation_error_is_half_a_step(fmt):
    rng = np.random.default_rng(1)
    x = np.float32(rng.standard_normal((20, 90))).astype(np.float64)
    code, byte, _ = X.quantize(x, fmt)
    v = X.values(code, byte, fmt, 90)
    s = np.repeat(X.scale_values(byte, fmt), X.BLOCK[fmt], 1)[:, :90]
    if fmt == "mxfp8":  # relative 2^-4 of a normal element, 2^-10 of the scale below
        assert (np.abs(v - x) <= np.maximum(2.0 ** -4 * np.abs(x), 2.0 ** -10 * s)).all()
    else:  # half of the step between 4 and 6, or a block scale rounded down by 2^-4 saturating at 6
        assert (np.abs(v - x) <= s).all()
    np.testing.assert_array_equal(X.scale_bytes(X.scale_tiles(byte), *byte.shape), byte)
    np.testing.assert_array_equal(X.element_codes(X.element_bytes(code, fmt), fmt), code)


# ------------------------------------------------------------------------------ sizes
@pytest.mark.parametrize("fmt,rows,cols,row,scale", [
    ("mxfp8", 1, 1, 32, 512), ("mxfp8", 128, 128, 128, 512), ("mxfp8", 129, 129, 160, 2 * 2 * 512),
    ("mxfp4", 1, 33, 32, 512), ("mxfp4", 300, 1000, 512, 3 * 8 * 512), ("nvfp4", 1, 64, 32, 512),
    ("nvfp4", 1, 65, 48, 1024), ("nvfp4", 257, 8192, 4096, 3 * 128 * 512), ("mxfp8", 0, 64, 64, 0),
    ("mxfp4", 5, 0, 0, 0)])
def test_layout(b200, fmt, rows, cols, row, scale):
    assert b200.mx_layout(fmt, rows, cols) == (row, scale)


def test_layout_refusals(b200):
    L = b200.lib()
    assert L.b200_mx_layout(3, 1, 1, None, None) == b200.ERR_INVALID_ARG
    assert L.b200_mx_layout(0, -1, 1, None, None) == b200.ERR_SHAPE
    assert L.b200_mx_layout(0, 1, 1 << 31, None, None) == b200.ERR_SHAPE


def test_struct_layouts_match_c(b200, tmp_path):
    for name, mirror in (("B200MxTensor", b200.MxDesc), ("B200MxNormArgs", b200.MxNormArgs)):
        fields = [f for f, _ in mirror._fields_]
        body = "\n".join(f'  printf("%zu\\n", offsetof({name}, {f}));' for f in fields)
        prog = tmp_path / f"{name}.c"
        prog.write_text(f'#include <stddef.h>\n#include <stdio.h>\n#include "b200gemm.h"\nint main(void) {{\n{body}\n'
                        f'  printf("%zu\\n", sizeof({name}));\n  return 0;\n}}\n')
        exe = tmp_path / name
        subprocess.run(["gcc", "-std=c99", f"-I{ROOT / 'include'}", str(prog), "-o", str(exe)], check=True)
        out = subprocess.run([str(exe)], capture_output=True, text=True, check=True).stdout.split()
        assert [int(v) for v in out] == [getattr(mirror, f).offset for f in fields] + [C.sizeof(mirror)]


# --------------------------------------------------------------------------- refusals
def _desc(b200, **kw):
    d = b200.MxDesc(1, 0, 200, 256, 128, 0x10000, 0x20000, None)
    for k, v in kw.items():
        setattr(d, k, v)
    return d


BAD = [
    ({"format": 3}, -1), ({"format": -1}, -1), ({"reserved": 1}, -1), ({"rows": -1}, -2), ({"cols": -1}, -2),
    ({"rows": (1 << 31) - 1}, -2), ({"cols": 1 << 31}, -2), ({"ld": 127}, -2), ({"ld": 112}, -2), ({"ld": 1 << 40}, -2),
    ({"ld": 136}, -3), ({"data": None}, -1), ({"scales": None}, -1), ({"data": 0x10008}, -3),
    ({"scales": 0x20004}, -3), ({"tensor_scale": 0x30000}, -1),  # no tensor scale in this format
    ({"format": 2, "tensor_scale": 0x30002}, -3)]


@pytest.mark.parametrize("kw,code", BAD)
def test_operand_refusals(b200, kw, code):
    L, bad, good = b200.lib(), _desc(b200, **kw), _desc(b200)
    if "format" in kw and kw["format"] == 2:
        good.format = 2
    assert L.b200_mx_quantize(0x40000, 1, 256, 0, 0, C.byref(bad), None) == code
    assert L.b200_mx_dequantize(C.byref(bad), 0x40000, 1, 256, None) == code
    assert L.b200_mx_gemm(C.byref(bad), C.byref(good), 0x40000, 1, 200, None) == code
    assert L.b200_mx_gemm(C.byref(good), C.byref(bad), 0x40000, 1, 200, None) == code
    args = b200.MxNormArgs(1, 1, 0x40000, 0x50000, None, None, 256, 0, 0, 1e-6, 0)
    assert L.b200_mx_rms_norm(C.byref(args), C.byref(bad), None) == code


def test_quantize_refusals(b200):
    L, d, nv = b200.lib(), _desc(b200), _desc(b200, format=2, tensor_scale=0x30010)
    call = lambda x, dt, ld, tr, find, t: L.b200_mx_quantize(x, dt, ld, tr, find, C.byref(t), None)  # noqa: E731
    assert L.b200_mx_quantize(0x40000, 1, 256, 0, 0, None, None) == -1
    assert call(0x40000, 2, 256, 0, 0, d) == -1      # e4m3 is not an input type
    assert call(None, 1, 256, 0, 0, d) == -1
    assert call(0x40000, 1, 255, 0, 0, d) == -2      # ldx < cols
    assert call(0x40000, 1, 199, 1, 0, d) == -2      # transposed: ldx < rows
    assert call(0x40001, 1, 256, 0, 0, d) == -3
    assert call(0x40002, 3, 256, 0, 0, d) == -3
    assert call(0x40000, 1, 256, 0, 1, d) == -1      # no tensor scale to find in an MX format
    assert call(0x40000, 1, 256, 0, 1, _desc(b200, format=2)) == -1
    assert call(0x40000, 1, 256, 0, 1, _desc(b200, format=2, tensor_scale=0x30004)) == -3  # not 16-byte aligned
    assert call(0x40000, 1, 256, 0, 0, _desc(b200, rows=0)) == 0
    if not _gpu():
        assert call(0x40000, 1, 256, 0, 1, nv) == b200.ERR_CUDA
        assert call(0x40000, 1, 256, 1, 0, d) == b200.ERR_CUDA


def test_dequantize_refusals(b200):
    L, d = b200.lib(), _desc(b200)
    call = lambda y, dt, ld, t: L.b200_mx_dequantize(C.byref(t), y, dt, ld, None)  # noqa: E731
    assert call(0x40000, 2, 256, d) == -1
    assert call(None, 1, 256, d) == -1
    assert call(0x40000, 1, 255, d) == -2
    assert call(0x40001, 1, 256, d) == -3
    assert call(0x40000, 1, 256, _desc(b200, cols=0)) == 0


def test_gemm_refusals(b200):
    L, a, b = b200.lib(), _desc(b200), _desc(b200, rows=100)
    call = lambda x, y, c, dt, ld: L.b200_mx_gemm(C.byref(x), C.byref(y), c, dt, ld, None)  # noqa: E731
    assert L.b200_mx_gemm(None, C.byref(b), 0x40000, 1, 100, None) == -1
    assert L.b200_mx_gemm(C.byref(a), None, 0x40000, 1, 100, None) == -1
    assert call(a, _desc(b200, format=2), 0x40000, 1, 200) == -1   # formats differ
    assert call(a, _desc(b200, cols=250), 0x40000, 1, 200) == -2   # K differs
    assert call(a, b, 0x40000, 2, 100) == -1                       # no e4m3 output
    assert call(a, b, None, 1, 100) == -1
    assert call(a, b, 0x40000, 1, 99) == -2
    assert call(a, b, 0x40001, 1, 100) == -3
    assert call(a, b, 0x40002, 3, 100) == -3
    assert call(_desc(b200, rows=0), b, None, 1, 100) == 0
    if not _gpu():
        assert call(a, b, 0x40000, 1, 100) == b200.ERR_CUDA


def test_norm_refusals(b200):
    L, d = b200.lib(), _desc(b200)
    ok = dict(dtype=1, weight_dtype=1, x=0x40000, weight=0x50000, residual=0x60000, h=0x70000, ldx=256, ldr=256,
              ldh=256, eps=1e-6, reserved=0)

    def call(t=d, **kw):
        a = b200.MxNormArgs(**{**ok, **kw})
        return L.b200_mx_rms_norm(C.byref(a), C.byref(t), None)

    assert L.b200_mx_rms_norm(None, C.byref(d), None) == -1
    for kw, code in (({"dtype": 2}, -1), ({"weight_dtype": 0}, -1), ({"x": None}, -1), ({"weight": None}, -1),
                     ({"h": None}, -1), ({"ldx": 255}, -2), ({"ldr": 255}, -2), ({"ldh": 255}, -2),
                     ({"x": 0x40001}, -3), ({"weight": 0x50001}, -3), ({"residual": 0x60001}, -3),
                     ({"h": 0x70001}, -3), ({"weight_dtype": 3, "weight": 0x50002}, -3), ({"eps": -1.0}, -1),
                     ({"eps": float("nan")}, -1), ({"eps": float("inf")}, -1), ({"reserved": 1}, -1)):
        assert call(**kw) == code, kw
    wide = _desc(b200, cols=b200.MX_NORM_MAX_COLS + 1, ld=1 << 15)
    assert call(wide, ldx=1 << 16, ldr=1 << 16, ldh=1 << 16) == -2
    assert call(_desc(b200, rows=0), x=None) == 0
    if not _gpu():
        assert call() == b200.ERR_CUDA
        assert call(residual=None, h=None, ldr=0, ldh=0) == b200.ERR_CUDA


def test_python_refusals(b200):
    import torch

    def mk(fmt="mxfp4", rows=4, cols=64, ts=None, device="cpu"):
        return b200.MxTensor.empty(rows, cols, fmt, device, ts)

    t = mk()
    assert t.shape == (4, 64) and t.data.shape == (4, 32) and t.scales.shape == (1, 1, 32, 16)
    with pytest.raises(ValueError):
        b200.MxTensor(t.data[:, :16], t.scales, "mxfp4", 4, 64)
    with pytest.raises(ValueError):
        b200.MxTensor(t.data, t.scales[..., :8], "mxfp4", 4, 64)
    with pytest.raises(TypeError):
        b200.MxTensor(t.data.to(torch.int8), t.scales, "mxfp4", 4, 64)
    with pytest.raises(ValueError):
        mk(ts=torch.ones(1))                      # an MX format has no tensor scale
    with pytest.raises(ValueError):
        mk("nvfp4", ts=torch.ones(2))
    with pytest.raises(KeyError):
        mk("mxfp6")
    x = torch.randn(4, 64)
    with pytest.raises(ValueError):
        b200.quantize_mx(x, "mxfp4")              # not on a GPU
    with pytest.raises(TypeError):
        b200.quantize_mx(x.double(), "mxfp4")
    with pytest.raises(ValueError):
        b200.quantize_mx(x[None], "mxfp4")
    with pytest.raises(ValueError):
        b200.quantize_mx(x[:, ::2], "mxfp4")
    with pytest.raises(TypeError):
        b200.gemm_mx(t, mk("mxfp8"))
    with pytest.raises(ValueError):
        b200.gemm_mx(t, mk(cols=32))
    with pytest.raises(ValueError):
        b200.gemm_mx(t, t)
    with pytest.raises(ValueError):
        b200.dequantize_mx(t)
    w = torch.ones(64)
    with pytest.raises(ValueError):
        b200.rms_norm_mx(x, w[:32])
    with pytest.raises(TypeError):
        b200.rms_norm_mx(x, w.half())
    with pytest.raises(ValueError):
        b200.rms_norm_mx(x, w, residual_out=x)
    with pytest.raises(ValueError):
        b200.rms_norm_mx(x, w)


def _gpu():
    import torch

    return torch.cuda.is_available()
