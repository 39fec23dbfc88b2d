"""GPU tests of the microscaled operators against plain 64-bit forms (mx_check.py).

Tolerances
- quantisation and dequantisation: every element and scale byte equals the definition's
  (only the sign of a zero element is free); dequantised values equal the exact ones rounded
  once, with a tensor scale within one fp32 rounding more (2^-24 relative, twice).
- products: with integer data the fp32 result is exact. With real data the tensor core adds
  32-byte slices of K (32 or 64 terms) to an fp32 accumulator; alignment and truncation lose
  at most one unit of the last place (2^-23) of the sum of magnitudes per slice, so the bound
  is (K / 32 + 2) * 2^-23 * sum|a b|, plus half a step of the output type.
- RMS norm: y in fp32 carries the roundings of a sum of positive terms (at most 64 deep,
  64 * 2^-24), of rsqrt (2^-22) and three products, together below 2^-17 relative; element
  and scale codes must be those of some value within 2^-17 of the exact one.
"""
from __future__ import annotations

import numpy as np
import pytest

import mx_check as X

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

FMTS = ["mxfp8", "mxfp4", "nvfp4"]
DT = {"f16": torch.float16, "bf16": torch.bfloat16, "f32": torch.float32}
HALF_STEP = {"f16": 2.0 ** -11, "bf16": 2.0 ** -8, "f32": 2.0 ** -24}


@pytest.fixture(scope="module", autouse=True)
def _cuda():
    if not torch.cuda.is_available():
        pytest.skip("no CUDA device")
    yield
    torch.cuda.synchronize()


def _f64(t):
    return t.double().cpu().numpy()


def _input(seed, rows, cols, dtype, spread=1.0):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(rows, cols, generator=g) * spread
    x = x * torch.exp2(torch.randint(-6, 7, (rows, 1), generator=g).float())
    return x.to(DT[dtype]).cuda()


def _check_quantized(b200, t, x64, tensor_scale=None):
    """t holds exactly the definition's bytes for x64, padding included."""
    code, byte, bad = X.quantize(x64, t.fmt, tensor_scale)
    got = X.element_codes(t.data.cpu().numpy(), t.fmt)
    good = ~np.repeat(bad, X.BLOCK[t.fmt], 1)
    np.testing.assert_array_equal(X.unsigned_zero(got, t.fmt)[good], X.unsigned_zero(code, t.fmt)[good])
    tiles = t.scales.cpu().numpy()
    want = X.scale_tiles(byte)
    assert tiles.shape == want.shape
    np.testing.assert_array_equal(tiles, want)


def _device_operand(b200, code, byte, fmt, cols, tensor_scale=None):
    data = torch.from_numpy(X.element_bytes(code, fmt)).cuda()
    scales = torch.from_numpy(X.scale_tiles(byte)).cuda()
    ts = None if tensor_scale is None else torch.tensor([tensor_scale], dtype=torch.float32, device="cuda")
    return b200.MxTensor(data, scales, fmt, code.shape[0], cols, ts)


def _ok(b200):
    rc, bits = b200.status()
    assert rc == 0, f"device status {bits:#x}"


# ------------------------------------------------------------------------ quantisation
SHAPES = [(1, 1), (1, 17), (3, 32), (5, 33), (31, 64), (127, 96), (128, 128), (129, 130), (257, 515), (40, 2049)]


@pytest.mark.parametrize("fmt", FMTS)
@pytest.mark.parametrize("dtype", ["f16", "bf16", "f32"])
@pytest.mark.parametrize("transpose", [False, True])
@pytest.mark.parametrize("rows,cols", SHAPES)
def test_quantize(b200, fmt, dtype, transpose, rows, cols):
    x = _input(rows * 7 + cols, cols if transpose else rows, rows if transpose else cols, dtype)
    ts = torch.tensor([0.37], device="cuda") if fmt == "nvfp4" else None
    t = b200.quantize_mx(x, fmt, transpose=transpose, tensor_scale=ts)
    assert t.shape == (rows, cols)
    x64 = _f64(x)
    _check_quantized(b200, t, x64.T if transpose else x64, None if ts is None else 0.37)


@pytest.mark.parametrize("transpose", [False, True])
@pytest.mark.parametrize("dtype", ["f16", "bf16", "f32"])
def test_quantize_finds_the_tensor_scale(b200, dtype, transpose):
    x = _input(3, 70, 301, dtype, 3.0)
    x[5, 7] = float("inf")
    x[6, 200] = float("nan")
    t = b200.quantize_mx(x, "nvfp4", transpose=transpose)
    x64 = _f64(x)
    amax = np.abs(x64[np.isfinite(x64)]).max()
    ts = X.found_scale(amax)
    assert float(t.tensor_scale) == float(ts)
    _check_quantized(b200, t, x64.T if transpose else x64, ts)
    # again into the same storage, with other data: the scale is found anew
    y = x * 0 + 2.0
    y[5, 7] = y[6, 200] = 2.0
    b200.quantize_mx(y, "nvfp4", transpose=transpose, out=t)
    ts = X.found_scale(2.0)
    assert float(t.tensor_scale) == float(ts)
    _check_quantized(b200, t, np.full(x64.T.shape if transpose else x64.shape, 2.0), ts)


@pytest.mark.parametrize("transpose", [False, True])
@pytest.mark.parametrize("dtype", ["f16", "bf16", "f32"])
@pytest.mark.parametrize("fmt", FMTS)
def test_quantize_large(b200, fmt, dtype, transpose):
    """Several segments per row and warp, several clusters behind the found scale; once as one
    matrix without gaps, once as a slice."""
    for x in (_input(9, 1300, 8200, dtype), _input(10, 1100, 2600, dtype)[:, 3:2500]):
        t = b200.quantize_mx(x, fmt, transpose=transpose)
        x64 = _f64(x)
        ts = X.found_scale(np.abs(x64).max()) if fmt == "nvfp4" else None
        if ts is not None:
            assert float(t.tensor_scale) == float(ts)
        _check_quantized(b200, t, x64.T if transpose else x64, ts)


def test_quantize_coarse_values_meet_scale_borders(b200):
    """Values of few bits with the tensor scale found: block maxima over the largest element
    are ratios of small integers, so max|u| / 6 falls on and next to e4m3 borders often."""
    rng = np.random.default_rng(12)
    for top in (37, 38, 40, 41, 43, 45, 56, 63):
        x64 = rng.integers(-top, top + 1, size=(301, 1003)) / 8.0
        x64[7, 9] = top / 8.0
        for dtype in ("f16", "bf16"):
            t = b200.quantize_mx(torch.from_numpy(x64).to(DT[dtype]).cuda(), "nvfp4")
            assert float(t.tensor_scale) == float(X.found_scale(top / 8.0))
            _check_quantized(b200, t, x64, X.found_scale(top / 8.0))


def test_quantize_zero_matrix(b200):
    for fmt in FMTS:
        t = b200.quantize_mx(torch.zeros(130, 70, device="cuda", dtype=torch.bfloat16), fmt)
        assert int(t.data.max()) == 0 and int(t.scales.max()) == 0
        if fmt == "nvfp4":
            assert float(t.tensor_scale) == 1.0


@pytest.mark.parametrize("fmt", FMTS)
def test_quantize_ties_and_borders(b200, fmt):
    """Every border between neighbouring elements, and its fp32 neighbours, under several block
    scales; block maxima at, just below and just above each power-of-two border."""
    table = X.E4M3 if fmt == "mxfp8" else X.E2M1
    mid = (table[1:] + table[:-1]) / 2
    rows = []
    for s in (1.0, 0.5, 4.0, 2.0 ** -20) if fmt != "nvfp4" else (1.0, 1.125, 13.0, 0.4375):
        base = np.float32(mid * s)
        for v in (base, np.nextafter(base, np.float32(0)), np.nextafter(base, np.float32(1e30))):
            for part in np.array_split(v, -(-len(v) // 15)):
                block = np.zeros(32, dtype=np.float32)
                block[:len(part)] = part
                if fmt == "nvfp4":
                    block[16:] = -block[:16]
                    block[15] = block[31] = np.float32(6.0 * s)
                else:
                    block[31] = np.float32(table[-1] * s)
                rows.append(block)
    top = 448.0 if fmt == "mxfp8" else 6.0
    for e in (-130, -126, -60, -3, 0, 9, 100):
        with np.errstate(over="ignore", under="ignore"):
            m = np.float32(top * 2.0 ** e)
        for v in (m, np.nextafter(m, np.float32(0)), np.nextafter(m, np.float32(1e30))):
            block = np.zeros(32, dtype=np.float32)
            block[3], block[20] = v, -v / 3
            rows.append(block)
    x = np.stack(rows)
    ts = torch.ones(1, device="cuda") if fmt == "nvfp4" else None
    for transpose in (False, True):
        xt = torch.from_numpy(np.ascontiguousarray(x.T if transpose else x)).cuda()
        t = b200.quantize_mx(xt, fmt, transpose=transpose, tensor_scale=ts)
        _check_quantized(b200, t, x.astype(np.float64), None if ts is None else 1.0)


@pytest.mark.parametrize("fmt", FMTS)
def test_quantize_nonfinite_blocks(b200, fmt):
    x = torch.randn(9, 160, device="cuda")
    x[2, 40] = float("inf")
    x[4, 159] = float("nan")
    x[7, 0] = -float("inf")
    ts = torch.ones(1, device="cuda") if fmt == "nvfp4" else None
    for transpose in (False, True):
        t = b200.quantize_mx(x.t().contiguous() if transpose else x, fmt, transpose=transpose, tensor_scale=ts)
        _check_quantized(b200, t, _f64(x), None if ts is None else 1.0)
        y = b200.dequantize_mx(t, out_dtype="f32")
        blk = X.BLOCK[fmt]
        nan = torch.zeros_like(x, dtype=torch.bool)
        for r, c in ((2, 40), (4, 159), (7, 0)):
            nan[r, c // blk * blk:(c // blk + 1) * blk] = True
        assert torch.equal(torch.isnan(y), nan)


@pytest.mark.parametrize("fmt", FMTS)
@pytest.mark.parametrize("transpose", [False, True])
def test_quantize_strided_and_misaligned_input(b200, fmt, transpose):
    buf = torch.randn(200, 333, device="cuda").to(torch.bfloat16)
    for x in (buf[3:150, 5:301], buf[:, :320], buf[1::2, 32:]):
        ts = torch.tensor([0.01], device="cuda") if fmt == "nvfp4" else None
        t = b200.quantize_mx(x, fmt, transpose=transpose, tensor_scale=ts)
        x64 = _f64(x)
        _check_quantized(b200, t, x64.T if transpose else x64, None if ts is None else 0.01)


def test_quantize_writes_nothing_beside_its_rows(b200):
    """Data rows with a pitch of their own: the bytes between the rows stay as they were."""
    row_bytes, scale_bytes = b200.mx_layout("mxfp4", 5, 100)
    buf = torch.full((7, row_bytes + 48), 0xAB, dtype=torch.uint8, device="cuda")
    scales = torch.full((scale_bytes + 32,), 0xCD, dtype=torch.uint8, device="cuda")
    t = b200.MxTensor(buf[1:6, 16:16 + row_bytes], scales[16:16 + scale_bytes], "mxfp4", 5, 100)
    x = torch.randn(5, 100, device="cuda")
    b200.quantize_mx(x, "mxfp4", out=t)
    code, byte, _ = X.quantize(_f64(x), "mxfp4")
    got = X.element_codes(t.data.cpu().numpy(), "mxfp4")
    np.testing.assert_array_equal(X.unsigned_zero(got, "mxfp4"), X.unsigned_zero(code, "mxfp4"))
    np.testing.assert_array_equal(t.scales.cpu().numpy(), X.scale_tiles(byte).reshape(-1))
    buf[1:6, 16:16 + row_bytes] = 0xAB
    scales[16:16 + scale_bytes] = 0xCD
    assert bool((buf == 0xAB).all()) and bool((scales == 0xCD).all())


# ---------------------------------------------------------------------- dequantisation
@pytest.mark.parametrize("fmt", FMTS)
@pytest.mark.parametrize("dtype", ["f16", "bf16", "f32"])
@pytest.mark.parametrize("rows,cols", [(1, 1), (3, 33), (130, 512), (77, 1001)])
def test_dequantize(b200, fmt, dtype, rows, cols):
    rng = np.random.default_rng(rows + cols)
    code, byte = X.random_operand(rng, rows, cols, fmt)
    ts = np.float32(0.3) if fmt == "nvfp4" else None
    t = _device_operand(b200, code, byte, fmt, cols, ts)
    y = b200.dequantize_mx(t, out_dtype=dtype)
    ref = X.values(code, byte, fmt, cols, ts)
    if ts is None:  # few significant bits: exact in fp32, one rounding after
        want = torch.from_numpy(ref.astype(np.float32)).to(DT[dtype]).double().numpy()
        np.testing.assert_array_equal(_f64(y), want)
    else:
        tol = (HALF_STEP[dtype] + 2.0 ** -24) * np.abs(ref) + (2.0 ** -25 if dtype == "f16" else 0)
        assert (np.abs(_f64(y) - ref) <= tol).all()
    # a strided output: what lies beside its columns stays
    buf = torch.full((rows, cols + 3), 7.0, dtype=DT[dtype], device="cuda")
    b200.dequantize_mx(t, buf[:, 1:cols + 1])
    assert torch.equal(buf[:, 1:cols + 1], y) and bool((buf[:, 0] == 7).all()) and bool((buf[:, cols + 1:] == 7).all())


def test_dequantize_every_code_and_scale(b200):
    for fmt in FMTS:
        n = 256 if fmt == "mxfp8" else 16
        code = np.tile(np.arange(n, dtype=np.uint8), (256, max(1, 32 // n)))
        byte = np.repeat(np.arange(256, dtype=np.uint8)[:, None], code.shape[1] // X.BLOCK[fmt], 1)
        if fmt == "nvfp4":
            byte &= 127
        t = _device_operand(b200, code, byte, fmt, code.shape[1])
        ref = X.values(code, byte, fmt, code.shape[1])
        with np.errstate(over="ignore"):
            np.testing.assert_array_equal(_f64(b200.dequantize_mx(t, out_dtype="f32")), ref.astype(np.float32))


# ---------------------------------------------------------------------------- products
PRODUCTS = [
    # M, N, K
    (1, 1, 1), (1, 128, 32), (1, 129, 33), (2, 100, 64), (16, 256, 96), (17, 300, 160), (33, 127, 256),
    (64, 512, 288), (65, 200, 512), (100, 384, 544), (128, 128, 1024), (129, 130, 130), (200, 640, 2048),
    (256, 256, 512), (257, 511, 320), (300, 1000, 777), (513, 260, 4096), (1, 2048, 8192), (5, 1000, 5000),
]


@pytest.mark.parametrize("fmt", FMTS)
@pytest.mark.parametrize("M,N,K", PRODUCTS)
def test_gemm_exact_on_integers(b200, fmt, M, N, K):
    rng = np.random.default_rng(M * 3 + N * 5 + K)
    ca, ba = X.random_operand(rng, M, K, fmt, exact=True)
    cb, bb = X.random_operand(rng, N, K, fmt, exact=True)
    a, b = _device_operand(b200, ca, ba, fmt, K), _device_operand(b200, cb, bb, fmt, K)
    c = b200.gemm_mx(a, b, out_dtype="f32")
    _ok(b200)
    ref = X.values(ca, ba, fmt, K) @ X.values(cb, bb, fmt, K).T
    np.testing.assert_array_equal(_f64(c), ref)


@pytest.mark.parametrize("fmt", FMTS)
@pytest.mark.parametrize("M,N,K", [(4096, 4096, 1056), (3700, 4000, 160), (8192, 8100, 96), (5000, 5001, 96)])
def test_gemm_exact_over_several_waves(b200, fmt, M, N, K):
    """Tiles in several waves, the last one ragged and its last columns partly or wholly behind
    the matrix; outputs of 16 and 32 bits."""
    rng = np.random.default_rng(M + N + K)
    ca, ba = X.random_operand(rng, M, K, fmt, exact=True)
    cb, bb = X.random_operand(rng, N, K, fmt, exact=True)
    a, b = _device_operand(b200, ca, ba, fmt, K), _device_operand(b200, cb, bb, fmt, K)
    ref = torch.from_numpy(X.values(ca, ba, fmt, K)).cuda() @ torch.from_numpy(X.values(cb, bb, fmt, K)).cuda().T
    for dtype in ("f32", "bf16"):
        c = b200.gemm_mx(a, b, out_dtype=dtype)
        _ok(b200)
        assert torch.equal(c, ref.float().to(DT[dtype]))


@pytest.mark.parametrize("fmt", FMTS)
@pytest.mark.parametrize("dtype", ["f16", "bf16", "f32"])
@pytest.mark.parametrize("M,N,K", [(1, 512, 4096), (24, 1000, 1024), (150, 333, 700), (384, 768, 1536)])
def test_gemm_real_data(b200, fmt, dtype, M, N, K):
    rng = np.random.default_rng(M + N + K)
    ca, ba = X.random_operand(rng, M, K, fmt)
    cb, bb = X.random_operand(rng, N, K, fmt)
    if fmt == "mxfp8":
        bb = (bb - 10).astype(np.uint8)  # keep f16 outputs in range
    ta, tb = (np.float32(0.011), np.float32(0.73)) if fmt == "nvfp4" else (None, None)
    a, b = _device_operand(b200, ca, ba, fmt, K, ta), _device_operand(b200, cb, bb, fmt, K, tb)
    va, vb = X.values(ca, ba, fmt, K, ta), X.values(cb, bb, fmt, K, tb)
    c = b200.gemm_mx(a, b, out_dtype=dtype)
    _ok(b200)
    ref, mag = va @ vb.T, np.abs(va) @ np.abs(vb).T
    # the two tensor scales' product and its product with the sum round once each
    tol = (K / 32 + 4) * 2.0 ** -23 * mag + HALF_STEP[dtype] * np.abs(ref) + (2.0 ** -25 if dtype == "f16" else 0)
    err = np.abs(_f64(c) - ref)
    assert (err <= tol).all(), float((err / tol).max())
    again = b200.gemm_mx(a, b, out_dtype=dtype)
    assert torch.equal(c, again)


@pytest.mark.parametrize("fmt", FMTS)
@pytest.mark.parametrize("M", [3, 140, 300])
@pytest.mark.parametrize("N,pitch,first", [(261, 268, 3), (262, 272, 2), (260, 264, 4), (248, 264, 8), (250, 272, 16),
                                           (255, 257, 0)])
def test_gemm_strided_output(b200, fmt, M, N, pitch, first):
    """A column slice of a wider matrix, at every alignment of its rows: only its columns are
    written."""
    rng = np.random.default_rng(M + N)
    K = 416
    ca, ba = X.random_operand(rng, M, K, fmt, exact=True)
    cb, bb = X.random_operand(rng, N, K, fmt, exact=True)
    a, b = _device_operand(b200, ca, ba, fmt, K), _device_operand(b200, cb, bb, fmt, K)
    ref = torch.from_numpy(X.values(ca, ba, fmt, K) @ X.values(cb, bb, fmt, K).T).float()
    for dtype in ("f32", "f16", "bf16"):
        buf = torch.full((M, pitch), 5.0, dtype=DT[dtype], device="cuda")
        b200.gemm_mx(a, b, buf[:, first:first + N])
        assert torch.equal(buf[:, first:first + N], ref.to(DT[dtype]).cuda())
        assert bool((buf[:, :first] == 5).all()) and bool((buf[:, first + N:] == 5).all())


@pytest.mark.parametrize("fmt", FMTS)
@pytest.mark.parametrize("M", [2, 200])
def test_gemm_nan_scale_stays_in_its_row_and_column(b200, fmt, M):
    rng = np.random.default_rng(5)
    N, K = 150, 512
    ca, ba = X.random_operand(rng, M, K, fmt, exact=True)
    cb, bb = X.random_operand(rng, N, K, fmt, exact=True)
    nan = 0x7F if fmt == "nvfp4" else 0xFF
    ba[1, 3] = nan
    bb[147, 0] = nan
    c = b200.gemm_mx(_device_operand(b200, ca, ba, fmt, K), _device_operand(b200, cb, bb, fmt, K), out_dtype="f32")
    want = np.zeros((M, N), dtype=bool)
    want[1, :] = True
    want[:, 147] = True
    np.testing.assert_array_equal(np.isnan(_f64(c)), want)


def test_gemm_empty_sum_and_empty_sides(b200):
    for fmt in FMTS:
        a, b = b200.MxTensor.empty(5, 0, fmt), b200.MxTensor.empty(9, 0, fmt)
        c = torch.full((5, 9), 3.0, device="cuda")
        b200.gemm_mx(a, b, c)
        assert bool((c == 0).all())
        assert b200.gemm_mx(b200.MxTensor.empty(0, 64, fmt), b200.MxTensor.empty(9, 64, fmt)).shape == (0, 9)
        q = b200.quantize_mx(torch.empty(0, 64, device="cuda"), fmt)
        assert q.shape == (0, 64)
        assert b200.dequantize_mx(q).shape == (0, 64)


# -------------------------------------------------------------------------------- norm
def _norm_ref(x, w, res, eps):
    h = x if res is None else x + res
    return h / np.sqrt((h * h).mean(1, keepdims=True) + eps) * w, h


DELTA = 2.0 ** -17


def _check_norm(t, y, tensor_scale=None):
    """Scale bytes and codes are those of values within DELTA of y."""
    fmt = t.fmt
    rows, n = y.shape[0], -(-y.shape[1] // 32) * 32 // X.BLOCK[fmt]
    tiles = t.scales.cpu().numpy()
    byte = X.scale_bytes(tiles, rows, n)
    np.testing.assert_array_equal(X.scale_tiles(byte), tiles)  # padding bytes are zero
    u = y if tensor_scale is None else y * np.float64(np.float32(1.0) / np.float32(tensor_scale))
    lo = X.quantize(u * (1 - DELTA), fmt)[1]
    hi = X.quantize(u * (1 + DELTA), fmt)[1]
    assert ((byte == lo) | (byte == hi)).all()
    s = np.repeat(X.scale_values(byte, fmt), X.BLOCK[fmt], 1)
    table, sign = (X.E4M3, 128) if fmt == "mxfp8" else (X.E2M1, 8)
    q = np.where(s > 0, X.pad_cols(u) / np.where(s > 0, s, 1), 0.0)
    code = X.element_codes(t.data.cpu().numpy(), fmt)
    mag = (code & (sign - 1)).astype(int)
    ok = (mag == X.nearest(q * (1 - DELTA), table)) | (mag == X.nearest(q * (1 + DELTA), table))
    assert ok.all(), int((~ok).sum())
    assert (((code & sign) != 0) == (q < 0))[mag > 0].all()


@pytest.mark.parametrize("fmt", FMTS)
@pytest.mark.parametrize("dtype", ["f16", "bf16", "f32"])
@pytest.mark.parametrize("rows,cols,residual", [
    (1, 1, True), (1, 4096, True), (2, 33, False), (7, 512, True), (130, 100, True), (33, 1000, False),
    (5, 2048, True), (3, 5000, True), (2, 8192, False), (2, 16384, True), (2, 20001, True), (1, 32768, True)])
def test_rms_norm(b200, fmt, dtype, rows, cols, residual):
    x, r = _input(rows + cols, rows, cols, dtype), _input(rows + cols + 1, rows, cols, dtype)
    w = (1 + 0.2 * torch.randn(cols, generator=torch.Generator().manual_seed(cols))).to(DT[dtype]).cuda()
    res = r if residual else None
    t, h = b200.rms_norm_mx(x, w, res, eps=1e-5, fmt=fmt)
    y, h64 = _norm_ref(_f64(x), _f64(w), _f64(r) if residual else None, 1e-5)
    _check_norm(t, y)
    if residual:  # x + residual rounds to fp32, then to the type
        tol = (HALF_STEP[dtype] + 2.0 ** -24) * np.abs(h64) + (2.0 ** -25 if dtype == "f16" else 0)
        assert (np.abs(_f64(h) - h64) <= tol).all()
    else:
        assert h is None


@pytest.mark.parametrize("fmt", FMTS)
@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("cols,residual", [(2056, True), (4096, False), (4096, True), (7000, True), (12000, False)])
def test_rms_norm_many_rows(b200, fmt, dtype, cols, residual):
    """Enough rows for the streaming kernel (with a ragged last band), h in place of the
    residual; x has a row pitch of its own."""
    rows = 601
    x = _input(cols, rows, cols + 8, dtype)[:, :cols]
    r = _input(cols + 1, rows, cols, dtype) if residual else None
    if cols == 7000:  # h at an odd pitch
        h1 = torch.full((rows, cols + 3), 4.0, dtype=DT[dtype], device="cuda")
        b200.rms_norm_mx(x, torch.ones(cols, device="cuda"), r, fmt=fmt, residual_out=h1[:, 1:cols + 1])
        assert torch.equal(h1[:, 1:cols + 1], x + r)
        assert bool((h1[:, 0] == 4).all()) and bool((h1[:, cols + 1:] == 4).all())
    w = (1 + 0.2 * torch.randn(cols, generator=torch.Generator().manual_seed(cols))).to(DT[dtype]).cuda()
    y, h64 = _norm_ref(_f64(x), _f64(w), _f64(r) if residual else None, 1e-6)
    t, h = b200.rms_norm_mx(x, w, r, fmt=fmt, residual_out=r)
    _ok(b200)
    _check_norm(t, y)
    if residual:
        assert h is r
        assert (np.abs(_f64(h) - h64) <= (HALF_STEP[dtype] + 2.0 ** -24) * np.abs(h64)).all()


@pytest.mark.parametrize("fmt", FMTS)
def test_rms_norm_in_place_strided_and_fp32_weight(b200, fmt):
    buf = torch.randn(40, 700, device="cuda").to(torch.bfloat16)
    x = buf[2:20, 3:600]
    res = torch.randn(18, 597, device="cuda").to(torch.bfloat16)
    w = 1 + 0.1 * torch.randn(597, device="cuda")
    before = buf.clone()
    y, h64 = _norm_ref(_f64(x), _f64(w), _f64(res), 1e-6)
    t0, h0 = b200.rms_norm_mx(x, w, res, fmt=fmt)
    assert torch.equal(buf, before)
    ts = torch.tensor([0.02], device="cuda") if fmt == "nvfp4" else None
    t1, h1 = b200.rms_norm_mx(x, w, res, fmt=fmt, residual_out=res, tensor_scale=ts)
    assert h1 is res and torch.equal(h0, h1)
    _check_norm(t0, y)
    _check_norm(t1, y, None if ts is None else 0.02)


def test_rms_norm_zero_and_nan_rows(b200):
    x = torch.randn(4, 300, device="cuda")
    x[1] = 0
    x[2, 299] = float("nan")
    w = torch.ones(300, device="cuda")
    for fmt in FMTS:
        t, _ = b200.rms_norm_mx(x, w, fmt=fmt)
        y = b200.dequantize_mx(t, out_dtype="f32")
        assert bool((y[1] == 0).all()) and bool(torch.isnan(y[2]).all())
        assert not bool(torch.isnan(y[[0, 1, 3]]).any())


@pytest.mark.parametrize("fmt", FMTS)
@pytest.mark.parametrize("rows,cols", [(3, 300), (3, 900), (40, 2000), (601, 4096), (601, 4200)])
@pytest.mark.parametrize("ex,ew", [(60, 80), (-50, -85), (110, 0), (-120, 0)])
def test_rms_norm_far_magnitudes(b200, fmt, rows, cols, ex, ew):
    """h * w, or the squares, leave fp32 (or most of its precision) where the normalised value
    does not."""
    if fmt == "nvfp4" and ew:  # with the tensor scale that such values need
        ex, ew = (40, 82) if ex > 0 else (-30, -86)
    x = _input(cols, rows, cols, "f32") * 2.0 ** ex
    x = x.to(torch.bfloat16)
    w = (1 + 0.2 * torch.randn(cols, generator=torch.Generator().manual_seed(cols))).cuda() * 2.0 ** ew
    ts = torch.tensor([2.0 ** ew], device="cuda") if fmt == "nvfp4" else None
    t, _ = b200.rms_norm_mx(x, w, eps=0.0, fmt=fmt, tensor_scale=ts)
    y, _ = _norm_ref(_f64(x), _f64(w), None, 0.0)
    _check_norm(t, y, None if ts is None else 2.0 ** ew)


# ------------------------------------------------------------------- the run of them all
@pytest.mark.parametrize("fmt", FMTS)
@pytest.mark.parametrize("M", [1, 20, 260])
def test_norm_into_projection(b200, fmt, M):
    """residual add + norm -> product with quantised weights, as a decoder's projection. The
    product is checked on the values that the norm's own output stands for."""
    N, K = 520, 1056
    x, r = _input(1, M, K, "bf16"), _input(2, M, K, "bf16")
    w = torch.ones(K, device="cuda", dtype=torch.bfloat16)
    wq = b200.quantize_mx(_input(3, N, K, "bf16", K ** -0.5), fmt)
    t, _ = b200.rms_norm_mx(x, w, r, fmt=fmt)
    c = b200.gemm_mx(t, wq)
    va, vb = _f64(b200.dequantize_mx(t, out_dtype="f32")), _f64(b200.dequantize_mx(wq, out_dtype="f32"))
    y, _ = _norm_ref(_f64(x), _f64(w), _f64(r), 1e-6)
    _check_norm(t, y)
    ref, mag = va @ vb.T, np.abs(va) @ np.abs(vb).T
    # vb in fp32 carries one rounding of element * tensor scale
    tol = (K / 32 + 6) * 2.0 ** -23 * mag + 2.0 ** -8 * np.abs(ref)
    assert (np.abs(_f64(c) - ref) <= tol).all()


@pytest.mark.parametrize("fmt", FMTS)
def test_linear_training_step(b200, fmt):
    """Y = X W^T, dX = dY W, dW = dY^T X on operands quantised along each product's summed
    axis, against the same products of the 64-bit quantised values; and dX, dW against
    differences of the loss sum(Y0 * dY) of the unquantised layer, as far as 64-bit
    differences of the quantised operands' products say: the loss is bilinear, so its
    difference quotient along one entry is that entry's gradient."""
    M, N, K = 200, 330, 290
    x, w, dy = _input(4, M, K, "bf16"), _input(5, N, K, "bf16", 0.1), _input(6, M, N, "bf16", 0.01)

    def pair(p, q, tp, tq):
        a, b = b200.quantize_mx(p, fmt, transpose=tp), b200.quantize_mx(q, fmt, transpose=tq)
        c = b200.gemm_mx(a, b, out_dtype="f32")
        va, vb = _f64(b200.dequantize_mx(a, out_dtype="f32")), _f64(b200.dequantize_mx(b, out_dtype="f32"))
        tol = (a.cols / 32 + 6) * 2.0 ** -23 * (np.abs(va) @ np.abs(vb).T)
        assert (np.abs(_f64(c) - va @ vb.T) <= tol).all()
        return c, va, vb

    y, _, _ = pair(x, w, False, False)
    dx, vdy, vwt = pair(dy, w, False, True)
    dw, vdyt, vxt = pair(dy, x, True, True)
    assert y.shape == (M, N) and dx.shape == (M, K) and dw.shape == (N, K)
    rng = np.random.default_rng(0)
    x64, w64 = _f64(x), _f64(w)
    for _ in range(5):
        m, n, k = rng.integers(M), rng.integers(N), rng.integers(K)
        step = 0.5

        def loss_x(v):  # sum(dY * (X W^T)) with X[m, k] = v
            row = x64[m].copy()
            row[k] = v
            return float(vdy[m] @ (vwt.T @ row))

        def loss_w(v):
            col = w64[n].copy()
            col[k] = v
            return float(vdyt[n] @ (vxt.T @ col))

        gx = (loss_x(x64[m, k] + step) - loss_x(x64[m, k] - step)) / (2 * step)
        gw = (loss_w(w64[n, k] + step) - loss_w(w64[n, k] - step)) / (2 * step)
        tx = (N / 32 + 6) * 2.0 ** -23 * float(np.abs(vdy[m]) @ np.abs(vwt[k])) + 1e-9 * abs(loss_x(x64[m, k]))
        tw = (M / 32 + 6) * 2.0 ** -23 * float(np.abs(vdyt[n]) @ np.abs(vxt[k])) + 1e-9 * abs(loss_w(w64[n, k]))
        assert abs(float(dx[m, k]) - gx) <= tx and abs(float(dw[n, k]) - gw) <= tw


# ------------------------------------------------------------- streams, graphs, big sizes
def test_gemm_of_a_matrix_with_itself(b200):
    rng = np.random.default_rng(8)
    for fmt in FMTS:
        for M in (20, 200):
            code, byte = X.random_operand(rng, M, 300, fmt, exact=True)
            a = _device_operand(b200, code, byte, fmt, 300)
            v = X.values(code, byte, fmt, 300)
            np.testing.assert_array_equal(_f64(b200.gemm_mx(a, a, out_dtype="f32")), v @ v.T)


@pytest.mark.parametrize("raw", [False, True])
def test_other_stream_than_the_current_one(b200, raw):
    """Inputs made on the side stream behind a long queue; nothing but the stream argument
    orders the calls after them, and what they allocate belongs to that stream."""
    side = torch.cuda.Stream()
    handle = side.cuda_stream if raw else side
    big = torch.randn(4096, 4096, device="cuda")
    x, w = torch.zeros(150, 512, device="cuda"), torch.ones(512, device="cuda")
    r = torch.zeros_like(x)
    torch.cuda.synchronize()
    with torch.cuda.stream(side):
        for _ in range(20):
            big = big @ big * 1e-3
        x.normal_()
        r.normal_()
    q = b200.quantize_mx(x, "nvfp4", stream=handle)
    y = b200.dequantize_mx(q, out_dtype="f32", stream=handle)
    n, h = b200.rms_norm_mx(x, w, r, fmt="nvfp4", stream=handle)
    c = b200.gemm_mx(n, q, out_dtype="f32", stream=handle)
    side.synchronize()
    ts = X.found_scale(float(x.abs().max()))
    _check_quantized(b200, q, _f64(x), ts)
    ref, h64 = _norm_ref(_f64(x), _f64(w), _f64(r), 1e-6)
    _check_norm(n, ref)
    assert (np.abs(_f64(h) - h64) <= 2.0 ** -23 * np.abs(h64)).all()
    va, vb = _f64(b200.dequantize_mx(n, out_dtype="f32")), _f64(y)
    tol = (512 / 32 + 6) * 2.0 ** -23 * (np.abs(va) @ np.abs(vb).T)
    assert (np.abs(_f64(c) - va @ vb.T) <= tol).all()


@pytest.mark.parametrize("M", [1, 40, 300])
def test_captured_and_replayed(b200, M):
    """Norm, quantisation with a found scale and products in a graph, replayed on new inputs;
    a second graph of the same calls interleaved with it; both give the eager results."""
    N, K = 390, 1000
    x = torch.randn(M, K, device="cuda").to(torch.bfloat16)
    r = torch.randn(M, K, device="cuda").to(torch.bfloat16)
    w = torch.ones(K, device="cuda", dtype=torch.bfloat16)
    wt = torch.randn(N, K, device="cuda").to(torch.bfloat16)

    def calls():
        n, h = b200.rms_norm_mx(x, w, r, fmt="nvfp4")
        q = b200.quantize_mx(wt, "nvfp4")
        t = b200.quantize_mx(h, "mxfp8", transpose=True)
        return b200.gemm_mx(n, q), b200.gemm_mx(t, t, out_dtype="f32"), b200.dequantize_mx(q), h

    calls()
    side = torch.cuda.Stream()
    graphs = []
    for _ in range(2):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=side):
            out = calls()
        graphs.append((g, out))
    for k in range(3):
        for t in (x, r, wt):
            t.copy_(torch.randn_like(t) * (k + 1))
        for g, out in graphs:
            for o in out:
                o.fill_(float("nan"))
        for g, _ in graphs + graphs:
            g.replay()
        want = calls()
        torch.cuda.synchronize()
        for _, out in graphs:
            for a, b in zip(out, want):
                assert torch.equal(a, b)
    _ok(b200)


def test_two_streams_at_once(b200):
    """Split-K and pair products, quantisation and norm on two streams without ordering."""
    rng = np.random.default_rng(11)
    jobs = []
    for fmt, M, N, K in (("nvfp4", 3, 1000, 8192), ("mxfp8", 600, 900, 4096), ("mxfp4", 100, 512, 8192)):
        ca, ba = X.random_operand(rng, M, K, fmt, exact=True)
        cb, bb = X.random_operand(rng, N, K, fmt, exact=True)
        ref = X.values(ca, ba, fmt, K) @ X.values(cb, bb, fmt, K).T
        jobs.append((_device_operand(b200, ca, ba, fmt, K), _device_operand(b200, cb, bb, fmt, K), ref))
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    outs = []
    for rep in range(20):
        for i, (a, b, ref) in enumerate(jobs):
            outs.append((b200.gemm_mx(a, b, out_dtype="f32", stream=streams[(rep + i) % 2]), ref))
    torch.cuda.synchronize()
    _ok(b200)
    for c, ref in outs:
        np.testing.assert_array_equal(_f64(c), ref)


def test_more_elements_than_32_bits(b200):
    """4.3e9 elements: every offset (x, elements, scales, C) passes 2^32; the last rows and
    columns are checked."""
    rows, cols = 70016, 62016
    x = torch.empty(rows, cols, dtype=torch.bfloat16, device="cuda")
    x[:] = torch.randn(cols, device="cuda").to(torch.bfloat16)
    x[-200:].normal_()
    t = b200.quantize_mx(x, "mxfp8")
    some = _f64(x[-200:])
    code, byte, _ = X.quantize(some, "mxfp8")
    np.testing.assert_array_equal(X.unsigned_zero(t.data[-200:].cpu().numpy(), "mxfp8"), X.unsigned_zero(code, "mxfp8"))
    got = X.scale_bytes(t.scales[-1:].cpu().numpy(), 128, cols // 32)  # 70016 rows are 547 whole bands
    np.testing.assert_array_equal(got, byte[-128:])
    y = b200.dequantize_mx(t)
    assert torch.equal(y[-200:].float().cpu(), torch.from_numpy(X.values(code, byte, "mxfp8", cols).astype(np.float32)))
    del y
    u = b200.quantize_mx(x, "mxfp8", transpose=True)  # cols x rows
    tail = _f64(x[:, -40:]).T
    code_t, byte_t, _ = X.quantize(tail, "mxfp8")
    np.testing.assert_array_equal(X.unsigned_zero(u.data[-40:].cpu().numpy(), "mxfp8"),
                                  X.unsigned_zero(code_t, "mxfp8"))
    del u
    w = torch.ones(1, device="cuda").expand(20000).contiguous()
    n, h = b200.rms_norm_mx(x[:, :20000], w, x[:, 40000:60000], fmt="mxfp8")
    assert torch.equal(h[-200:], x[-200:, :20000] + x[-200:, 40000:60000])
    ref, _ = _norm_ref(_f64(x[-8:, :20000]), np.ones(20000), _f64(x[-8:, 40000:60000]), 1e-6)
    v = _f64(b200.dequantize_mx(n)[-8:])
    assert (np.abs(v - ref) <= 2.0 ** -4 * np.abs(ref) * 1.01 + 2.0 ** -10 * 0.02).all()
    del n, h
    b = b200.quantize_mx(x[-300:], "mxfp8")
    c = b200.gemm_mx(t, b, out_dtype="f32")  # A beyond 2^32 bytes
    va, vb = X.values(code, byte, "mxfp8", cols), _f64(b200.dequantize_mx(b, out_dtype="f32"))
    tol = (cols / 32 + 4) * 2.0 ** -23 * (np.abs(va) @ np.abs(vb).T)
    assert (np.abs(_f64(c[-200:]) - va @ vb.T) <= tol).all()
    del t, b, c, x
    a, b = torch.randn(rows, 64, device="cuda"), torch.randn(cols, 64, device="cuda")
    qa, qb = b200.quantize_mx(a, "mxfp8"), b200.quantize_mx(b, "mxfp8")
    c = b200.gemm_mx(qa, qb)  # C beyond 2^32 elements
    va, vb = _f64(b200.dequantize_mx(qa, out_dtype="f32")), _f64(b200.dequantize_mx(qb, out_dtype="f32"))
    ref = va[-100:] @ vb[-100:].T
    tol = 6 * 2.0 ** -23 * (np.abs(va[-100:]) @ np.abs(vb[-100:]).T) + 2.0 ** -8 * np.abs(ref)
    assert (np.abs(_f64(c[-100:, -100:]) - ref) <= tol).all()
    _ok(b200)
