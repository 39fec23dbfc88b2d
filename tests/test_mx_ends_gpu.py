"""GPU tests of the microscaled operators at the ends of what they take, against plain 64-bit
forms (mx_check.py).

Tolerances
- a found tensor scale is one fp32 product, so it is compared for equality.
- products of integer data with far tensor scales: the sum is exact, the scales' product and its
  product with the sum round once each (2^-24), a result below the normal numbers once more
  (2^-150); bf16 adds its half step, 2^-8, or 2^-134 below the normal numbers.
- the norm: codes of a value within 2^-17 of the exact one (test_mx_gpu.py); the detour of a far
  factor adds two roundings (2^-24 each), for which the 2^-17 has room.
"""
from __future__ import annotations

import numpy as np
import pytest

import mx_check as X
from test_mx_gpu import _check_norm, _f64, _input, _norm_ref

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module", autouse=True)
def _cuda():
    if not torch.cuda.is_available():
        pytest.skip("no CUDA device")
    yield
    torch.cuda.synchronize()


def _ok(b200):
    rc, bits = b200.status()
    assert rc == 0, hex(bits)


@pytest.mark.parametrize("n", [4096, 8 * 8192 - 512, 8 * 8192, 8 * 8192 + 512, 9 * 65536 + 8192, 600 * 8192 + 32])
@pytest.mark.parametrize("dtype", ["bf16", "f32"])
def test_found_scale_sees_every_part(b200, dtype, n):
    """The largest magnitude in turn in each part of the matrix, so that each CTA of the clusters
    that look for it holds it once, those of a last cluster that is partly without work too."""
    dt = {"bf16": torch.bfloat16, "f32": torch.float32}[dtype]
    x = torch.full((1, n), 0.25, dtype=dt, device="cuda")
    places = sorted({*np.linspace(0, n - 1, 40).astype(int).tolist(), *range(0, n, max(1, n // 24))})
    found = []
    for k, at in enumerate(places):
        x[0, at] = -(2 + k)
        found.append((b200.quantize_mx(x, "nvfp4").tensor_scale, 2 + k))
        x[0, at] = 0.25
    torch.cuda.synchronize()
    _ok(b200)
    for ts, top in found:
        assert float(ts) == float(X.found_scale(top))


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("rows,cols,pitch,first", [(1, 1, 9, 3), (5, 7, 9, 1), (70, 33, 47, 5), (131, 517, 523, 3),
                                                   (200, 1023, 1025, 1)])
def test_column_slices_are_as_their_copies(b200, dtype, rows, cols, pitch, first):
    """What lies between the rows of a slice (NaN here) has no part in any result, and a whole
    matrix gives the same bytes as its slice."""
    dt = {"bf16": torch.bfloat16, "f32": torch.float32}[dtype]
    g = torch.Generator().manual_seed(rows + cols)
    slices = []
    for _ in range(2):
        buf = torch.full((rows, pitch), float("nan"), dtype=dt, device="cuda")
        buf[:, first:first + cols] = torch.randn(rows, cols, generator=g).to(dt).cuda()
        slices.append(buf[:, first:first + cols])
    x, r = slices
    w = torch.full((cols + 5,), float("nan"), dtype=dt, device="cuda")
    w[5:] = (1 + 0.1 * torch.randn(cols, generator=g)).to(dt).cuda()
    w = w[5:]
    for fmt in ("mxfp8", "mxfp4", "nvfp4"):
        for transpose in (False, True):
            a = b200.quantize_mx(x, fmt, transpose=transpose)
            b = b200.quantize_mx(x.contiguous(), fmt, transpose=transpose)
            assert torch.equal(a.data, b.data) and torch.equal(a.scales, b.scales)
            if fmt == "nvfp4":
                assert float(a.tensor_scale) == float(b.tensor_scale) == float(X.found_scale(float(x.abs().max())))
        a, h = b200.rms_norm_mx(x, w, r, fmt=fmt)
        b, k = b200.rms_norm_mx(x.contiguous(), w.clone(), r.contiguous(), fmt=fmt)
        assert torch.equal(a.data, b.data) and torch.equal(a.scales, b.scales) and torch.equal(h, k)
    _ok(b200)


@pytest.mark.parametrize("rows,cols", [(300, 597), (70, 5743), (20, 20001)])
@pytest.mark.parametrize("dtype", ["bf16", "f32"])
def test_norm_in_place_at_odd_pitches(b200, dtype, rows, cols):
    """h written over x or over the residual, at pitches where a thread reads whole chunks around
    its elements: the same bytes as into a matrix of its own."""
    dt = {"bf16": torch.bfloat16, "f32": torch.float32}[dtype]
    g = torch.Generator().manual_seed(cols)
    x, r = (torch.randn(rows, cols + 2, generator=g).to(dt).cuda()[:, 1:cols + 1] for _ in range(2))
    w = (1 + 0.1 * torch.randn(cols, generator=g)).to(dt).cuda()
    want, h = b200.rms_norm_mx(x, w, r)
    assert torch.equal(h, x + r)
    for rep in range(5):
        for over_x in (True, False):
            bx, br = (torch.empty(rows, cols + 2, dtype=dt, device="cuda") for _ in range(2))
            a, b = bx[:, 1:cols + 1].copy_(x), br[:, 1:cols + 1].copy_(r)
            t, k = b200.rms_norm_mx(a, w, b, residual_out=a if over_x else b)
            assert torch.equal(k, h) and torch.equal(t.data, want.data) and torch.equal(t.scales, want.scales)
    _ok(b200)


def _operand(b200, code, byte, fmt, cols, ts):
    s = torch.tensor([ts], dtype=torch.float32, device="cuda")
    return b200.MxTensor(torch.from_numpy(X.element_bytes(code, fmt)).cuda(),
                         torch.from_numpy(X.scale_tiles(byte)).cuda(), fmt, code.shape[0], cols, s)


@pytest.mark.parametrize("M", [3, 40, 300])
@pytest.mark.parametrize("small,ta,tb", [
    (False, 1.3 * 2.0 ** -100, 1.7 * 2.0 ** -40),  # the scales' product is subnormal, results are not
    (False, 1.3 * 2.0 ** -90, 1.7 * 2.0 ** -75),   # it rounds to zero, results are subnormal or 0
    (False, 2.0 ** -126, 2.0 ** -126),
    (True, 1.3 * 2.0 ** 67, 1.7 * 2.0 ** 66),      # it overflows, results do not
    (False, 1.3 * 2.0 ** 67, 1.7 * 2.0 ** 66),     # both do, but for sums of zero
    (False, 1.9 * 2.0 ** 127, 1.9 * 2.0 ** 127),
    (False, 1.9 * 2.0 ** 127, 1.5 * 2.0 ** -126),
])
def test_product_with_far_tensor_scales(b200, M, small, ta, tb):
    rng = np.random.default_rng(M)
    N, K = 390, 352
    (ca, ba), (cb, bb) = (X.random_operand(rng, n, K, "nvfp4", exact=True) for n in (M, N))
    if small:  # every block scale 2^-9
        ba[:], bb[:] = 1, 1
    ca[1], cb[7] = 0, 0  # sums of zero
    a, b = _operand(b200, ca, ba, "nvfp4", K, ta), _operand(b200, cb, bb, "nvfp4", K, tb)
    ref = X.values(ca, ba, "nvfp4", K) @ X.values(cb, bb, "nvfp4", K).T
    ref = ref * np.float64(np.float32(ta)) * np.float64(np.float32(tb))
    for dtype, half, low in ((torch.float32, 0.0, 0.0), (torch.bfloat16, 2.0 ** -8, 2.0 ** -134)):
        c = b200.gemm_mx(a, b, out_dtype="f32" if dtype is torch.float32 else "bf16").double().cpu().numpy()
        top = float(torch.finfo(dtype).max)
        tol = (half + 2.02 * 2.0 ** -24) * np.abs(ref) + 2.0 ** -150 + low
        assert not np.isnan(c).any() and bool((c[1] == 0).all()) and bool((c[:, 7] == 0).all())
        big = np.abs(ref) > top * (1 + 2.0 ** -7)  # certain to round beyond the type
        assert (np.abs(c[big]) == np.inf).all() and (np.sign(c[big]) == np.sign(ref[big])).all()
        fits = np.abs(ref) < top * (1 - 2.0 ** -7)
        assert (np.abs(c - ref)[fits] <= tol[fits]).all()
    _ok(b200)


@pytest.mark.parametrize("rows,cols", [(3, 300), (3, 900), (40, 2000), (601, 4096), (601, 4200), (5, 20001)])
@pytest.mark.parametrize("ex,ew,et", [(-9, -115, -120), (0, -124, -122), (0, -110, -126), (-60, -100, -108),
                                      (60, -100, -104), (9, 112, 118), (-60, 100, 104), (60, 110, 112), (0, 0, -30),
                                      (0, 0, 20)])
def test_norm_with_far_tensor_scales(b200, rows, cols, ex, ew, et):
    """The row's factor, the weights or the tensor scale near the ends of fp32, where the value
    that is quantised is an ordinary one."""
    x = (_input(cols, rows, cols, "f32") * 2.0 ** ex).to(torch.bfloat16)
    x[1] = 0
    w = (1 + 0.2 * torch.randn(cols, generator=torch.Generator().manual_seed(cols))).cuda() * 2.0 ** ew
    ts = 1.25 * 2.0 ** et
    t, _ = b200.rms_norm_mx(x, w, eps=0.0, fmt="nvfp4", tensor_scale=torch.tensor([ts], device="cuda"))
    with np.errstate(invalid="ignore"):
        y, _ = _norm_ref(_f64(x), _f64(w), None, 0.0)
    _check_norm(t, np.where(np.isnan(y), 0.0, y), ts)  # a row of zeros stays zero
    _ok(b200)


@pytest.fixture
def waits(b200):
    yield b200.lib().b200_mx_wait_limit
    assert b200.lib().b200_mx_wait_limit(0, 0) == 0


# rows kernel with and without K splits, and at both ring depths; pairs of every tile width
@pytest.mark.parametrize("fmt,M,N,K", [("nvfp4", 3, 1000, 8192), ("mxfp8", 20, 3000, 160), ("mxfp4", 100, 30000, 2048),
                                       ("nvfp4", 600, 900, 512), ("mxfp8", 2500, 2500, 1024),
                                       ("mxfp4", 4000, 4000, 1056)])
@pytest.mark.parametrize("hook", [1, 2])
def test_product_waits_run_out(b200, waits, fmt, M, N, K, hook):
    """Loads that never come, or an MMA warp that gives up with loads in flight: the kernel ends,
    the status word says so, and the next call is right."""
    rng = np.random.default_rng(K)
    (ca, ba), (cb, bb) = (X.random_operand(rng, n, K, fmt, exact=True) for n in (M, N))
    a, b = (b200.MxTensor(torch.from_numpy(X.element_bytes(c, fmt)).cuda(), torch.from_numpy(X.scale_tiles(s)).cuda(),
                          fmt, c.shape[0], K) for c, s in ((ca, ba), (cb, bb)))
    want = X.values(ca, ba, fmt, K) @ X.values(cb, bb, fmt, K).T
    c = torch.empty(M, N, device="cuda")
    for rep in range(3):
        assert waits(10_000_000, hook) == 0
        b200.gemm_mx(a, b, c)
        rc, bits = b200.status()
        assert rc == b200.ERR_DEVICE_TIMEOUT and bits & 0x80000000, (rc, hex(bits))
        assert waits(0, 0) == 0
        c.fill_(float("nan"))
        b200.gemm_mx(a, b, c)
        _ok(b200)
        np.testing.assert_array_equal(_f64(c), want)


# column counts that stream: the register kernel, which takes 4096, has no waits
@pytest.mark.parametrize("cols,residual", [(4112, True), (12000, False), (2056, True), (5008, False)])
@pytest.mark.parametrize("hook", [1, 2])
def test_norm_waits_run_out(b200, waits, cols, residual, hook):
    g = torch.Generator().manual_seed(cols)
    rows = 1500  # several rounds of the ring
    x, r = (torch.randn(rows, cols, generator=g).to(torch.bfloat16).cuda() for _ in range(2))
    r = r if residual else None
    w = torch.ones(cols, device="cuda", dtype=torch.bfloat16)
    want, h = b200.rms_norm_mx(x, w, r)
    _ok(b200)
    for rep in range(3):
        assert waits(10_000_000, hook) == 0
        b200.rms_norm_mx(x, w, r)
        rc, bits = b200.status()
        assert rc == b200.ERR_DEVICE_TIMEOUT and bits & 0x80000000, (rc, hex(bits))
        assert waits(0, 0) == 0
        t, k = b200.rms_norm_mx(x, w, r)
        _ok(b200)
        assert torch.equal(t.data, want.data) and torch.equal(t.scales, want.scales)
        assert not residual or torch.equal(k, h)


def test_refused_call_leaves_out_as_it_was(b200):
    """`out` takes a call's tensor scale; a call that is refused must not change what it stands
    for."""
    x, w = torch.randn(20, 96, device="cuda"), torch.ones(96, device="cuda")
    ts = torch.tensor([0.01], device="cuda")
    found = b200.quantize_mx(x, "nvfp4")
    given = b200.quantize_mx(x, "nvfp4", tensor_scale=ts)
    own = b200.MxTensor(given.data.clone(), given.scales.clone(), "nvfp4", 20, 96, ts)
    flat = torch.randn(1, 96, device="cuda").expand(20, 96)  # rows at one address: refused
    for t in (found, given, own):
        before, scale = b200.dequantize_mx(t, out_dtype="f32"), float(t.tensor_scale)
        for call in (lambda: b200.rms_norm_mx(x, w, eps=-1.0, fmt="nvfp4", out=t),
                     lambda: b200.rms_norm_mx(flat, w, fmt="nvfp4", out=t, tensor_scale=torch.ones(1, device="cuda")),
                     lambda: b200.quantize_mx(flat, "nvfp4", out=t),
                     lambda: b200.quantize_mx(flat, "nvfp4", out=t, tensor_scale=torch.ones(1, device="cuda"))):
            with pytest.raises(b200.B200Error):
                call()
            assert t.tensor_scale is not None and float(t.tensor_scale) == scale
            assert torch.equal(b200.dequantize_mx(t, out_dtype="f32"), before)
    _ok(b200)
