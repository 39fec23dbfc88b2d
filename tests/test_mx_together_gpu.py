"""GPU tests of microscaled operators run together: a layer's three products against the
unquantised layer's, and quantisers, norms and products on two streams at once.

Tolerances. An element is rounded to the nearest of its grid, so with A the largest magnitude of
its block it is off by at most
  mxfp8   2^-4 |x| (half a step of e4m3) or half the smallest step, 2^-10 times the block's scale,
          which is the smallest 2^e >= A / 448 and so below A / 224
  mxfp4   half the widest step of e2m1, 1 times the block's scale, below A / 3
  nvfp4   1 times the block's scale: A / 6 and its rounding to e4m3, 2^-4 of it or half the
          smallest step, 2^-10 times the tensor scale; a value beyond 6 scales is off by as much
          as the scale was rounded down, 6 times 2^-4 A / 6 or 6 times 2^-10 tensor scales. The
          tensor scale's own roundings (2^-22 of it in all) are far below the bound's slack.
With errors E of both operands a product is off by |A| E_B + E_A |B| + E_A E_B at most, and by
(K / 32 + 6) * 2^-23 * sum |a b| for its fp32 sums.
"""
from __future__ import annotations

import numpy as np
import pytest

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

FMTS = ["mxfp8", "mxfp4", "nvfp4"]


@pytest.fixture(scope="module", autouse=True)
def _cuda():
    if not torch.cuda.is_available():
        pytest.skip("no CUDA device")
    yield
    torch.cuda.synchronize()


def _f64(t):
    return t.double().cpu().numpy()


def _rounding(x, fmt):
    """Bound of the error of each element of x, quantised along its rows."""
    size = 16 if fmt == "nvfp4" else 32
    p = np.pad(np.abs(x), ((0, 0), (0, -x.shape[1] % 32))).reshape(x.shape[0], -1, size)
    top = p.max(-1, keepdims=True)
    if fmt == "mxfp8":
        e = np.maximum(2.0 ** -4 * p, 2.0 ** -10 * top / 224)
    elif fmt == "mxfp4":
        e = np.broadcast_to(top / 3, p.shape)
    else:
        ts = np.abs(x).max() / 2688
        e = np.broadcast_to(np.maximum(top / 6 * (1 + 2.0 ** -4) + 2.0 ** -10 * ts,
                                       6 * (2.0 ** -4 * top / 6 + 2.0 ** -10 * ts)), p.shape)
    return e.reshape(x.shape[0], -1)[:, :x.shape[1]]


@pytest.mark.parametrize("fmt", FMTS)
@pytest.mark.parametrize("M,N,K", [(200, 330, 290), (33, 64, 1056)])
def test_layer_is_near_the_unquantised_one(b200, fmt, M, N, K):
    """Y = X W^T, dX = dY W and dW = dY^T X on quantised operands against the same products of
    what was quantised, and dX and dW against differences of the unquantised layer's loss
    sum(Y * dY), of which they are the gradients."""
    g = torch.Generator().manual_seed(M + N + K)
    x, w, dy = (torch.randn(r, c, generator=g).to(torch.bfloat16).cuda() * s
                for r, c, s in ((M, K, 1.0), (N, K, 0.125), (M, N, 2.0 ** -7)))
    x64, w64, dy64 = _f64(x), _f64(w), _f64(dy)

    def product(a, b, ta, tb):
        got = _f64(b200.gemm_mx(b200.quantize_mx(a, fmt, transpose=ta), b200.quantize_mx(b, fmt, transpose=tb),
                                out_dtype="f32"))
        va, vb = (_f64(t).T if s else _f64(t) for t, s in ((a, ta), (b, tb)))
        ea, eb = _rounding(va, fmt), _rounding(vb, fmt)
        mag = np.abs(va) @ np.abs(vb).T
        off = np.abs(va) @ eb.T + ea @ np.abs(vb).T + ea @ eb.T
        tol = off + (va.shape[1] / 32 + 6) * 2.0 ** -23 * (mag + off)
        assert (np.abs(got - va @ vb.T) <= tol).all()
        return got, tol

    product(x, w, False, False)
    dx, tx = product(dy, w, False, True)
    dw, tw = product(dy, x, True, True)

    def loss(xv, wv):
        return float((dy64 * (xv @ wv.T)).sum())

    rng, size = np.random.default_rng(M), np.abs(dy64) * (np.abs(x64) @ np.abs(w64).T)
    slack = 1e-12 * float(size.sum())  # 64-bit sums, divided by a step of 1
    for _ in range(4):
        m, n, k = rng.integers(M), rng.integers(N), rng.integers(K)
        for of, at, got, tol in ((0, (m, k), dx, tx), (1, (n, k), dw, tw)):
            up, down = [x64.copy(), w64.copy()], [x64.copy(), w64.copy()]
            up[of][at] += 0.5
            down[of][at] -= 0.5
            assert abs(got[at] - (loss(*up) - loss(*down))) <= tol[at] + slack


@pytest.mark.parametrize("da,db", [(-100, -27), (-60, -70), (50, -110)])
def test_operands_far_from_one(b200, da, db):
    """Found tensor scales whose product leaves fp32's normal numbers, from the operands on."""
    M, N, K = 70, 90, 2080
    g = torch.Generator().manual_seed(3)
    x, w = (torch.randn(r, K, generator=g).cuda() for r in (M, N))
    x, w = x * 2.0 ** da, w * 2.0 ** db
    a, b = b200.quantize_mx(x, "nvfp4"), b200.quantize_mx(w, "nvfp4")
    got = _f64(b200.gemm_mx(a, b, out_dtype="f32"))
    x64, w64 = _f64(x), _f64(w)
    ea, eb = _rounding(x64, "nvfp4"), _rounding(w64, "nvfp4")
    mag = np.abs(x64) @ np.abs(w64).T
    off = np.abs(x64) @ eb.T + ea @ np.abs(w64).T + ea @ eb.T
    assert (np.abs(got - x64 @ w64.T) <= off + (K / 32 + 6) * 2.0 ** -23 * (mag + off) + 2.0 ** -150).all()


def test_quantisers_norms_and_products_on_two_streams(b200):
    """The scale-finding quantiser (its partial maxima and dependent launch), the norm's register
    and streaming kernels and both products, on two streams without any order between them, with
    other data on each: the bytes of the same calls one after the other."""
    g = torch.Generator().manual_seed(9)

    def data(scale):
        d = {"x": torch.randn(700, 4160, generator=g), "r": torch.randn(700, 4160, generator=g),
             "odd": torch.randn(331, 1001, generator=g), "w": torch.randn(640, 4160, generator=g)}
        return {k: (v * scale).to(torch.bfloat16).cuda() for k, v in d.items()}

    ones = torch.ones(4160, device="cuda", dtype=torch.bfloat16)

    def calls(d):
        q = b200.quantize_mx(d["w"], "nvfp4")
        t = b200.quantize_mx(d["odd"], "nvfp4", transpose=True)
        few, h0 = b200.rms_norm_mx(d["x"][:50], ones, d["r"][:50], fmt="nvfp4")
        many, h1 = b200.rms_norm_mx(d["x"], ones, d["r"], fmt="nvfp4")
        odd, _ = b200.rms_norm_mx(d["odd"], ones[:1001], fmt="mxfp8")
        out = [few.data, many.data, odd.data, h0, h1, q.data, q.tensor_scale, t.data, t.tensor_scale]
        return out + [q.scales, t.scales, many.scales, b200.gemm_mx(few, q), b200.gemm_mx(many, q),
                      b200.gemm_mx(t, t, out_dtype="f32"), b200.dequantize_mx(q)]

    sets = [data(1.0), data(3.0)]
    want = [calls(d) for d in sets]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    got = []
    for rep in range(10):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                got.append((i, calls(sets[i])))
    torch.cuda.synchronize()
    rc, bits = b200.status()
    assert rc == 0, hex(bits)
    for i, out in got:
        for a, b in zip(out, want[i]):
            assert torch.equal(a.view(torch.uint8), b.view(torch.uint8))
