"""hopper-lab_b200 — Python host mirror of the B200 GEMM C ABI (include/b200gemm.h).

The reference drives each GEMM experiment through
``dispatch(stages, flag, tmap_a, tmap_b, tmap_d, D, M, N, K[, group_m])``
(src/05_gemm/gemm_ws.cu:214-235, src/08_persistent/gemm_fp8_persist.cu:244-270),
which exits the process on any error. Here the same knobs (stages, group_m,
epilogue/variant) are arguments of :func:`gemm`, which calls ``b200_gemm`` in
``lib/libb200gemm.so`` through ctypes on torch-owned device memory and raises
:class:`B200Error` with the library's code instead of exiting.

There is no CPU fallback: if the shared library is missing, :func:`lib` raises.
The directory name contains a hyphen, so load it with
``importlib`` (see ``__graft_entry__.py``) or add the repository root to a
loader of your own; it registers itself as ``hopper_lab_b200``.
"""
from __future__ import annotations

import ctypes as C
import os
from pathlib import Path

PKG = Path(__file__).resolve().parent
# The in-tree build; B200GEMM_LIB names another build of the same ABI (e.g. one made
# with different compile-time options) to load instead.
LIB_PATH = Path(os.environ.get("B200GEMM_LIB") or PKG / "lib" / "libb200gemm.so")

DT_F16, DT_BF16, DT_E4M3, DT_F32 = 0, 1, 2, 3
VARIANTS = {"auto": 0, "1cta": 1, "2cta": 2, "persistent": 3, "clc": 4, "2cta_clc": 5,
            "2cta_streamk": 6}
VARIANT_NAMES = {v: k for k, v in VARIANTS.items()}

OK = 0
ERR_INVALID_ARG = -1
ERR_SHAPE = -2
ERR_ALIGN = -3
ERR_TMAP = -4
ERR_LAUNCH = -5
ERR_DEVICE_TIMEOUT = -6
ERR_UNSUPPORTED = -7
ERR_CUDA = -8
ERR_SCRATCH_LIMIT = -9

# Symbols declared in include/b200gemm.h (tests check the library exports them all).
EXPORTS = [
    "b200_gemm",
    "b200_gemm_strerror",
    "b200_gemm_status",
    "b200_gemm_variant_info",
    "b200_gemm_pick_variant",
    "b200_gemm_pick_config",
    "b200_quantize_e4m3",
    "b200_gemm_abi_version",
    "b200_gemm_noalloc",
    "b200_gemm_allgather",
    "b200_gemm_plan_create",
    "b200_gemm_plan_launch",
    "b200_gemm_plan_destroy",
    "b200_mx_layout",
    "b200_mx_quantize",
    "b200_mx_dequantize",
    "b200_mx_gemm",
    "b200_mx_rms_norm",
    "b200_mx_wait_limit",
]
GATHER_MULTICAST, GATHER_PEERS = 1, 2
MX_FORMATS = {"mxfp8": 0, "mxfp4": 1, "nvfp4": 2}
MX_NORM_MAX_COLS = 32768
MX_SCALE_BYTES = 272
_MX_GAP = 512  # MX_SCALE_BYTES in whole 256-byte units


class GemmArgs(C.Structure):
    """Mirror of ``B200GemmArgs`` (include/b200gemm.h)."""

    _fields_ = [
        ("ab_dtype", C.c_int32),
        ("c_dtype", C.c_int32),
        ("M", C.c_int64),
        ("N", C.c_int64),
        ("K", C.c_int64),
        ("lda", C.c_int64),
        ("ldb", C.c_int64),
        ("ldc", C.c_int64),
        ("A", C.c_void_p),
        ("B", C.c_void_p),
        ("C", C.c_void_p),
        ("scale_a", C.c_void_p),
        ("scale_b", C.c_void_p),
        ("variant", C.c_int32),
        ("group_m", C.c_int32),
        ("stages", C.c_int32),
        ("fault_inject", C.c_int32),
        ("wait_limit_ns", C.c_uint64),
        ("tile_n", C.c_int32),
        ("reserved", C.c_int32),
    ]


class MxDesc(C.Structure):
    """Mirror of ``B200MxTensor`` (include/b200gemm.h)."""

    _fields_ = [
        ("format", C.c_int32),
        ("reserved", C.c_int32),
        ("rows", C.c_int64),
        ("cols", C.c_int64),
        ("ld", C.c_int64),
        ("data", C.c_void_p),
        ("scales", C.c_void_p),
        ("tensor_scale", C.c_void_p),
    ]


class MxNormArgs(C.Structure):
    """Mirror of ``B200MxNormArgs`` (include/b200gemm.h)."""

    _fields_ = [
        ("dtype", C.c_int32),
        ("weight_dtype", C.c_int32),
        ("x", C.c_void_p),
        ("weight", C.c_void_p),
        ("residual", C.c_void_p),
        ("h", C.c_void_p),
        ("ldx", C.c_int64),
        ("ldr", C.c_int64),
        ("ldh", C.c_int64),
        ("eps", C.c_float),
        ("reserved", C.c_int32),
    ]


class B200Error(RuntimeError):
    def __init__(self, code: int, what: str = ""):
        self.code = code
        msg = strerror(code)
        super().__init__(f"{what}: {msg} ({code})" if what else f"{msg} ({code})")


_LIB = None


def lib():
    """Load libb200gemm.so (raises if it was not built — there is no fallback)."""
    global _LIB
    if _LIB is None:
        if not LIB_PATH.exists():
            raise RuntimeError(
                f"{LIB_PATH} is missing: build it with `python hopper-lab_b200/build.py` "
                "(there is no CPU fallback)")
        L = C.CDLL(str(LIB_PATH))
        L.b200_gemm.argtypes = [C.POINTER(GemmArgs), C.c_void_p]
        L.b200_gemm.restype = C.c_int
        L.b200_gemm_strerror.argtypes = [C.c_int]
        L.b200_gemm_strerror.restype = C.c_char_p
        L.b200_gemm_status.argtypes = [C.c_void_p, C.c_int, C.POINTER(C.c_uint32)]
        L.b200_gemm_status.restype = C.c_int
        L.b200_gemm_variant_info.argtypes = [C.c_int32, C.c_int32] + [C.POINTER(C.c_int32)] * 4
        L.b200_gemm_variant_info.restype = C.c_int
        L.b200_gemm_pick_variant.argtypes = [C.POINTER(GemmArgs)]
        L.b200_gemm_pick_variant.restype = C.c_int
        L.b200_gemm_pick_config.argtypes = [C.POINTER(GemmArgs), C.POINTER(C.c_int32),
                                            C.POINTER(C.c_int32)]
        L.b200_gemm_pick_config.restype = C.c_int
        L.b200_quantize_e4m3.argtypes = [C.c_void_p, C.c_int64, C.c_void_p, C.c_void_p, C.c_void_p]
        L.b200_quantize_e4m3.restype = C.c_int
        L.b200_gemm_abi_version.argtypes = []
        L.b200_gemm_abi_version.restype = C.c_int
        L.b200_gemm_allgather.argtypes = [C.POINTER(GemmArgs), C.c_void_p, C.c_int32, C.c_int32,
                                          C.c_int64, C.c_int64, C.c_void_p]
        L.b200_gemm_allgather.restype = C.c_int
        L.b200_gemm_plan_create.argtypes = [C.POINTER(GemmArgs), C.POINTER(C.c_void_p)]
        L.b200_gemm_plan_create.restype = C.c_int
        L.b200_gemm_plan_launch.argtypes = [C.c_void_p, C.c_void_p]
        L.b200_gemm_plan_launch.restype = C.c_int
        L.b200_gemm_plan_destroy.argtypes = [C.c_void_p]
        L.b200_gemm_plan_destroy.restype = None
        L.b200_mx_layout.argtypes = [C.c_int32, C.c_int64, C.c_int64, C.POINTER(C.c_int64),
                                     C.POINTER(C.c_int64)]
        L.b200_mx_quantize.argtypes = [C.c_void_p, C.c_int32, C.c_int64, C.c_int32, C.c_int32,
                                       C.POINTER(MxDesc), C.c_void_p]
        L.b200_mx_dequantize.argtypes = [C.POINTER(MxDesc), C.c_void_p, C.c_int32, C.c_int64, C.c_void_p]
        L.b200_mx_gemm.argtypes = [C.POINTER(MxDesc), C.POINTER(MxDesc), C.c_void_p, C.c_int32, C.c_int64,
                                   C.c_void_p]
        L.b200_mx_rms_norm.argtypes = [C.POINTER(MxNormArgs), C.POINTER(MxDesc), C.c_void_p]
        L.b200_mx_wait_limit.argtypes = [C.c_uint64, C.c_int32]
        _LIB = L
    return _LIB


def strerror(code: int) -> str:
    try:
        return lib().b200_gemm_strerror(code).decode()
    except Exception:  # library missing: still produce a message
        return f"error {code}"


def variant_info(variant: str | int, ab_dtype: int = DT_F16, tile_n: int = 0):
    v = VARIANTS[variant] if isinstance(variant, str) else int(variant)
    out = [C.c_int32() for _ in range(4)]
    out[1].value = tile_n
    rc = lib().b200_gemm_variant_info(v, ab_dtype, *[C.byref(o) for o in out])
    if rc != OK:
        raise B200Error(rc, "variant_info")
    return {"tile_m": out[0].value, "tile_n": out[1].value, "max_stages": out[2].value,
            "default_stages": out[3].value}


# ---------------------------------------------------------------------------- torch glue
def _torch():
    import torch  # noqa: WPS433 — torch is plumbing (device memory, streams) only

    return torch


def _dt_of(t) -> int:
    torch = _torch()
    if t.dtype == torch.float16:
        return DT_F16
    if t.dtype == torch.bfloat16:
        return DT_BF16
    if t.dtype in (torch.float8_e4m3fn, torch.uint8):
        return DT_E4M3
    if t.dtype == torch.float32:
        return DT_F32
    raise TypeError(f"unsupported dtype {t.dtype}")


def _torch_dtype(dt: int):
    torch = _torch()
    return {DT_F16: torch.float16, DT_BF16: torch.bfloat16, DT_F32: torch.float32,
            DT_E4M3: torch.float8_e4m3fn}[dt]


def _dtype_code(name) -> int:
    if isinstance(name, int):
        return name
    return {"f16": DT_F16, "fp16": DT_F16, "float16": DT_F16, "bf16": DT_BF16,
            "bfloat16": DT_BF16, "e4m3": DT_E4M3, "fp8": DT_E4M3, "f32": DT_F32,
            "fp32": DT_F32, "float32": DT_F32}[name]


def _stream_handle(stream) -> int:
    torch = _torch()
    if stream is None:
        return torch.cuda.current_stream().cuda_stream
    if isinstance(stream, int):
        return stream
    return stream.cuda_stream


def make_args(a, b, c, *, scale_a=None, scale_b=None, variant="auto", group_m=0, stages=0,
              wait_limit_ns=0, fault_inject=0, tile_n=0) -> GemmArgs:
    """Fill B200GemmArgs from 2-D torch tensors (row-major, unit column stride)."""
    for name, t in (("A", a), ("B", b), ("C", c)):
        if t.dim() != 2 or (t.numel() > 0 and t.stride(1) != 1):
            raise ValueError(f"{name} must be a 2-D row-major tensor with unit column stride")
    M, K = a.shape
    N, K2 = b.shape
    if K != K2 or tuple(c.shape) != (M, N):
        raise ValueError(f"shape mismatch: A {tuple(a.shape)}, B {tuple(b.shape)}, C {tuple(c.shape)}")
    args = GemmArgs()
    args.ab_dtype = _dt_of(a)
    if _dt_of(b) != args.ab_dtype:
        raise TypeError("A and B must have the same element type")
    args.c_dtype = _dt_of(c)
    args.M, args.N, args.K = M, N, K
    args.lda = a.stride(0) if M > 1 else max(K, 1)
    args.ldb = b.stride(0) if N > 1 else max(K, 1)
    args.ldc = c.stride(0) if M > 1 else max(N, 1)
    args.A, args.B, args.C = a.data_ptr(), b.data_ptr(), c.data_ptr()
    args.scale_a = scale_a.data_ptr() if scale_a is not None else None
    args.scale_b = scale_b.data_ptr() if scale_b is not None else None
    args.variant = VARIANTS[variant] if isinstance(variant, str) else int(variant)
    args.group_m = group_m
    args.stages = stages
    args.fault_inject = fault_inject
    args.wait_limit_ns = wait_limit_ns
    args.tile_n = tile_n
    return args


def gemm(a, b, c=None, *, out_dtype="bf16", scale_a=None, scale_b=None, variant="auto",
         group_m: int = 0, stages: int = 0, wait_limit_ns: int = 0, fault_inject: int = 0,
         tile_n: int = 0, stream=None):
    """C = scale_a * scale_b * A . B^T on the GPU (A: M x K, B: N x K, both row-major).

    A/B: torch.float16 | torch.bfloat16 | torch.float8_e4m3fn (or uint8 bits).
    C is allocated with ``out_dtype`` when not given. scale_a/scale_b are 1-element
    fp32 device tensors (or None). Returns C. Raises B200Error on any failure.
    """
    torch = _torch()
    if c is None:
        c = torch.empty((a.shape[0], b.shape[0]), dtype=_torch_dtype(_dtype_code(out_dtype)),
                        device=a.device)
    args = make_args(a, b, c, scale_a=scale_a, scale_b=scale_b, variant=variant, group_m=group_m,
                     stages=stages, wait_limit_ns=wait_limit_ns, fault_inject=fault_inject,
                     tile_n=tile_n)
    rc = lib().b200_gemm(C.byref(args), C.c_void_p(_stream_handle(stream)))
    if rc != OK:
        raise B200Error(rc, "b200_gemm")
    return c


def gemm_allgather(a, b, c, dst: int, mode: int, npeers: int, ldg: int, col_off: int, *,
                   scale_a=None, scale_b=None, variant="auto", tile_n: int = 0, stream=None):
    """b200_gemm_allgather: C = scale_a*scale_b*A.B^T on this GPU, and every C tile also
    stored at G[row*ldg + col_off + col] on every GPU of the node. `dst` is the multicast
    address of G (mode GATHER_MULTICAST) or the device address of an array of `npeers`
    peer base addresses (GATHER_PEERS). The caller synchronises the GPUs before reading G."""
    args = make_args(a, b, c, scale_a=scale_a, scale_b=scale_b, variant=variant, tile_n=tile_n)
    rc = lib().b200_gemm_allgather(C.byref(args), C.c_void_p(dst), mode, npeers, ldg, col_off,
                                   C.c_void_p(_stream_handle(stream)))
    if rc != OK:
        raise B200Error(rc, "b200_gemm_allgather")
    return c


class Plan:
    """b200_gemm_plan_*: a GEMM resolved once (variant, tensor maps, kernel parameters)
    on fixed buffers; `launch()` only launches. Keeps references to the tensors so the
    buffers outlive the plan."""

    def __init__(self, a, b, c, **kw):
        self._h = None
        self._keep = (a, b, c, kw.get("scale_a"), kw.get("scale_b"))
        args = make_args(a, b, c, **kw)
        h = C.c_void_p()
        rc = lib().b200_gemm_plan_create(C.byref(args), C.byref(h))
        if rc != OK:
            raise B200Error(rc, "b200_gemm_plan_create")
        self._h = h

    def launch(self, stream=None):
        rc = lib().b200_gemm_plan_launch(self._h, C.c_void_p(_stream_handle(stream)))
        if rc != OK:
            raise B200Error(rc, "b200_gemm_plan_launch")

    def close(self):
        if self._h:
            lib().b200_gemm_plan_destroy(self._h)
            self._h = None

    def __del__(self):
        try:
            self.close()
        except Exception:
            pass


def gemm_raw(args: GemmArgs, stream=None) -> int:
    """Call b200_gemm with a prepared argument block; returns the raw code."""
    return lib().b200_gemm(C.byref(args), C.c_void_p(_stream_handle(stream)))


def pick_variant(a, b, c) -> str:
    args = make_args(a, b, c)
    v = lib().b200_gemm_pick_variant(C.byref(args))
    if v < 0:
        raise B200Error(v, "pick_variant")
    return VARIANT_NAMES[v]


def pick_config(args: GemmArgs) -> tuple[str, int]:
    """(variant name, tile width) that b200_gemm launches for a prepared argument block."""
    v, tn = C.c_int32(), C.c_int32()
    rc = lib().b200_gemm_pick_config(C.byref(args), C.byref(v), C.byref(tn))
    if rc != OK:
        raise B200Error(rc, "pick_config")
    return VARIANT_NAMES[v.value], tn.value


def status(stream=None, clear: bool = True):
    """(code, bits): B200_OK or B200_ERR_DEVICE_TIMEOUT with the raw device bits."""
    bits = C.c_uint32()
    rc = lib().b200_gemm_status(C.c_void_p(_stream_handle(stream)), 1 if clear else 0,
                                C.byref(bits))
    return rc, bits.value


def quantize_e4m3(x, q=None, scale=None, stream=None):
    """Device per-tensor quantiser: returns (q float8_e4m3fn, scale fp32[1])."""
    torch = _torch()
    if x.dtype != torch.float32 or not x.is_contiguous():
        raise ValueError("x must be a contiguous float32 tensor")
    if q is None:
        q = torch.empty(x.shape, dtype=torch.float8_e4m3fn, device=x.device)
    if scale is None:
        scale = torch.empty(1, dtype=torch.float32, device=x.device)
    rc = lib().b200_quantize_e4m3(C.c_void_p(x.data_ptr()), x.numel(), C.c_void_p(q.data_ptr()),
                                  C.c_void_p(scale.data_ptr()),
                                  C.c_void_p(_stream_handle(stream)))
    if rc != OK:
        raise B200Error(rc, "b200_quantize_e4m3")
    return q, scale


# ------------------------------------------------------------------ microscaled operands
# These calls are short kernels, so their host side is kept short too: one allocation for a
# microscaled matrix, views of it only when asked for, raw stream handles, names looked up
# once (_mx_setup).


def mx_layout(fmt: str, rows: int, cols: int) -> tuple[int, int]:
    """(bytes of one row of elements, bytes of all scale tiles) of a microscaled matrix."""
    row, scale = C.c_int64(), C.c_int64()
    rc = lib().b200_mx_layout(MX_FORMATS[fmt], rows, cols, C.byref(row), C.byref(scale))
    if rc != OK:
        raise B200Error(rc, "b200_mx_layout")
    return row.value, scale.value


class MxTensor:
    """A microscaled matrix (``B200MxTensor``): 8- or 4-bit elements with a scale per block
    of consecutive elements of a row.

    ``fmt``           "mxfp8" (e4m3, blocks of 32), "mxfp4" (e2m1, blocks of 32) or "nvfp4"
                      (e2m1, blocks of 16 with e4m3 scales and one fp32 scale)
    ``rows, cols``    logical size; products sum over ``cols``
    ``data``          uint8, rows x row bytes (cols padded to a multiple of 32 with zeros)
    ``scales``        uint8, (ceil(rows / 128), tiles along the row, 32, 16), contiguous
    ``tensor_scale``  1-element fp32 tensor or None ("nvfp4" only)
    """

    __slots__ = ("_data", "_scales", "fmt", "rows", "cols", "device", "_ts", "_desc", "_ref", "_own", "_off")

    def __init__(self, data, scales, fmt: str, rows: int, cols: int, tensor_scale=None):
        torch = _torch()
        row_bytes, scale_bytes = mx_layout(fmt, rows, cols)
        if data.dtype != torch.uint8 or scales.dtype != torch.uint8:
            raise TypeError("data and scales must be uint8 tensors")
        if tuple(data.shape) != (rows, row_bytes) or (data.numel() > 0 and data.stride(1) != 1):
            raise ValueError(f"data must be ({rows}, {row_bytes}) with unit column stride, not {tuple(data.shape)}")
        if scales.numel() != scale_bytes or not scales.is_contiguous():
            raise ValueError(f"scales must hold {scale_bytes} contiguous bytes, not {scales.numel()}")
        if scales.device != data.device:
            raise ValueError("data and scales must be on one device")
        self._data, self._scales, self._own, self._off, self._ts = data, scales, None, 0, None
        self.fmt, self.rows, self.cols, self.device = fmt, rows, cols, data.device
        self._desc = MxDesc(MX_FORMATS[fmt], 0, rows, cols, data.stride(0) if rows > 1 else row_bytes,
                            data.data_ptr(), scales.data_ptr(), None)
        self._ref = C.byref(self._desc)
        self.tensor_scale = tensor_scale

    @classmethod
    def empty(cls, rows: int, cols: int, fmt: str, device="cuda", tensor_scale=None) -> "MxTensor":
        """Uninitialised storage for a rows x cols matrix."""
        mx_layout(fmt, rows, cols)  # refuses what has no layout
        t = cls._new(rows, cols, fmt, device)
        if tensor_scale is not None:
            t.tensor_scale = tensor_scale
        return t

    @classmethod
    def _new(cls, rows, cols, fmt, device):
        # one buffer: scale tiles, the tensor scale and its scratch, element rows
        kp = (cols + 31) // 32 * 32
        if fmt == "nvfp4":
            groups, row_bytes, code = (kp + 63) // 64, kp // 2, 2
        elif fmt == "mxfp8":
            groups, row_bytes, code = (kp + 127) // 128, kp, 0
        else:
            groups, row_bytes, code = (kp + 127) // 128, kp // 2, 1
        scale_bytes = (rows + 127) // 128 * groups * 512
        self = _new_object(cls)
        self._own = buf = (_empty or _mx_setup())(scale_bytes + _MX_GAP + rows * row_bytes, dtype=_uint8,
                                                  device=device)
        self._off = scale_bytes
        ptr = buf.data_ptr()
        self._data = self._scales = self._ts = None
        self.fmt, self.rows, self.cols, self.device = fmt, rows, cols, buf.device
        self._desc = desc = MxDesc(code, 0, rows, cols, row_bytes, ptr + scale_bytes + _MX_GAP, ptr, None)
        self._ref = C.byref(desc)
        return self

    @property
    def data(self):
        if self._data is None:
            ld = self._desc.ld
            self._data = self._own.as_strided((self.rows, ld), (ld, 1), self._off + _MX_GAP)
        return self._data

    @property
    def scales(self):
        if self._scales is None:
            bands = (self.rows + 127) // 128
            tiles = self._off // 512 // max(bands, 1)
            self._scales = self._own.as_strided((bands, tiles, 32, 16), (tiles * 512, 512, 16, 1), 0)
        return self._scales

    @property
    def tensor_scale(self):
        if self._ts is None and self._desc.tensor_scale is not None:
            # found by the quantiser into this matrix's own buffer
            self._ts = self._own[self._off:self._off + 4].view(_torch().float32)
        return self._ts

    @tensor_scale.setter
    def tensor_scale(self, ts):
        if ts is not None:
            if self.fmt != "nvfp4":
                raise ValueError(f"{self.fmt} has no tensor scale")
            if ts.dtype != _torch().float32 or ts.numel() != 1 or ts.device != self.device:
                raise ValueError("tensor_scale must be one float32 on the data's device")
        self._ts = ts
        self._desc.tensor_scale = None if ts is None else ts.data_ptr()

    def _scratch(self):
        """Room for a tensor scale to be found into."""
        if self._own is None:  # data and scales are the caller's: a buffer beside them
            self._own = _torch().empty(_MX_GAP, dtype=_torch().uint8, device=self.device)
        self._ts = None
        self._desc.tensor_scale = self._own.data_ptr() + self._off

    @property
    def shape(self) -> tuple[int, int]:
        return self.rows, self.cols


_MX_TORCH = {}  # torch dtype -> code and the names of output types -> (torch dtype, code)
_empty = _empty_strided = _uint8 = _get_device = _raw_stream = None
_new_object = object.__new__


def _mx_setup():
    global _empty, _empty_strided, _uint8, _get_device, _raw_stream
    torch = _torch()
    for dt, code, names in ((torch.float16, DT_F16, ("f16", "fp16", "float16")),
                            (torch.bfloat16, DT_BF16, ("bf16", "bfloat16")),
                            (torch.float32, DT_F32, ("f32", "fp32", "float32"))):
        for name in names + (code,):
            _MX_TORCH[name] = (dt, code)
        _MX_TORCH[dt] = code
    _uint8, _empty_strided = torch.uint8, torch.empty_strided
    _get_device, _raw_stream = torch._C._cuda_getDevice, torch._C._cuda_getCurrentRawStream
    lib()
    _empty = torch.empty  # last: the others are there once it is
    return _empty


def _mx_input(name, t):
    """dtype code and row stride of a 2-D fp tensor with unit column stride."""
    if _empty is None:
        _mx_setup()
    dt = _MX_TORCH.get(t.dtype)
    if dt is None:
        raise TypeError(f"{name} must be float16, bfloat16 or float32, not {t.dtype}")
    stride = t.stride()
    if len(stride) != 2:
        raise ValueError(f"{name} must be a 2-D row-major tensor with unit column stride")
    rows, cols = t.shape
    if stride[1] != 1 and cols > 1 and rows > 0:
        raise ValueError(f"{name} must be a 2-D row-major tensor with unit column stride")
    return dt, stride[0] if rows > 1 else cols or 1


def _mx_output(name, rows, cols, device):
    """A new matrix of the named output type, its code and row stride."""
    kind = _MX_TORCH.get(name)
    if type(kind) is not tuple:
        raise ValueError(f"output type {name!r} is not f16, bf16 or f32")
    ld = cols or 1
    return _empty_strided((rows, cols), (ld, 1), dtype=kind[0], device=device), kind[1], ld


def _mx_failed(rc, what, out, kept):
    """Raise for a refused call that was to write `out`, which keeps the scale it had."""
    if out is not None:
        out._ts, out._desc.tensor_scale = kept
    raise B200Error(rc, what)


def _mx_out(out, rows, cols, fmt, device, tensor_scale):
    if out is None:
        if fmt not in MX_FORMATS:
            raise ValueError(f"unknown format {fmt!r}")
        out = MxTensor._new(rows, cols, fmt, device)
        if tensor_scale is not None:
            out.tensor_scale = tensor_scale
        return out
    if out.fmt != fmt or out.rows != rows or out.cols != cols or out.device != device:
        raise ValueError(f"out is {out.fmt} {out.shape} on {out.device}, needed {fmt} {(rows, cols)} on {device}")
    out.tensor_scale = tensor_scale
    return out


class _On:
    """Makes a call's device and stream the current ones, so that what it allocates belongs to
    the stream that its kernels run on. ``stream``: None (the device's current one), a torch
    stream or a raw handle."""

    __slots__ = ("_device", "_stream")

    def __init__(self, device, stream):
        cuda = _torch().cuda
        if device.type != "cuda":
            raise ValueError(f"tensors must be on a CUDA device, not {device}")
        self._device = cuda.device(device)
        if stream is not None:
            if not isinstance(stream, int) and stream.device != device:
                raise ValueError(f"stream is on {stream.device}, the tensors are on {device}")
            stream = cuda.stream(cuda.ExternalStream(stream, device=device) if isinstance(stream, int) else stream)
        self._stream = stream

    def __enter__(self):
        self._device.__enter__()
        if self._stream is not None:
            self._stream.__enter__()

    def __exit__(self, *exc):
        if self._stream is not None:
            self._stream.__exit__(*exc)
        self._device.__exit__(*exc)


def _here(device, stream):
    """Handle of the current stream for a call on the current device and stream, else None:
    the call then makes them current (_On) and starts over."""
    index = device.index
    if stream is None and index is not None:
        if _empty is None:
            _mx_setup()
        if _get_device() == index:
            return _raw_stream(index)
    return None


def quantize_mx(x, fmt: str = "nvfp4", *, transpose: bool = False, tensor_scale=None, out: MxTensor | None = None,
                stream=None) -> MxTensor:
    """Quantise a matrix (f16, bf16 or f32) to a microscaled one; with ``transpose`` its
    transpose, for products that sum over x's rows. For "nvfp4", ``tensor_scale`` is one
    positive fp32 on the device, used as given; None finds max|x| / 2688 in an extra pass.
    ``out`` is written in place and takes the tensor scale."""
    dt, ldx = _mx_input("x", x)
    device = x.device
    here = _here(device, stream)
    if here is None:
        with _On(device, stream):
            return quantize_mx(x, fmt, transpose=transpose, tensor_scale=tensor_scale, out=out)
    rows, cols = x.shape
    if transpose:
        rows, cols = cols, rows
    kept = None if out is None else (out._ts, out._desc.tensor_scale)
    t = _mx_out(out, rows, cols, fmt, device, tensor_scale)
    find = fmt == "nvfp4" and tensor_scale is None
    if find:
        t._scratch()
    rc = _LIB.b200_mx_quantize(x.data_ptr(), dt, ldx, transpose, find, t._ref, here)
    if rc != OK:
        _mx_failed(rc, "b200_mx_quantize", out, kept)
    return t


def dequantize_mx(t: MxTensor, out=None, *, out_dtype="bf16", stream=None):
    """The values a microscaled matrix stands for, rounded to f16, bf16 or f32 (behind a tensor
    scale to fp32 first)."""
    device = t.device
    here = _here(device, stream)
    if here is None:
        with _On(device, stream):
            return dequantize_mx(t, out, out_dtype=out_dtype)
    if out is None:
        out, dt, ldy = _mx_output(out_dtype, t.rows, t.cols, device)
    else:
        if tuple(out.shape) != t.shape or out.device != device:
            raise ValueError(f"out is {tuple(out.shape)} on {out.device}, needed {t.shape} on {device}")
        dt, ldy = _mx_input("out", out)
    rc = _LIB.b200_mx_dequantize(t._ref, out.data_ptr(), dt, ldy, here)
    if rc != OK:
        raise B200Error(rc, "b200_mx_dequantize")
    return out


def gemm_mx(a: MxTensor, b: MxTensor, c=None, *, out_dtype="bf16", stream=None):
    """C = A . B^T of the values two microscaled matrices stand for (A: M x K, B: N x K,
    same format), fp32 accumulation, to f16, bf16 or f32. Any row stride of C is accepted. A
    device wait that runs out leaves C undefined and shows in :func:`status`."""
    device = a.device
    if a.fmt != b.fmt:
        raise TypeError(f"A and B must have the same format, not {a.fmt} and {b.fmt}")
    if a.cols != b.cols or device != b.device:
        raise ValueError(f"shape or device mismatch: A {a.shape} on {device}, B {b.shape} on {b.device}")
    here = _here(device, stream)
    if here is None:
        with _On(device, stream):
            return gemm_mx(a, b, c, out_dtype=out_dtype)
    if c is None:
        c, dt, ldc = _mx_output(out_dtype, a.rows, b.rows, device)
    else:
        if tuple(c.shape) != (a.rows, b.rows) or c.device != device:
            raise ValueError(f"C is {tuple(c.shape)} on {c.device}, needed {(a.rows, b.rows)} on {device}")
        dt, ldc = _mx_input("C", c)
    rc = _LIB.b200_mx_gemm(a._ref, b._ref, c.data_ptr(), dt, ldc, here)
    if rc != OK:
        raise B200Error(rc, "b200_mx_gemm")
    return c


def rms_norm_mx(x, weight, residual=None, *, eps: float = 1e-6, fmt: str = "mxfp8", tensor_scale=None,
                out: MxTensor | None = None, residual_out=None, stream=None):
    """RMS norm with the residual's addition, to a microscaled matrix: h = x + residual,
    out = quantised(h / sqrt(mean(h^2) + eps) * weight), up to 2^-17 of that value. Returns
    (out, h), h rounded to x's type, or (out, None) without a residual. ``residual_out`` may be ``residual`` or ``x``,
    and overlaps neither otherwise. ``weight`` has x's type or is float32; ``tensor_scale``
    ("nvfp4") is used as given, None stands for 1, which suits normalised rows (block maxima
    from 0.006 to 2688)."""
    dt, ldx = _mx_input("x", x)
    device = x.device
    shape = x.shape
    rows, cols = shape
    wt = _MX_TORCH.get(weight.dtype)
    if weight.shape != (cols,) or not weight.is_contiguous() or weight.device != device:
        raise ValueError(f"weight must hold {cols} contiguous elements on {device}")
    if wt != dt and wt != DT_F32:
        raise TypeError(f"weight must be {x.dtype} or float32, not {weight.dtype}")
    if residual is None and residual_out is not None:
        raise ValueError("residual_out needs a residual")
    here = _here(device, stream)
    if here is None:
        with _On(device, stream):
            return rms_norm_mx(x, weight, residual, eps=eps, fmt=fmt, tensor_scale=tensor_scale, out=out,
                               residual_out=residual_out)
    if residual is None:
        args = MxNormArgs(dt, wt, x.data_ptr(), weight.data_ptr(), None, None, ldx, 0, 0, eps, 0)
    else:
        if residual.shape != shape or residual.device != device:
            raise ValueError(f"residual must match x: {tuple(shape)} on {device}")
        rt, ldr = _mx_input("residual", residual)
        if residual_out is None:
            residual_out, ht, ldh = _mx_output(dt, rows, cols, device)
        else:
            if residual_out.shape != shape or residual_out.device != device:
                raise ValueError(f"residual_out must match x: {tuple(shape)} on {device}")
            ht, ldh = _mx_input("residual_out", residual_out)
        if rt != dt or ht != dt:
            raise TypeError(f"residual and residual_out must be {x.dtype}")
        args = MxNormArgs(dt, wt, x.data_ptr(), weight.data_ptr(), residual.data_ptr(), residual_out.data_ptr(),
                          ldx, ldr, ldh, eps, 0)
    kept = None if out is None else (out._ts, out._desc.tensor_scale)
    t = _mx_out(out, rows, cols, fmt, device, tensor_scale)
    rc = _LIB.b200_mx_rms_norm(C.byref(args), t._ref, here)
    if rc != OK:
        _mx_failed(rc, "b200_mx_rms_norm", out, kept)
    return t, residual_out
