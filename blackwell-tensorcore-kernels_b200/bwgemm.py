"""Python face of libbwgemm.so (the C ABI declared in include/bwgemm.h).

Used by bench.py, tests/ and __graft_entry__. Device memory and streams come from torch;
every call goes through the C ABI with raw pointers, so what runs is the in-tree CUDA
library. There is no fallback: if the shared library is missing or fails to load, every
entry point raises.

Reference interface mirrored (paths within waynehacking8/blackwell-tensorcore-kernels):
  launch_<name>(A, B, C, M, N, K)  src/main.cu:18-39 -> launch(name, A, B, C) below, with the
  same staging semantics (FP32 inputs are cast/quantised by the launcher, cached by pointer
  identity and shape, src/gemm_mma.cu:152-168, src/gemm_mma_fp8.cu:230-264).
"""
from __future__ import annotations

import contextlib
import ctypes
import functools
import os
import re
import subprocess

_HERE = os.path.dirname(os.path.abspath(__file__))
REPO = os.path.dirname(_HERE)
LIB_PATH = os.path.join(_HERE, "libbwgemm.so")
HEADER = os.path.join(REPO, "include", "bwgemm.h")

BW_OK, BW_ERR_INVALID, BW_ERR_CUDA, BW_ERR_TIMEOUT, BW_ERR_UNSUPPORTED = 0, 1, 2, 3, 4
OUT_F32, OUT_BF16 = 0, 1
SCALE_NONE, SCALE_FIXED8, SCALE_AMAX = 0, 1, 2
FP4_PACKED, FP4_BYTE_SHL2 = 0, 1
MX_UNIT_FIXED8, MX_BLOCK32 = 0, 1
DTYPE_F16, DTYPE_FP8, DTYPE_FP4, DTYPE_MXFP4, DTYPE_BF16, DTYPE_F32 = 0, 1, 2, 3, 4, 5


class Shard(ctypes.Structure):
    """bw_shard_t: one GPU's part of a single-process sharded GEMM (include/bwgemm.h)."""

    _fields_ = [("device", ctypes.c_int), ("A", ctypes.c_void_p), ("B", ctypes.c_void_p),
                ("sfA", ctypes.c_void_p), ("sfB", ctypes.c_void_p), ("scale_a", ctypes.c_void_p),
                ("scale_b", ctypes.c_void_p), ("C", ctypes.c_void_p), ("C_gathered", ctypes.c_void_p),
                ("stream", ctypes.c_void_p)]


class BwError(RuntimeError):
    def __init__(self, code: int, msg: str):
        super().__init__(f"bwgemm error {code}: {msg}")
        self.code = code


_lib = None


def build(tools: bool = False) -> None:
    """Compile the library (and optionally gemm_bench / tc_rate_probe) for sm_100a in-tree."""
    targets = ["all"] + (["tools"] if tools else [])
    subprocess.run(["make", "-s", "-C", _HERE, *targets], check=True)


def declared_functions() -> list[str]:
    """Names of the entry points include/bwgemm.h declares."""
    text = open(HEADER).read()
    text = re.sub(r"/\*.*?\*/", "", text, flags=re.S)
    return re.findall(r"^\s*(?:int|size_t|const char\*)\s+(bw_\w+)\s*\(", text, flags=re.M)


def lib():
    global _lib
    if _lib is not None:
        return _lib
    if not os.path.exists(LIB_PATH):
        raise RuntimeError(f"{LIB_PATH} is missing: run __graft_entry__.build() (make -C {_HERE})")
    L = ctypes.CDLL(LIB_PATH)
    P, I, LL = ctypes.c_void_p, ctypes.c_int, ctypes.c_longlong
    F, SZ = ctypes.c_float, ctypes.c_size_t
    sig = {
        "bw_init": [I],
        "bw_shutdown": [],
        "bw_version": [],
        "bw_num_sms": [I],
        "bw_device_state_ready": [I],
        "bw_device_status": [P, P],
        "bw_set_wait_budget_ns": [ctypes.c_ulonglong],
        "bw_set_trace_buffer": [P, I],
        "bw_selftest_bounded_wait": [ctypes.c_ulonglong, P],
        "bw_selftest_grouped_wait": [I, I, P, P, P, I, P, I, I, I, I, I, I, ctypes.c_ulonglong, P, P],
        "bw_gemm_f16": [P, P, P, I, I, I, P],
        "bw_gemm_f16_bt": [P, P, P, I, I, I, P],
        "bw_gemm_fp8": [P, P, P, P, P, I, I, I, I, P],
        "bw_gemm_mxfp4": [P, P, P, P, P, P, P, I, I, I, I, P],
        "bw_gemm_fp4": [P, P, P, P, P, I, I, I, I, P],
        "bw_quantize_f16": [P, P, LL, P],
        "bw_quantize_fp8": [P, P, P, I, I, I, I, P],
        "bw_quantize_fp8_noalloc": [P, P, P, I, I, I, I, P],
        "bw_quantize_fp4": [P, P, P, I, I, I, I, I, P],
        "bw_quantize_mxfp4": [P, P, P, I, I, I, I, P],
        "bw_rmsnorm": [P, LL, P, LL, P, I, I, F, P, LL, P, LL, P, I, I, P],
        "bw_rmsnorm_fp8": [P, LL, P, LL, P, I, I, F, P, LL, P, P, LL, P, I, I, P],
        "bw_rmsnorm_backward": [P, LL, P, LL, P, I, I, P, P, LL, P, LL, P, P, SZ, I, I, P],
        "bw_gemm_grouped": [I, P, LL, P, I, P, I, P, P, P, LL, I, I, I, I, P],
        "bw_gemm_grouped_wgrad": [I, P, LL, P, LL, P, I, P, I, I, I, I, P],
        "bw_unshard_columns": [P, P, I, I, I, P],
        "bw_unshard_columns_bf16": [P, P, I, I, I, P],
        "bw_gemm_sharded": [I, I, P, I, I, I, I, I],
        "bw_gemm_f16_allgather": [P, P, P, P, I, I, I, I, I, P],
        "bw_gemm_fp8_allgather": [P, P, P, P, P, I, P, I, I, I, I, I, P],
        "bw_gemm_f16_allgather_multicast": [P, P, P, I, I, I, I, I, P],
        "bw_gemm_fp8_allgather_multicast": [P, P, P, P, P, I, I, I, I, I, I, P],
        "bw_ipc_malloc": [ctypes.c_size_t, P, P],
        "bw_ipc_free": [P],
        "bw_ipc_open": [P, P],
        "bw_ipc_close": [P],
    }
    for name, args in sig.items():
        f = getattr(L, name)
        f.argtypes = args
        f.restype = I
    L.bw_last_error_string.argtypes = []
    L.bw_last_error_string.restype = ctypes.c_char_p
    L.bw_sf_bytes.argtypes = [I, I]
    L.bw_sf_bytes.restype = ctypes.c_size_t
    L.bw_rmsnorm_backward_workspace.argtypes = [I, I]
    L.bw_rmsnorm_backward_workspace.restype = ctypes.c_size_t
    L.bw_sf_offset.argtypes = [I, I, I]
    L.bw_sf_offset.restype = ctypes.c_size_t
    _lib = L
    return L


def _check(rc: int) -> None:
    if rc != BW_OK:
        raise BwError(rc, lib().bw_last_error_string().decode(errors="replace"))


def _ptr(t) -> int | None:
    if t is None:
        return None
    return t.data_ptr()


def _stream(stream) -> int | None:
    import torch

    if stream is None:
        return torch.cuda.current_stream().cuda_stream
    if isinstance(stream, int):
        return stream
    return stream.cuda_stream


# ------------------------------------------------------------------ runtime
def init(device: int = 0) -> None:
    _check(lib().bw_init(device))


def device_status(stream=None) -> int:
    out = ctypes.c_int(0)
    rc = lib().bw_device_status(_stream(stream), ctypes.byref(out))
    if rc not in (BW_OK, BW_ERR_TIMEOUT):
        _check(rc)
    return out.value


def set_wait_budget_ns(ns: int) -> None:
    _check(lib().bw_set_wait_budget_ns(int(ns)))


def set_trace_buffer(buf=None) -> None:
    """Arm the per-CTA wait-time trace with a torch int64 CUDA tensor of shape (ctas, 8)."""
    if buf is None:
        _check(lib().bw_set_trace_buffer(None, 0))
    else:
        _check(lib().bw_set_trace_buffer(buf.data_ptr(), buf.shape[0]))


def sf_bytes(outer: int, K: int) -> int:
    return int(lib().bw_sf_bytes(outer, K))


# ------------------------------------------------------------------ GEMMs
def gemm_f16(A, B, C=None, stream=None, b_transposed: bool = False):
    """C (fp32) = A (fp16 MxK) x B (fp16 KxN, or NxK when b_transposed)."""
    import torch

    M, K = A.shape
    N = B.shape[0] if b_transposed else B.shape[1]
    if C is None:
        C = torch.empty((M, N), dtype=torch.float32, device=A.device)
    fn = lib().bw_gemm_f16_bt if b_transposed else lib().bw_gemm_f16
    _check(fn(_ptr(A), _ptr(B), _ptr(C), M, N, K, _stream(stream)))
    return C


def gemm_fp8(A, Bt, scale_a=None, scale_b=None, C=None, out_dtype=OUT_BF16, stream=None):
    """C = (A (e4m3 MxK) x Bt^T (e4m3 NxK)) * scale_a * scale_b."""
    import torch

    M, K = A.shape
    N = Bt.shape[0]
    if C is None:
        C = torch.empty((M, N), dtype=torch.bfloat16 if out_dtype == OUT_BF16 else torch.float32, device=A.device)
    _check(lib().bw_gemm_fp8(_ptr(A), _ptr(Bt), _ptr(scale_a), _ptr(scale_b), _ptr(C), out_dtype, M, N, K,
                             _stream(stream)))
    return C


def gemm_mxfp4(A, Bt, sfa, sfb, K: int, scale_a=None, scale_b=None, C=None, out_dtype=OUT_BF16, stream=None):
    import torch

    M, N = A.shape[0], Bt.shape[0]
    if C is None:
        C = torch.empty((M, N), dtype=torch.bfloat16 if out_dtype == OUT_BF16 else torch.float32, device=A.device)
    _check(lib().bw_gemm_mxfp4(_ptr(A), _ptr(Bt), _ptr(sfa), _ptr(sfb), _ptr(scale_a), _ptr(scale_b), _ptr(C),
                               out_dtype, M, N, K, _stream(stream)))
    return C


def gemm_fp4(A, Bt, K: int, scale_a=None, scale_b=None, C=None, out_dtype=OUT_BF16, stream=None):
    import torch

    M, N = A.shape[0], Bt.shape[0]
    if C is None:
        C = torch.empty((M, N), dtype=torch.bfloat16 if out_dtype == OUT_BF16 else torch.float32, device=A.device)
    _check(lib().bw_gemm_fp4(_ptr(A), _ptr(Bt), _ptr(scale_a), _ptr(scale_b), _ptr(C), out_dtype, M, N, K,
                             _stream(stream)))
    return C


# ------------------------------------------------------------------ quantisers
def quantize_f16(src, dst=None, stream=None):
    import torch

    if dst is None:
        dst = torch.empty(src.shape, dtype=torch.float16, device=src.device)
    _check(lib().bw_quantize_f16(_ptr(src), _ptr(dst), src.numel(), _stream(stream)))
    return dst


def quantize_fp8(src, transpose=False, scale_mode=SCALE_AMAX, dst=None, scale_out=None, stream=None):
    import torch

    rows, cols = src.shape
    if dst is None:
        dst = torch.empty((cols, rows) if transpose else (rows, cols), dtype=torch.uint8, device=src.device)
    if scale_out is None:
        scale_out = torch.empty(1, dtype=torch.float32, device=src.device)
    _check(lib().bw_quantize_fp8(_ptr(src), _ptr(dst), _ptr(scale_out), rows, cols, int(transpose), scale_mode,
                                 _stream(stream)))
    return dst, scale_out


def quantize_fp8_noalloc(src, transpose=False, scale_mode=SCALE_AMAX, dst=None, scale_out=None, stream=None):
    """bw_quantize_fp8 through the entry point that allocates nothing (fixed library scratch).
    `dst` and `scale_out` must be supplied by callers that cannot allocate; the defaults here
    allocate them with torch for convenience."""
    import torch

    rows, cols = src.shape
    if dst is None:
        dst = torch.empty((cols, rows) if transpose else (rows, cols), dtype=torch.uint8, device=src.device)
    if scale_out is None:
        scale_out = torch.empty(1, dtype=torch.float32, device=src.device)
    _check(lib().bw_quantize_fp8_noalloc(_ptr(src), _ptr(dst), _ptr(scale_out), rows, cols, int(transpose),
                                         scale_mode, _stream(stream)))
    return dst, scale_out


def quantize_fp4(src, transpose=False, scale_mode=SCALE_AMAX, container=FP4_PACKED, dst=None, scale_out=None,
                 stream=None):
    import torch

    rows, cols = src.shape
    orows, ocols = (cols, rows) if transpose else (rows, cols)
    if dst is None:
        dst = torch.empty((orows, ocols if container == FP4_BYTE_SHL2 else ocols // 2), dtype=torch.uint8,
                          device=src.device)
    if scale_out is None:
        scale_out = torch.empty(1, dtype=torch.float32, device=src.device)
    _check(lib().bw_quantize_fp4(_ptr(src), _ptr(dst), _ptr(scale_out), rows, cols, int(transpose), scale_mode,
                                 container, _stream(stream)))
    return dst, scale_out


def quantize_mxfp4(src, transpose=False, mode=MX_BLOCK32, dst=None, sf=None, stream=None):
    import torch

    rows, cols = src.shape
    K, outer = (rows, cols) if transpose else (cols, rows)
    if dst is None:
        dst = torch.empty((outer, K // 2), dtype=torch.uint8, device=src.device)
    if sf is None:
        sf = torch.empty(sf_bytes(outer, K), dtype=torch.uint8, device=src.device)
    _check(lib().bw_quantize_mxfp4(_ptr(src), _ptr(dst), _ptr(sf), rows, cols, int(transpose), mode,
                                   _stream(stream)))
    return dst, sf


# ------------------------------------------------------------------ operands of the calls below
# The wrappers below are called once or twice a layer on a few rows, where their own time counts:
# checks compare without building anything, and outputs come from the cheapest allocation call.
_type_codes = {}  # torch dtype -> (BW_DTYPE_*); filled on first use, torch being imported lazily


def _codes():
    if not _type_codes:
        import torch

        _type_codes.update({torch.float32: DTYPE_F32, torch.float16: DTYPE_F16, torch.bfloat16: DTYPE_BF16,
                             torch.uint8: DTYPE_FP8})
    return _type_codes


def _dtype_code(t, what: str, allowed: tuple[int, ...]) -> int:
    code = _codes().get(t.dtype, -1)
    if code not in allowed:
        names = " or ".join(str(k) for k, v in _codes().items() if v in allowed)
        raise TypeError(f"{what} must be {names}, not {t.dtype}")
    return code


_INT_MAX = 2 ** 31 - 1  # ctypes would pass on the low 32 bits of more


def _too_large(*sizes):
    raise ValueError(f"a size of {max(sizes)} exceeds {_INT_MAX}")


def _refuse(what: str, t, shape, dtype, dev: int):
    if t.dtype != dtype:
        raise TypeError(f"{what} must be {dtype}, not {t.dtype}")
    if tuple(t.shape) != tuple(shape):
        raise ValueError(f"{what} has shape {tuple(t.shape)}, expected {tuple(shape)}")
    if t.get_device() != dev:
        raise ValueError(f"{what} is on {t.device}, the other operands are on cuda:{dev}")
    raise ValueError(f"{what} must be contiguous (strides {t.stride()})")


def _rows(what: str, t, shape, dtype, dev: int) -> int:
    """Row pitch of a 2-D operand with contiguous rows."""
    if t.dtype is not dtype or t.shape != shape or t.get_device() != dev:
        _refuse(what, t, shape, dtype, dev)
    ld, step = t.stride()
    if step != 1 and shape[1] > 1:
        _refuse(what, t, shape, dtype, dev)
    return ld if shape[0] > 1 else shape[1]


def _flat(what: str, t, shape, dtype, dev: int) -> None:
    if t.dtype is not dtype or t.shape != shape or t.get_device() != dev or not t.is_contiguous():
        _refuse(what, t, shape, dtype, dev)


_NO_SCOPE = contextlib.nullcontext()


def _scope(t, stream):
    """Makes the operands' device and `stream` current: what a call allocates belongs to the stream
    that it runs on."""
    import torch

    dev = t.get_device()
    if dev < 0:
        raise ValueError(f"operands must be on a CUDA device, not {t.device}")
    if stream is None:
        return _NO_SCOPE if dev == torch.cuda.current_device() else torch.cuda.device(dev)
    if isinstance(stream, int):
        stream = torch.cuda.ExternalStream(stream, device=dev)
    if stream.device.index != dev:
        raise ValueError(f"stream is of {stream.device}, operands are on cuda:{dev}")
    return torch.cuda.stream(stream)


def _current_stream(dev: int) -> int:
    import torch

    raw = getattr(torch._C, "_cuda_getCurrentRawStream", None)  # the handle alone, without a Stream object
    return raw(dev) if raw is not None else torch.cuda.current_stream(dev).cuda_stream


# ------------------------------------------------------------------ root-mean-square norm
_NORM_TYPES = (DTYPE_F32, DTYPE_F16, DTYPE_BF16)


def _norm_operands(x, weight, residual):
    if x.dim() != 2 or weight.dim() != 1:
        raise ValueError(f"rmsnorm takes x (rows x cols) and weight (cols), not {x.dim()}-D and {weight.dim()}-D")
    dtype, shape, dev = x.dtype, x.shape, x.get_device()
    if shape[0] > _INT_MAX or shape[1] > _INT_MAX:
        _too_large(*shape)
    code = _dtype_code(x, "x", _NORM_TYPES)
    wtype = weight.dtype
    if wtype is not dtype and _codes().get(wtype) != DTYPE_F32:
        raise TypeError(f"weight must be {dtype} or torch.float32, not {wtype}")
    _flat("weight", weight, shape[1:], wtype, dev)
    ldx = _rows("x", x, shape, dtype, dev)
    ldr = _rows("residual", residual, shape, dtype, dev) if residual is not None else 0
    return code, code if wtype is dtype else DTYPE_F32, dtype, shape, dev, ldx, ldr


def _norm_outputs(x, shape, dtype, dev, residual, h, rstd):
    """(h, its pitch, the h to be written or None, rstd)."""
    import torch

    if rstd is None:
        rstd = torch.empty_strided((shape[0],), (1,), dtype=torch.float32, device=x.device)
    else:
        _flat("rstd", rstd, shape[:1], torch.float32, dev)
    if h is None:
        if residual is None:
            return x, 0, None, rstd
        h = torch.empty_strided(shape, (shape[1], 1), dtype=dtype, device=x.device)
        return h, shape[1], h, rstd
    return h, _rows("h", h, shape, dtype, dev), h, rstd


def rmsnorm(x, weight, residual=None, eps: float = 1e-6, y=None, h=None, rstd=None, stream=None):
    """y = norm(h) * weight with h = x + residual (x without one); returns (y, h, rstd).

    x, residual, y, h: rows x cols of float32, float16 or bfloat16 with contiguous rows; weight of
    the same type or float32. h (x itself where there is no residual) and rstd are what
    rmsnorm_backward takes. y and h may each be x's or the residual's own tensor, not both the same one.
    Where y is written over x without a residual, x no longer holds h: the h returned is None unless one is given."""
    import torch

    code, wcode, dtype, shape, dev, ldx, ldr = _norm_operands(x, weight, residual)
    with _scope(x, stream):
        h, ldh, hout, rstd = _norm_outputs(x, shape, dtype, dev, residual, h, rstd)
        if y is None:
            ldy = shape[1]
            y = torch.empty_strided(shape, (ldy, 1), dtype=dtype, device=x.device)
        else:
            ldy = _rows("y", y, shape, dtype, dev)
        _check(lib().bw_rmsnorm(x.data_ptr(), ldx, _ptr(residual), ldr, weight.data_ptr(), code, wcode, eps,
                                y.data_ptr(), ldy, _ptr(hout), ldh, rstd.data_ptr(), shape[0], shape[1],
                                _current_stream(dev)))
    if h is x and hout is None and y.data_ptr() == x.data_ptr() and shape[0] > 0:  # (of no rows all pointers are null)
        h = None
    return y, h, rstd


def rmsnorm_fp8(x, weight, residual=None, eps: float = 1e-6, q=None, row_scale=None, h=None, rstd=None, stream=None):
    """rmsnorm with E4M3 output: q (uint8 codes) and row_scale (float32, one a row) with
    y = q * row_scale, as gemm_grouped takes them; returns (q, row_scale, h, rstd)."""
    import torch

    code, wcode, dtype, shape, dev, ldx, ldr = _norm_operands(x, weight, residual)
    with _scope(x, stream):
        h, ldh, hout, rstd = _norm_outputs(x, shape, dtype, dev, residual, h, rstd)
        if q is None:
            ldq = shape[1]
            q = torch.empty_strided(shape, (ldq, 1), dtype=torch.uint8, device=x.device)
        else:
            ldq = _rows("q", q, shape, torch.uint8, dev)
        if row_scale is None:
            row_scale = torch.empty_strided((shape[0],), (1,), dtype=torch.float32, device=x.device)
        else:
            _flat("row_scale", row_scale, shape[:1], torch.float32, dev)
        _check(lib().bw_rmsnorm_fp8(x.data_ptr(), ldx, _ptr(residual), ldr, weight.data_ptr(), code, wcode, eps,
                                    q.data_ptr(), ldq, row_scale.data_ptr(), _ptr(hout), ldh, rstd.data_ptr(),
                                    shape[0], shape[1], _current_stream(dev)))
    return q, row_scale, h, rstd


@functools.lru_cache(maxsize=256)
def rmsnorm_backward_workspace(rows: int, cols: int) -> int:
    """Bytes of workspace that rmsnorm_backward needs for these sizes."""
    if rows > _INT_MAX or cols > _INT_MAX:
        _too_large(rows, cols)
    return int(lib().bw_rmsnorm_backward_workspace(rows, cols))


def rmsnorm_backward(dy, h, weight, rstd, dresidual=None, dx=None, dweight=None, workspace=None, stream=None):
    """Gradient of rmsnorm from the h and rstd it returned: (dx, dweight). dx is the gradient of x
    and of the residual alike, with dresidual (the gradient that reached h past the norm) added;
    dweight is float32. dx may be dy's, h's or dresidual's own tensor. `workspace`: uint8 tensor of
    rmsnorm_backward_workspace(rows, cols) bytes; one of the call's own where None."""
    import torch

    code, wcode, dtype, shape, dev, ldh, lddr = _norm_operands(h, weight, dresidual)
    lddy = _rows("dy", dy, shape, dtype, dev)
    _flat("rstd", rstd, shape[:1], torch.float32, dev)
    with _scope(h, stream):
        if dx is None:
            lddx = shape[1]
            dx = torch.empty_strided(shape, (lddx, 1), dtype=dtype, device=h.device)
        else:
            lddx = _rows("dx", dx, shape, dtype, dev)
        if dweight is None:
            dweight = torch.empty_strided((shape[1],), (1,), dtype=torch.float32, device=h.device)
        else:
            _flat("dweight", dweight, shape[1:], torch.float32, dev)
        if workspace is None:
            nbytes = rmsnorm_backward_workspace(*shape)
            workspace = torch.empty_strided((nbytes,), (1,), dtype=torch.uint8, device=h.device)
        else:
            nbytes = workspace.numel()
            _flat("workspace", workspace, (nbytes,), torch.uint8, dev)
        _check(lib().bw_rmsnorm_backward(dy.data_ptr(), lddy, h.data_ptr(), ldh, weight.data_ptr(), code, wcode,
                                         rstd.data_ptr(), _ptr(dresidual), lddr, dx.data_ptr(), lddx,
                                         dweight.data_ptr(), workspace.data_ptr(), nbytes, shape[0], shape[1],
                                         _current_stream(dev)))
    return dx, dweight


# ------------------------------------------------------------------ products grouped by expert
def _out_type(out_dtype: int):
    import torch

    if out_dtype == OUT_BF16:
        return torch.bfloat16
    if out_dtype == OUT_F32:
        return torch.float32
    raise ValueError(f"out_dtype must be OUT_F32 or OUT_BF16, not {out_dtype}")


def _groups(offsets, dev: int) -> int:
    import torch

    if offsets.dim() != 1 or offsets.shape[0] < 2:
        raise ValueError(f"offsets must hold groups + 1 ints, not a tensor of shape {tuple(offsets.shape)}")
    if offsets.shape[0] > _INT_MAX:
        _too_large(offsets.shape[0])
    _flat("offsets", offsets, offsets.shape, torch.int32, dev)
    return offsets.shape[0] - 1


def gemm_grouped(A, B, offsets, C=None, b_transposed: bool = False, row_scale=None, group_scale=None,
                 out_dtype=OUT_BF16, stream=None):
    """C[r] = (A[r] x B[g]) * row_scale[r] * group_scale[g] for offsets[g] <= r < offsets[g + 1].

    A: rows x K float16, bfloat16 or uint8 (E4M3 codes); B: groups x K x N, or groups x N x K with
    b_transposed (E4M3: only that). offsets: groups + 1 int32 on the device. The product with the
    other layout of B is the input gradient. Rows outside offsets[0]..offsets[groups] are left as
    they were (a C allocated here holds arbitrary values there)."""
    import torch

    if A.dim() != 2 or B.dim() != 3:
        raise ValueError(f"gemm_grouped takes A (rows x K) and B (groups x K x N), not {A.dim()}-D and {B.dim()}-D")
    code = _dtype_code(A, "A", (DTYPE_F16, DTYPE_BF16, DTYPE_FP8))
    (rows, K), dev = A.shape, A.get_device()
    N = B.shape[1] if b_transposed else B.shape[2]
    if rows > _INT_MAX or K > _INT_MAX or N > _INT_MAX:
        _too_large(rows, K, N)
    groups = _groups(offsets, dev)
    _flat("B", B, (groups, N, K) if b_transposed else (groups, K, N), A.dtype, dev)
    lda = _rows("A", A, A.shape, A.dtype, dev)
    if row_scale is not None:
        _flat("row_scale", row_scale, (rows,), torch.float32, dev)
    if group_scale is not None:
        _flat("group_scale", group_scale, (groups,), torch.float32, dev)
    otype = _out_type(out_dtype)
    with _scope(A, stream):
        if C is None:
            ldc = N
            C = torch.empty_strided((rows, N), (N, 1), dtype=otype, device=A.device)
        else:
            ldc = _rows("C", C, (rows, N), otype, dev)
        _check(lib().bw_gemm_grouped(code, A.data_ptr(), lda, B.data_ptr(), int(b_transposed), offsets.data_ptr(),
                                     groups, _ptr(row_scale), _ptr(group_scale), C.data_ptr(), ldc, out_dtype, rows,
                                     N, K, _current_stream(dev)))
    return C


def gemm_grouped_wgrad(X, Y, offsets, D=None, out_dtype=OUT_F32, stream=None):
    """D[g] = X[rows of g]^T x Y[rows of g], zeros for a group without rows: the weight gradient of
    gemm_grouped (X = A, Y = dC for a groups x K x N matrix; X = dC, Y = A for groups x N x K).
    X: rows x M, Y: rows x N, both float16 or both bfloat16; D: groups x M x N."""
    import torch

    if X.dim() != 2 or Y.dim() != 2:
        raise ValueError(f"gemm_grouped_wgrad takes X (rows x M) and Y (rows x N), not {X.dim()}-D and {Y.dim()}-D")
    code = _dtype_code(X, "X", (DTYPE_F16, DTYPE_BF16))
    (rows, M), N, dev = X.shape, Y.shape[1], X.get_device()
    if rows > _INT_MAX or M > _INT_MAX or N > _INT_MAX:
        _too_large(rows, M, N)
    groups = _groups(offsets, dev)
    ldx = _rows("X", X, X.shape, X.dtype, dev)
    ldy = _rows("Y", Y, (rows, N), X.dtype, dev)
    otype = _out_type(out_dtype)
    with _scope(X, stream):
        if D is None:
            D = torch.empty_strided((groups, M, N), (M * N, N, 1), dtype=otype, device=X.device)
        else:
            _flat("D", D, (groups, M, N), otype, dev)
        _check(lib().bw_gemm_grouped_wgrad(code, X.data_ptr(), ldx, Y.data_ptr(), ldy, offsets.data_ptr(), groups,
                                           D.data_ptr(), out_dtype, rows, M, N, _current_stream(dev)))
    return D


def unshard_columns(C_shardmajor, M: int, N: int, world: int, out=None, stream=None):
    """[world][M][N/world] -> row-major M x N on the device; FP32 or BF16 elements."""
    import torch

    if C_shardmajor.dtype not in (torch.float32, torch.bfloat16):
        raise TypeError(f"unshard_columns takes float32 or bfloat16, not {C_shardmajor.dtype}")
    if C_shardmajor.numel() != M * N:
        raise ValueError(f"shard-major buffer holds {C_shardmajor.numel()} elements, expected {M} x {N}")
    if out is None:
        out = torch.empty((M, N), dtype=C_shardmajor.dtype, device=C_shardmajor.device)
    if out.dtype != C_shardmajor.dtype or out.numel() != M * N:
        raise ValueError("out must match the input's dtype and hold M x N elements")
    fn = lib().bw_unshard_columns if C_shardmajor.dtype == torch.float32 else lib().bw_unshard_columns_bf16
    _check(fn(_ptr(C_shardmajor), _ptr(out), M, N, world, _stream(stream)))
    return out


def gemm_sharded(dtype: int, parts: list[dict], M: int, N: int, K: int, out_dtype: int = OUT_F32,
                 gather: bool = False) -> None:
    """One process, len(parts) GPUs: parts[r] = {"A", "B", "C", optional "sfA", "sfB", "scale_a",
    "scale_b", "C_gathered", "stream"} with torch tensors on the shard's device (B is the shard
    of columns r*N/g .. (r+1)*N/g in the layout of the dtype's single-GPU call). Enqueues the
    shards' GEMMs and, with gather, the NCCL all-gather + unshard into every C_gathered."""
    import torch

    arr = (Shard * max(1, len(parts)))()
    for r, part in enumerate(parts):
        dev = part["C"].device.index if part.get("C") is not None else 0
        st = part.get("stream")
        if st is None:
            st = torch.cuda.current_stream(dev)
        arr[r] = Shard(dev, _ptr(part.get("A")), _ptr(part.get("B")), _ptr(part.get("sfA")), _ptr(part.get("sfB")),
                       _ptr(part.get("scale_a")), _ptr(part.get("scale_b")), _ptr(part.get("C")),
                       _ptr(part.get("C_gathered")), _stream(st))
    _check(lib().bw_gemm_sharded(dtype, out_dtype, ctypes.cast(arr, ctypes.c_void_p) if parts else None,
                                 len(parts), M, N, K, int(gather)))


# ------------------------------------------------------------------ fused all-gather (IPC)
IPC_HANDLE_BYTES = 64


class IpcBuffer:
    """A device buffer other processes can map (CUDA IPC). `tensor` views it as a torch tensor
    (through __cuda_array_interface__, no copy); `handle` is the 64-byte IPC handle."""

    def __init__(self, shape, dtype, device):
        import math

        import torch

        self.shape, self.dtype = tuple(shape), dtype
        nbytes = math.prod(self.shape) * torch.empty((), dtype=dtype).element_size()
        ptr = ctypes.c_void_p()
        h = ctypes.create_string_buffer(IPC_HANDLE_BYTES)
        with torch.cuda.device(device):
            _check(lib().bw_ipc_malloc(nbytes, ctypes.byref(ptr), h))
        self.ptr, self.handle, self.device = ptr.value, h.raw, torch.device(device)
        typestr = {torch.float32: "<f4", torch.bfloat16: "<i2", torch.float16: "<f2"}[dtype]
        self.__cuda_array_interface__ = {"shape": self.shape, "typestr": typestr, "data": (self.ptr, False),
                                         "version": 3, "strides": None}
        t = torch.as_tensor(self, device=self.device)
        self.tensor = t.view(dtype) if dtype == torch.bfloat16 else t

    def close(self):
        if self.ptr:
            _check(lib().bw_ipc_free(self.ptr))
            self.ptr = None


def ipc_open(handle: bytes, device) -> int:
    import torch

    ptr = ctypes.c_void_p()
    with torch.cuda.device(device):
        _check(lib().bw_ipc_open(ctypes.create_string_buffer(handle, IPC_HANDLE_BYTES), ctypes.byref(ptr)))
    return ptr.value


def ipc_close(ptr: int) -> None:
    _check(lib().bw_ipc_close(ptr))


def _peer_array(peers):
    return (ctypes.c_void_p * len(peers))(*[p or 0 for p in peers])


def gemm_f16_allgather(A, B_shard, C_full, peers, rank: int, stream=None):
    """This rank's columns of C_full = A x B_shard, stored locally and into every peer's C_full
    (peers[q] = rank q's buffer mapped here; entry [rank] ignored)."""
    M, K = A.shape
    world = len(peers)
    _check(lib().bw_gemm_f16_allgather(_ptr(A), _ptr(B_shard), _ptr(C_full), _peer_array(peers), world, rank, M,
                                       C_full.shape[1], K, _stream(stream)))


def gemm_fp8_allgather(A, Bt_shard, scale_a, scale_b, C_full, peers, rank: int, out_dtype=OUT_BF16, stream=None):
    M, K = A.shape
    world = len(peers)
    _check(lib().bw_gemm_fp8_allgather(_ptr(A), _ptr(Bt_shard), _ptr(scale_a), _ptr(scale_b), _ptr(C_full),
                                       out_dtype, _peer_array(peers), world, rank, M, C_full.shape[1], K,
                                       _stream(stream)))


def gemm_f16_allgather_multicast(A, B_shard, mc_ptr: int, world: int, rank: int, N_total: int, stream=None):
    """This rank's columns of the M x N_total product, written once through the multicast
    address `mc_ptr` (every rank's buffer bound to one NVLink multicast object) and so into
    every rank's C."""
    M, K = A.shape
    _check(lib().bw_gemm_f16_allgather_multicast(_ptr(A), _ptr(B_shard), mc_ptr, world, rank, M, N_total, K,
                                                 _stream(stream)))


def gemm_fp8_allgather_multicast(A, Bt_shard, scale_a, scale_b, mc_ptr: int, world: int, rank: int, N_total: int,
                                 out_dtype=OUT_BF16, stream=None):
    M, K = A.shape
    _check(lib().bw_gemm_fp8_allgather_multicast(_ptr(A), _ptr(Bt_shard), _ptr(scale_a), _ptr(scale_b), mc_ptr,
                                                 out_dtype, world, rank, M, N_total, K, _stream(stream)))
