"""Python binding of libreng_hip.so (include/reng_hip.h) over ctypes.

The names follow the reference's reng-fp8 API (crates/reng-fp8/src/lib.rs):
`quantize_with`, `quantize`, `encode`, `decode`, `row_absmax`, `row_errors`,
`sample_row_errors`, `choose_exp_bias`, `Quantized.dequantize`, and the
consumer `gemm_w8a16` / `gemm_fp8_scaled` (crates/reng-synapse/src/fp8.rs).

Device work takes torch tensors that live on the GPU (torch is only the
allocator and the stream here) and runs on torch's current stream. There is no
CPU path: if the library is missing or a call fails, this module raises.
Argument errors that reng-fp8 turns into panics (lib.rs:527-532) raise
`ValueError` with the library's message.
"""
import ctypes
import operator
import os

HERE = os.path.dirname(os.path.abspath(__file__))
LIB_PATH = os.path.join(HERE, "lib", "libreng_hip.so")

OK, EINVAL, EDEVICE, ENOMEM, EUNSUPPORTED = 0, 1, 2, 3, 4
E4M3, E5M2 = 0, 1
PCS, HW, UNIT = 0, 1, 2
BF16, F32 = 0, 1
DEFAULT_BACKOFF = 1.0

FORMAT_NAMES = {"e4m3": E4M3, "fp8_143": E4M3, "hf8": E4M3, "e5m2": E5M2, "fp8_152": E5M2, "f8": E5M2}
SCALING_NAMES = {"pcs": PCS, "per-channel": PCS, "perchannel": PCS, "hw": HW, "hw-exp-bias": HW,
                 "expbias": HW, "unit": UNIT, "none": UNIT}
MAX_FINITE = {E4M3: 240.0, E5M2: 57344.0}
EXPONENT_BIAS = {E4M3: 7, E5M2: 15}


class RengHipError(RuntimeError):
    pass


class _Matrix(ctypes.Structure):
    _fields_ = [("w", ctypes.c_void_p), ("codes", ctypes.c_void_p), ("scales", ctypes.c_void_p),
                ("exp_bias", ctypes.c_void_p), ("rows", ctypes.c_size_t), ("cols", ctypes.c_size_t),
                ("ld", ctypes.c_size_t)]


class _MxCache(ctypes.Structure):
    _fields_ = [("k_codes", ctypes.c_void_p), ("k_scales", ctypes.c_void_p), ("v_codes", ctypes.c_void_p),
                ("v_scales", ctypes.c_void_p), ("n_kv_heads", ctypes.c_size_t), ("head_dim", ctypes.c_size_t),
                ("capacity", ctypes.c_size_t)]


class _Rope(ctypes.Structure):
    _fields_ = [("sin_table", ctypes.c_void_p), ("cos_table", ctypes.c_void_p), ("table_rows", ctypes.c_size_t),
                ("rot_dim", ctypes.c_size_t), ("axes", ctypes.c_size_t), ("pair_axis", ctypes.c_char_p)]


_lib = None
_P, _SZ, _I, _F, _U32 = ctypes.c_void_p, ctypes.c_size_t, ctypes.c_int, ctypes.c_float, ctypes.c_uint32

SIGNATURES = {
    "reng_hip_version": (ctypes.c_char_p, []),
    "reng_hip_last_error": (ctypes.c_char_p, []),
    "reng_hip_device_info": (_I, [ctypes.c_char_p, _SZ]),
    "reng_hip_quantize": (_I, [_P, _I, _SZ, _SZ, _SZ, _I, _I, _F, _P, _P, _P, _P]),
    "reng_hip_quantize_host": (_I, [_P, _I, _SZ, _SZ, _I, _I, _F, _P, _P, _P]),
    "reng_hip_quantize_batch": (_I, [ctypes.POINTER(_Matrix), _SZ, _I, _I, _I, _F, _P]),
    "reng_hip_row_absmax": (_I, [_P, _I, _SZ, _SZ, _SZ, _P, _P]),
    "reng_hip_choose_exp_bias": (_U32, [_F, _I]),
    "reng_hip_encode": (_I, [_P, _SZ, _I, _P, _P]),
    "reng_hip_decode": (_I, [_P, _SZ, _I, _P, _P]),
    "reng_hip_dequantize": (_I, [_P, _P, _SZ, _SZ, _I, _I, _P, _P]),
    "reng_hip_row_errors": (_I, [_P, _P, _P, _SZ, _SZ, _I, _SZ, _P, _P, _P]),
    "reng_hip_gemm_w8a16": (_I, [_P, _P, _P, _SZ, _SZ, _SZ, _I, _P, _P]),
    "reng_hip_gemm_w8a16_noalloc": (_I, [_P, _P, _P, _SZ, _SZ, _SZ, _I, _P, _P]),
    "reng_hip_gemm_fp8_scaled": (_I, [_P, _I, _P, _SZ, _P, _I, _P, _SZ, _SZ, _SZ, _SZ, _P, _P]),
    "reng_hip_quantize_blocks": (_I, [_P, _I, _SZ, _SZ, _SZ, _I, _SZ, _F, _P, _P, _P]),
    "reng_hip_gemm_fp8_blocks": (_I, [_P, _I, _P, _P, _I, _P, _SZ, _SZ, _SZ, _P, _P]),
    "reng_hip_residual_norm_bf16": (_I, [_P, _P, _P, _P, _SZ, _F, _P, _SZ, _SZ, _F, _P, _P, _P]),
    "reng_hip_residual_norm_fp8": (_I, [_P, _P, _P, _P, _SZ, _F, _P, _SZ, _SZ, _F, _I, _F, _P, _P, _P, _P]),
    "reng_hip_attention_tree_workspace_bytes": (_SZ, [_SZ, _SZ, _SZ, _SZ, _SZ]),
    "reng_hip_attention_tree": (_I, [_P, _P, _P, _SZ, _SZ, _SZ, _SZ, _SZ, _P, _F, _P, _SZ, _P, _P]),
    "reng_hip_quantize_mxfp4": (_I, [_P, _I, _SZ, _SZ, _SZ, _P, _P, _P]),
    "reng_hip_dequantize_mxfp4": (_I, [_P, _P, _SZ, _SZ, _I, _P, _P]),
    "reng_hip_gemm_mxfp4": (_I, [_P, _P, _P, _P, _SZ, _SZ, _SZ, _P, _P]),
    "reng_hip_cache_read_mxfp4": (_I, [_P, _SZ, _SZ, _P, _P, _P]),
    "reng_hip_head_norm_rope_bf16": (_I, [_P, _SZ, _P, _P, _SZ, _SZ, _SZ, _SZ, _SZ, _P, _P, _F, _P, _P, _P, _P, _P, _P]),
    "reng_hip_head_norm_rope_mxfp4": (_I, [_P, _SZ, _P, _P, _SZ, _SZ, _SZ, _P, _P, _F, _P, _P, _P, _P, _SZ, _P]),
    "reng_hip_attention_mxfp4_workspace_bytes": (_SZ, [_SZ, _SZ, _SZ, _SZ, _SZ]),
    "reng_hip_attention_mxfp4": (_I, [_P, _P, _SZ, _SZ, _SZ, _P, _F, _P, _SZ, _P, _P]),
    "reng_hip_verify_hw_convert": (_I, [_I, ctypes.POINTER(ctypes.c_uint64), ctypes.POINTER(ctypes.c_uint32)]),
    "reng_hip_rms_norm_bf16": (_I, [_P, _P, _SZ, _SZ, _F, _P, _P]),
    "reng_hip_add_rms_norm_bf16": (_I, [_P, _P, _P, _SZ, _SZ, _F, _P, _P, _P]),
    "reng_hip_gemv_w8a16_residual": (_I, [_P, _P, _P, _SZ, _SZ, _I, _P, _P, _P]),
    "reng_hip_gemv_w8a16_swiglu": (_I, [_P, _P, _P, _SZ, _SZ, _I, _P, _P]),
    "reng_hip_gemv_w8a16_rmsnorm": (_I, [_P, _P, _F, _P, _P, _SZ, _SZ, _I, _P, _P]),
    "reng_hip_gemv_w8a16_rmsnorm_swiglu": (_I, [_P, _P, _F, _P, _P, _SZ, _SZ, _I, _P, _P]),
    "reng_hip_gemv_w8a16_rmsnorm_qkv_rope": (_I, [_P, _P, _F, _P, _P, _SZ, _SZ, _SZ, _SZ, _I, _P, _P, _P, _P, _P,
                                                   _P]),
    "reng_hip_rope_append": (_I, [_P, _P, _P, _SZ, _SZ, _SZ, _P, _P, _P, _P, _P]),
    "reng_hip_attention_decode": (_I, [_P, _P, _P, _SZ, _SZ, _SZ, _SZ, _F, _P, _P]),
    "reng_hip_attention_workspace_bytes": (_SZ, [_SZ, _SZ, _SZ]),
    "reng_hip_attention_decode_split": (_I, [_P, _P, _P, _SZ, _SZ, _SZ, _SZ, _F, _P, _SZ, _P, _P]),
    "reng_hip_silu_mul_bf16": (_I, [_P, _P, _SZ, _P, _P]),
    "reng_hip_add_bf16_f32": (_I, [_P, _P, _SZ, _P, _P]),
    "reng_hip_stream_read_sink_bytes": (_SZ, []),
    "reng_hip_stream_read": (_I, [_P, _SZ, _P, _P]),
    "reng_hip_stream_narrow": (_I, [_P, _SZ, _P, _P]),
    "reng_hip_stream_stage": (_I, [_P, _P, _SZ, _SZ, _SZ, _P, _P]),
}


def lib():
    """Load libreng_hip.so (raises if it has not been built)."""
    global _lib
    if _lib is None:
        # torch ships its own HIP runtime under the same soname; loading torch
        # first makes libreng_hip.so bind to that one, so the process holds a
        # single runtime (two runtimes on one device: the second to initialise
        # finds no device).
        try:
            import torch  # noqa: F401
        except ImportError:
            pass
        if not os.path.exists(LIB_PATH):
            raise RengHipError(f"{LIB_PATH} is missing: build it with `make -C reciprocating-engine_amd`")
        L = ctypes.CDLL(LIB_PATH)
        for name, (res, args) in SIGNATURES.items():
            f = getattr(L, name)
            f.restype = res
            f.argtypes = args
        _lib = L
    return _lib


def _check(rc):
    if rc != OK:
        msg = lib().reng_hip_last_error().decode()
        if rc == EINVAL:
            raise ValueError(msg)
        raise RengHipError(f"status {rc}: {msg}")


def _fmt(f):
    if isinstance(f, str):
        if f.strip().lower() not in FORMAT_NAMES:
            raise ValueError(f"unknown format {f}")
        return FORMAT_NAMES[f.strip().lower()]
    return int(f)


def _sc(s):
    if isinstance(s, str):
        if s.strip().lower() not in SCALING_NAMES:
            raise ValueError(f"unknown scaling {s}")
        return SCALING_NAMES[s.strip().lower()]
    return int(s)


def _stream():
    import torch

    return ctypes.c_void_p(torch.cuda.current_stream().cuda_stream)


def _dev(t, what, nbytes=None):
    """The device address of a contiguous GPU tensor; with nbytes, refuse a
    tensor smaller than the bytes the C call will touch (the reference refuses
    a weight slice of the wrong length, crates/reng-fp8/src/lib.rs:528; here a
    short buffer would be read or written past its end on the device)."""
    if not t.is_cuda:
        raise ValueError(f"{what} must be a GPU tensor")
    if not t.is_contiguous():
        raise ValueError(f"{what} must be contiguous")
    if nbytes is not None:
        have = t.numel() * t.element_size()
        if have < nbytes:
            raise ValueError(f"{what} length against the shape: {have} bytes, the call touches {nbytes}")
    return ctypes.c_void_p(t.data_ptr())


def _opt(t, what, nbytes=None):
    return None if t is None else _dev(t, what, nbytes)


def _span(rows, cols, ld):
    """Elements a [rows, cols] window of row pitch ld spans."""
    return 0 if rows == 0 or cols == 0 else (rows - 1) * ld + cols


def _dtype_code(t):
    import torch

    if t.dtype in (torch.bfloat16, torch.int16, torch.uint16):
        return BF16
    if t.dtype == torch.float32:
        return F32
    raise ValueError(f"weights must be bf16 (or its bits as int16/uint16) or f32, not {t.dtype}")


def version():
    return lib().reng_hip_version().decode()


def device_info():
    buf = ctypes.create_string_buffer(512)
    _check(lib().reng_hip_device_info(buf, 512))
    return buf.value.decode()


def choose_exp_bias(absmax, fmt):
    return int(lib().reng_hip_choose_exp_bias(float(absmax), _fmt(fmt)))


class Quantized:
    """reng_fp8::Quantized (lib.rs:291-345), holding device tensors."""

    def __init__(self, format, scaling, rows, cols, codes, scales, exp_bias):
        self.format, self.scaling = format, scaling
        self.rows, self.cols = rows, cols
        self.codes, self.scales = codes, scales
        self.exp_bias = exp_bias

    def code_bytes(self):
        return self.rows * self.cols

    def scale_operand(self):
        return self.scales if _sc(self.scaling) == PCS else None

    def dequantize(self):
        import torch

        out = torch.empty(self.rows * self.cols, dtype=torch.float32, device=self.codes.device)
        _check(lib().reng_hip_dequantize(_dev(self.codes, "codes", self.rows * self.cols),
                                         _dev(self.scales, "scales", 4 * self.rows), self.rows,
                                         self.cols, _fmt(self.format), F32, _dev(out, "out"), _stream()))
        return out

    def dequantize_bf16(self):
        import torch

        out = torch.empty(self.rows * self.cols, dtype=torch.int16, device=self.codes.device)
        _check(lib().reng_hip_dequantize(_dev(self.codes, "codes", self.rows * self.cols),
                                         _dev(self.scales, "scales", 4 * self.rows), self.rows,
                                         self.cols, _fmt(self.format), BF16, _dev(out, "out"), _stream()))
        return out


def quantize_into(w, rows, cols, fmt, scaling, backoff, codes, scales, exp_bias=None, ld=None):
    """Device quantize into caller-owned tensors (no allocation)."""
    ld = cols if ld is None else ld
    dt = _dtype_code(w)
    _check(lib().reng_hip_quantize(_dev(w, "weight", _span(rows, cols, ld) * (2 if dt == BF16 else 4)), dt, rows,
                                   cols, ld, _fmt(fmt), _sc(scaling), float(backoff),
                                   _dev(codes, "codes", rows * cols), _dev(scales, "scales", 4 * rows),
                                   _opt(exp_bias, "exp_bias", 4), _stream()))


def quantize_with(w, rows, cols, fmt, scaling, backoff=DEFAULT_BACKOFF, ld=None):
    """reng_fp8::quantize_with (lib.rs:519-563) on the GPU: w is a device tensor
    of bf16 (or its int16 bits) or f32, [rows, ld] row-major."""
    import torch

    codes = torch.empty(rows * cols, dtype=torch.uint8, device=w.device)
    scales = torch.empty(rows, dtype=torch.float32, device=w.device)
    eb = torch.empty(1, dtype=torch.int32, device=w.device)
    quantize_into(w, rows, cols, fmt, scaling, backoff, codes, scales, eb, ld)
    return Quantized(fmt, scaling, rows, cols, codes, scales, int(eb.item()))


def quantize(w, rows, cols, fmt, scaling):
    return quantize_with(w, rows, cols, fmt, scaling, DEFAULT_BACKOFF)


def quantize_host(w, rows, cols, fmt, scaling, backoff=DEFAULT_BACKOFF):
    """The host-pointer entry (numpy in, numpy out), as Rust's quantize_with calls it."""
    import numpy as np

    w = np.ascontiguousarray(w)
    dt = BF16 if w.dtype == np.uint16 else F32 if w.dtype == np.float32 else None
    if dt is None:
        raise ValueError(f"weights must be uint16 (bf16 bits) or float32, not {w.dtype}")
    if rows > 0 and cols > 0 and w.size != rows * cols:   # lib.rs:528 (an empty shape is the library's refusal)
        raise ValueError(f"weight length against the shape: {w.size} elements for [{rows}, {cols}]")
    codes = np.empty(rows * cols, dtype=np.uint8)
    scales = np.empty(rows, dtype=np.float32)
    eb = ctypes.c_uint32(0)
    _check(lib().reng_hip_quantize_host(ctypes.c_void_p(w.ctypes.data), dt, rows, cols, _fmt(fmt), _sc(scaling),
                                        float(backoff), ctypes.c_void_p(codes.ctypes.data),
                                        ctypes.c_void_p(scales.ctypes.data), ctypes.byref(eb)))
    return codes, scales, int(eb.value)


def quantize_batch(mats, fmt, scaling, backoff=DEFAULT_BACKOFF):
    """mats: list of (w, rows, cols, codes, scales, exp_bias_or_None) device
    tensors, all bf16 (or its int16 bits) or all f32."""
    if not mats:
        raise ValueError("empty batch")
    dts = {_dtype_code(m[0]) for m in mats}
    if len(dts) != 1:
        raise ValueError("a batch holds one weight dtype (bf16 or f32), not a mix")
    dtype = dts.pop()
    esz = 2 if dtype == BF16 else 4
    arr = (_Matrix * len(mats))()
    for i, (w, rows, cols, codes, scales, eb) in enumerate(mats):
        arr[i] = _Matrix(_dev(w, f"weight {i}", rows * cols * esz).value, _dev(codes, f"codes {i}", rows * cols).value,
                         _dev(scales, f"scales {i}", 4 * rows).value,
                         0 if eb is None else _dev(eb, f"exp_bias {i}", 4).value, rows, cols, cols)
    _check(lib().reng_hip_quantize_batch(arr, len(mats), dtype, _fmt(fmt), _sc(scaling), float(backoff),
                                         _stream()))


def row_absmax(w, rows, cols, ld=None):
    import torch

    out = torch.empty(rows, dtype=torch.float32, device=w.device)
    ld = cols if ld is None else ld
    dt = _dtype_code(w)
    _check(lib().reng_hip_row_absmax(_dev(w, "weight", _span(rows, cols, ld) * (2 if dt == BF16 else 4)), dt, rows,
                                     cols, ld, _dev(out, "out"), _stream()))
    return out


def encode(x, fmt):
    """encode over a device f32 tensor -> uint8 codes."""
    import torch

    out = torch.empty(x.numel(), dtype=torch.uint8, device=x.device)
    _check(lib().reng_hip_encode(_dev(x, "x"), x.numel(), _fmt(fmt), _dev(out, "out"), _stream()))
    return out


def decode(codes, fmt):
    import torch

    out = torch.empty(codes.numel(), dtype=torch.float32, device=codes.device)
    _check(lib().reng_hip_decode(_dev(codes, "codes"), codes.numel(), _fmt(fmt), _dev(out, "out"), _stream()))
    return out


def _errors(w, q, max_rows):
    import torch

    n = q.rows if max_rows == 0 else min(max_rows, q.rows)
    step = -(-q.rows // n)
    k = -(-q.rows // step)
    mean = torch.empty(k, dtype=torch.float32, device=q.codes.device)
    mx = torch.empty(k, dtype=torch.float32, device=q.codes.device)
    _check(lib().reng_hip_row_errors(_dev(w, "weight", 2 * q.rows * q.cols), _dev(q.codes, "codes", q.rows * q.cols),
                                     _dev(q.scales, "scales", 4 * q.rows), q.rows,
                                     q.cols, _fmt(q.format), max_rows, _dev(mean, "mean"), _dev(mx, "max"),
                                     _stream()))
    return mean, mx


def row_errors(w, q):
    return _errors(w, q, 0)


def sample_row_errors(w, q, max_rows):
    if max_rows == 0:
        raise ValueError("max_rows must be positive")
    return _errors(w, q, max_rows)


def gemm_w8a16(x, codes, scales, M, N, K, fmt, y=None):
    """y[M, N] bf16 = x[M, K] bf16 . (decode(codes[N, K]) * scales[N])^T."""
    import torch

    if y is None:
        y = torch.empty(M * N, dtype=torch.bfloat16, device=x.device)
    _check(lib().reng_hip_gemm_w8a16(_dev(x, "x", 2 * M * K), _dev(codes, "codes", N * K),
                                     _opt(scales, "scales", 4 * N), M, N, K, _fmt(fmt),
                                     _dev(y, "y", 2 * M * N), _stream()))
    return y


def gemm_fp8_scaled(a, a_fmt, scale_a, b, b_fmt, scale_b, M, N, K, out=None):
    """gemm_fp8_scaled (crates/reng-synapse/src/fp8.rs:295-331): bf16 out[M, N]."""
    import torch

    if out is None:
        out = torch.empty(M * N, dtype=torch.bfloat16, device=a.device)
    na = 0 if scale_a is None else scale_a.numel()
    nb = 0 if scale_b is None else scale_b.numel()
    _check(lib().reng_hip_gemm_fp8_scaled(_dev(a, "a", M * K), _fmt(a_fmt), _opt(scale_a, "scale_a", 4 * na),
                                          na, _dev(b, "b", N * K), _fmt(b_fmt), _opt(scale_b, "scale_b", 4 * nb), nb,
                                          M, N, K, _dev(out, "out", 2 * M * N), _stream()))
    return out


# ---------------------------------------------------------------- block scales
# One scale per 128 x 128 block of a weight, per 1 x 128 group of an activation row.

SCALE_BLOCK = 128

# What these calls ask of torch on every call, looked up once: the module, its types by what a
# call accepts, whether tensors can be on another device than the current one, and the current
# stream's handle (torch.cuda.current_stream() builds an object around it, 2.8 us of a call's 13).
_T = None


class _Torch:
    def __init__(self):
        import torch

        self.empty, self.u8, self.f32, self.bf16 = torch.empty, torch.uint8, torch.float32, torch.bfloat16
        self.is16 = frozenset((torch.bfloat16, torch.int16, torch.uint16))
        self.is32 = frozenset((torch.int32, torch.uint32))
        self.i32 = torch.int32
        self.several = torch.cuda.device_count() > 1
        self.current_device = torch.cuda.current_device
        # Without a look at whether the GPU is initialised, which tensors on it say.
        self.device_index = getattr(torch._C, "_cuda_getDevice", torch.cuda.current_device)
        raw = getattr(torch._C, "_cuda_getCurrentRawStream", None)
        self.raw_stream = raw or (lambda i: torch.cuda.current_stream(i).cuda_stream)

    def stream(self):
        return self.raw_stream(self.device_index())


def _torch():
    global _T
    if _T is None:
        _T = _Torch()
    return _T


def _nblocks(n, of=SCALE_BLOCK):
    return -(-n // of)


def _at(t, what, n, size):
    """The device address of a contiguous tensor of at least n elements of `size` bytes on the
    current device (whose current stream the call runs on)."""
    if not (t.is_cuda and t.is_contiguous() and t.numel() * t.element_size() >= n * size):
        return _dev(t, what, n * size).value   # raises
    if _T.several and t.get_device() != _T.current_device():
        raise ValueError(f"{what} is on cuda:{t.get_device()}, the current device is cuda:{_T.current_device()}")
    return t.data_ptr()


def _f32(t, what, n):
    if t.dtype != _T.f32:
        raise ValueError(f"{what} must be f32, not {t.dtype}")
    return _at(t, what, n, 4)


def _16bit(t, what, n):
    if t.dtype not in _T.is16:
        raise ValueError(f"{what} must be bf16 (or its bits as int16/uint16), not {t.dtype}")
    return _at(t, what, n, 2)


def _8bit(t, what, n):
    if t.element_size() != 1:
        raise ValueError(f"{what} must hold one code per byte, not {t.dtype}")
    return _at(t, what, n, 1)


def quantize_blocks_into(w, rows, cols, fmt, block_rows, backoff, codes, scales, ld=None):
    """quantize_blocks into caller-owned tensors (no allocation)."""
    T = _torch()
    ld = cols if ld is None else ld
    if block_rows not in (1, SCALE_BLOCK):
        raise ValueError(f"blocks of {block_rows} rows; expected 1 or {SCALE_BLOCK}")
    dt = _dtype_code(w)
    _check(lib().reng_hip_quantize_blocks(_at(w, "weight", _span(rows, cols, ld), 2 if dt == BF16 else 4), dt, rows, cols,
                                          ld, _fmt(fmt), block_rows, backoff, _8bit(codes, "codes", rows * cols),
                                          _f32(scales, "scales", _nblocks(rows, block_rows) * _nblocks(cols)),
                                          T.stream()))


def quantize_blocks(w, rows, cols, fmt, block_rows=SCALE_BLOCK, backoff=DEFAULT_BACKOFF, ld=None):
    """(codes [rows * cols], scales [blocks]) of a device tensor of bf16 (or its
    int16 bits) or f32, [rows, ld] row-major: one scale per block of block_rows x
    128 values, block_rows 128 for weights or 1 for activation rows."""
    T, dev = _torch(), w.device
    codes = T.empty(rows * cols, dtype=T.u8, device=dev)
    scales = T.empty(_nblocks(rows, max(1, block_rows)) * _nblocks(cols), dtype=T.f32, device=dev)
    quantize_blocks_into(w, rows, cols, fmt, block_rows, backoff, codes, scales, ld)
    return codes, scales


def gemm_fp8_blocks(a, a_fmt, scale_a, b, b_fmt, scale_b, M, N, K, out=None):
    """bf16 out[M, N] of codes a [M, K] with scale_a [M, ceil(K / 128)] and codes
    b [N, K] with scale_b [ceil(N / 128), ceil(K / 128)]."""
    T = _torch()
    if out is None:
        out = T.empty(M * N, dtype=T.bf16, device=a.device)
    kb = _nblocks(K)
    _check(lib().reng_hip_gemm_fp8_blocks(_8bit(a, "a", M * K), _fmt(a_fmt), _f32(scale_a, "scale_a", M * kb),
                                          _8bit(b, "b", N * K), _fmt(b_fmt), _f32(scale_b, "scale_b", _nblocks(N) * kb),
                                          M, N, K, _16bit(out, "out", M * N), T.stream()))
    return out


def _residual_norm_args(T, x, d, gamma, rows, cols, post_gamma, gate, residual_scale, h):
    """The arguments both output forms share, h (allocated where a branch needs it) and its address."""
    n = rows * cols
    if h is None and d is not None:
        h = T.empty(n, dtype=T.f32, device=x.device)
    gate_ld = 0 if gate is None or gate.numel() == cols else cols
    args = (_f32(x, "x", n), None if d is None else _16bit(d, "d", n),
            None if post_gamma is None else _f32(post_gamma, "post_gamma", cols),
            None if gate is None else _16bit(gate, "gate", n if gate_ld else cols), gate_ld, residual_scale,
            _f32(gamma, "gamma", cols), rows, cols)
    return args, h, None if h is None else _f32(h, "h", n)


def residual_norm_bf16(x, d, gamma, rows, cols, eps, post_gamma=None, gate=None, residual_scale=1.0, h=None, out=None):
    """(h, out): h = x + residual_scale * gate * rms_norm(d) * post_gamma (f32; the
    post-norm where post_gamma is given, the gate of [cols] or [rows, cols] bf16
    values where it is) and bf16 out = rms_norm(h) * gamma. h may be x. With d None
    there is no branch: h = x, returned as given."""
    T = _torch()
    if out is None:
        out = T.empty(rows * cols, dtype=T.bf16, device=x.device)
    args, h, hp = _residual_norm_args(T, x, d, gamma, rows, cols, post_gamma, gate, residual_scale, h)
    _check(lib().reng_hip_residual_norm_bf16(*args, eps, hp, _16bit(out, "out", rows * cols), T.stream()))
    return h, out


def residual_norm_fp8(x, d, gamma, rows, cols, eps, fmt, post_gamma=None, gate=None, residual_scale=1.0,
                      backoff=DEFAULT_BACKOFF, h=None, codes=None, scales=None):
    """(h, codes, scales): residual_norm_bf16 with the normalised rows as fp8 codes
    and one scale per 128 columns, gemm_fp8_blocks' a operand."""
    T = _torch()
    kb = _nblocks(cols)
    if codes is None:
        codes = T.empty(rows * cols, dtype=T.u8, device=x.device)
    if scales is None:
        scales = T.empty(rows * kb, dtype=T.f32, device=x.device)
    args, h, hp = _residual_norm_args(T, x, d, gamma, rows, cols, post_gamma, gate, residual_scale, h)
    _check(lib().reng_hip_residual_norm_fp8(*args, eps, _fmt(fmt), backoff, hp, _8bit(codes, "codes", rows * cols),
                                            _f32(scales, "scales", rows * kb), T.stream()))
    return h, codes, scales


def attention_tree_workspace_bytes(n_heads, n_kv_heads, head_dim, length, tokens):
    """Device workspace attention_tree needs for up to `length` context rows and `tokens` tokens."""
    return lib().reng_hip_attention_tree_workspace_bytes(n_heads, n_kv_heads, head_dim, length, tokens)


def attention_tree(q, k_cache, v_cache, n_heads, n_kv_heads, head_dim, length, tokens, scale, mask=None,
                   workspace=None, out=None):
    """bf16 out [tokens, n_heads * head_dim]: attention of drafted tokens over cache
    rows 0 .. length - 1 and, of their own rows length .. length + tokens - 1, those
    whose bit is set in mask (int32 or uint32 words [tokens, ceil(tokens / 32)]; None:
    a chain, token i sees drafted rows 0 .. i). workspace: a device tensor of at least
    attention_tree_workspace_bytes(...) bytes (allocated here when None). The weights
    meet the values as bf16; for one token attention_decode_split keeps them in f32."""
    T = _torch()
    if out is None:
        out = T.empty(tokens * n_heads * head_dim, dtype=T.bf16, device=q.device)
    if workspace is None:
        wb = attention_tree_workspace_bytes(n_heads, n_kv_heads, head_dim, length, tokens)
        workspace = T.empty(wb, dtype=T.u8, device=q.device) if wb else None
    else:
        wb = workspace.numel() * workspace.element_size()
    nq, nc = tokens * n_heads * head_dim, (length + tokens) * n_kv_heads * head_dim
    if mask is not None and mask.dtype not in T.is32:
        raise ValueError(f"mask must hold 32-bit words, not {mask.dtype}")
    _check(lib().reng_hip_attention_tree(
        _16bit(q, "q", nq), _16bit(k_cache, "k_cache", nc), _16bit(v_cache, "v_cache", nc), n_heads, n_kv_heads,
        head_dim, length, tokens, None if mask is None else _at(mask, "mask", tokens * _nblocks(tokens, 32), 4), scale,
        None if workspace is None else _at(workspace, "workspace", 0, 1), wb, _16bit(out, "out", nq), T.stream()))
    return out


# ---------------------------------------------------------------- a layer held in 4 bits
# MXFP4: e2m1 codes, two a byte, with a power-of-two scale byte for 32 columns of a row.

MX_BLOCK = 32
ROPE_MAX_AXES = 4


def _out16(T, t, what, n, like):
    """(t, its address), allocated like `like` where t is None."""
    if t is None:
        t = T.empty(n, dtype=T.bf16, device=like.device)
        return t, t.data_ptr()
    return t, _16bit(t, what, n)


def mx_scale_pitch(cols):
    """Bytes of a row's scales: one for 32 columns, in words of four."""
    return 4 * _nblocks(cols)


def quantize_mxfp4_into(w, rows, cols, codes, scales, ld=None):
    """quantize_mxfp4 into caller-owned tensors (no allocation)."""
    T = _torch()
    ld = cols if ld is None else ld
    dt = _dtype_code(w)
    _check(lib().reng_hip_quantize_mxfp4(_at(w, "weight", _span(rows, cols, ld), 2 if dt == BF16 else 4), dt, rows, cols, ld,
                                         _8bit(codes, "codes", rows * _nblocks(cols, 2)),
                                         _8bit(scales, "scales", rows * mx_scale_pitch(cols)), T.stream()))


def quantize_mxfp4(w, rows, cols, ld=None):
    """(codes [rows * ceil(cols / 2)], scales [rows * mx_scale_pitch(cols)]) of a device tensor of bf16 (or its
    int16 bits) or f32, [rows, ld] row-major: e2m1 codes under the smallest power of two that leaves a block's
    largest magnitude below 7."""
    T, ld = _torch(), cols if ld is None else ld
    dt = _dtype_code(w)
    at = _at(w, "weight", _span(rows, cols, ld), 2 if dt == BF16 else 4)
    codes = T.empty(rows * _nblocks(cols, 2), dtype=T.u8, device=w.device)
    scales = codes.new_empty(rows * mx_scale_pitch(cols))
    _check(lib().reng_hip_quantize_mxfp4(at, dt, rows, cols, ld, codes.data_ptr(), scales.data_ptr(), T.stream()))
    return codes, scales


def dequantize_mxfp4(codes, scales, rows, cols, out=None):
    """The values of quantize_mxfp4's codes, [rows * cols] as bf16, or as `out` is: bf16 (or its bits) or f32."""
    T = _torch()
    if out is None:
        out = T.empty(rows * cols, dtype=T.bf16, device=codes.device)
    dt = _dtype_code(out)
    _check(lib().reng_hip_dequantize_mxfp4(_8bit(codes, "codes", rows * _nblocks(cols, 2)),
                                           _8bit(scales, "scales", rows * mx_scale_pitch(cols)), rows, cols, dt,
                                           _at(out, "out", rows * cols, 2 if dt == BF16 else 4), T.stream()))
    return out


def gemm_mxfp4(a, scale_a, b, scale_b, M, N, K, out=None):
    """bf16 out[M, N] of codes a [M, K / 2] and b [N, K / 2] with their scales, as quantize_mxfp4 gives them."""
    T, sp, kb = _torch(), mx_scale_pitch(K), _nblocks(K, 2)
    out, op = _out16(T, out, "out", M * N, a)
    _check(lib().reng_hip_gemm_mxfp4(_8bit(a, "a", M * kb), _8bit(scale_a, "scale_a", M * sp), _8bit(b, "b", N * kb),
                                     _8bit(scale_b, "scale_b", N * sp), M, N, K, op, T.stream()))
    return out


class MxCache:
    """A key/value cache held in 4 bits: per key/value head a matrix of [capacity, head_dim] as quantize_mxfp4 lays
    it out. Its tensors are allocated here, or given as (k_codes, k_scales, v_codes, v_scales); rows that
    nothing was written to hold what was there."""

    def __init__(self, n_kv_heads, head_dim, capacity, device="cuda", tensors=None):
        T = _torch()
        self.n_kv_heads, self.head_dim, self.capacity = n_kv_heads, head_dim, capacity
        rows, sp = n_kv_heads * capacity, mx_scale_pitch(head_dim)
        if tensors is None:
            tensors = tuple(T.empty(rows * n, dtype=T.u8, device=device) for n in (head_dim // 2, sp) * 2)
        self.tensors = tuple(tensors)
        at = [_8bit(t, what, rows * n) for t, what, n in zip(self.tensors, ("k_codes", "k_scales", "v_codes", "v_scales"),
                                                             (head_dim // 2, sp) * 2)]
        self.device = self.tensors[0].device
        self._struct = _MxCache(*at, n_kv_heads, head_dim, capacity)
        self._ref = ctypes.addressof(self._struct)

    def _here(self):
        """The descriptor's address, for a call on the current device."""
        if _T.several and self.device.index != _T.current_device():
            raise ValueError(f"the cache is on {self.device}, the current device is cuda:{_T.current_device()}")
        return self._ref

    def write(self, k, v, first, tokens):
        """Rows first .. first + tokens - 1 from bf16 k and v [tokens, n_kv_heads * head_dim] (rows may be strided)."""
        head_norm_rope_mxfp4(None, k, v, tokens, 0, self, first)

    def read(self, first, rows, k=None, v=None):
        """(k, v) bf16 [rows * n_kv_heads * head_dim] of rows first .. first + rows - 1."""
        T, n = _torch(), rows * self.n_kv_heads * self.head_dim
        (k, kp), (v, vp) = _out16(T, k, "k", n, self.tensors[0]), _out16(T, v, "v", n, self.tensors[0])
        _check(lib().reng_hip_cache_read_mxfp4(self._here(), first, rows, kp, vp, T.stream()))
        return k, v


class Rope:
    """Rotation tables: sin and cos f32 [rows, rot_dim], and which axis' position each of the rot_dim / 2 pairs
    takes: sections (s0, s1, ..) for the first s0 pairs axis 0, the next s1 axis 1 and so on, or pair_axis with an
    axis for each pair; without either all take axis 0."""

    def __init__(self, sin, cos, sections=None, pair_axis=None):
        _torch()
        if sin.dim() != 2 or sin.shape != cos.shape:
            raise ValueError(f"tables of shapes {tuple(sin.shape)} and {tuple(cos.shape)}; expected the same [rows, rot_dim]")
        rows, rot = sin.shape
        if sections is not None:
            if pair_axis is not None:
                raise ValueError("sections and pair_axis both given")
            if any(n < 0 for n in sections):
                raise ValueError(f"sections {tuple(sections)}; expected numbers of pairs")
            pair_axis = [a for a, n in enumerate(sections) for _ in range(n)]
        if pair_axis is not None:
            pair_axis = [operator.index(a) for a in pair_axis]   # an array's own bytes would be its elements' words
            if len(pair_axis) != rot // 2:
                raise ValueError(f"axes for {len(pair_axis)} pairs; the tables rotate {rot // 2}")
        self.axes = 1 if pair_axis is None else len(sections) if sections is not None else max(pair_axis) + 1
        if self.axes > ROPE_MAX_AXES or (pair_axis is not None and min(pair_axis) < 0):
            raise ValueError(f"pairs of axes {min(pair_axis)} to {self.axes - 1}; expected 0 to {ROPE_MAX_AXES - 1} at most")
        self.device, self.tables = sin.device, (sin, cos)
        # ctypes keeps the bytes alive with the descriptor; one axis needs no map.
        self._struct = _Rope(_f32(sin, "sin", rows * rot), _f32(cos, "cos", rows * rot), rows, rot, self.axes,
                             bytes(pair_axis) if self.axes > 1 else None)
        self._ref = ctypes.addressof(self._struct)


def _rows16(t, what, tokens, width):
    """(address, row pitch) of bf16 rows: a contiguous tensor of any shape but two dimensions, or [>= tokens, >= width]
    with contiguous columns."""
    if t.dim() != 2:
        return _16bit(t, what, tokens * width), width
    (rows, cols), (ld, one) = t.shape, t.stride()
    if t.dtype not in _T.is16 or not t.is_cuda or one != 1 or rows < tokens or cols < width:
        raise ValueError(f"{what} must be bf16 (or its bits) rows on the GPU, [{tokens}, {width}] with contiguous columns, "
                         f"not {t.dtype} {tuple(t.shape)} of strides {t.stride()}")
    if _T.several and t.get_device() != _T.current_device():
        raise ValueError(f"{what} is on cuda:{t.get_device()}, the current device is cuda:{_T.current_device()}")
    return t.data_ptr(), ld if tokens > 1 else width   # one row has no pitch


def _heads_args(T, q, k, v, tokens, n_heads, n_kv_heads, head_dim, q_gamma, k_gamma, rope, positions):
    """What both calls share: the rows' addresses and pitches, and gammas, rope and positions."""
    nk = n_kv_heads * head_dim
    kp, k_ld = _rows16(k, "k", tokens, nk)
    vp, v_ld = (None, k_ld) if v is None else _rows16(v, "v", tokens, nk)
    if k_ld != v_ld:
        raise ValueError(f"k and v must have one row pitch, not {k_ld} and {v_ld}")
    qp, q_ld = (None, 0) if q is None else _rows16(q, "q", tokens, n_heads * head_dim)
    ref = pos = None
    if rope is not None:
        if T.several and rope.device.index != T.current_device():
            raise ValueError(f"the tables are on {rope.device}, the current device is cuda:{T.current_device()}")
        if positions is None or positions.dtype != T.i32 or (rope.axes > 1 and positions.numel() != rope.axes * tokens):
            raise ValueError(f"positions must be int32 [{rope.axes}, {tokens}]")
        ref, pos = rope._ref, _at(positions, "positions", rope.axes * tokens, 4)
    gq = None if q_gamma is None else _f32(q_gamma, "q_gamma", head_dim)
    gk = None if k_gamma is None else _f32(k_gamma, "k_gamma", head_dim)
    return (qp, q_ld, kp, vp, k_ld), (gq, gk), (ref, pos)


def head_norm_rope_bf16(q, k, v, tokens, n_heads, n_kv_heads, head_dim, q_gamma=None, k_gamma=None, eps=1e-6, rope=None,
                        positions=None, q_out=None, k_rows=None, v_rows=None):
    """(q_out, k_rows, v_rows): queries and keys normalised per head (where gammas f32 [head_dim] are given) and rotated
    (rope, a Rope, at positions int32 [axes, tokens]), values as they are, bf16 [tokens, heads * head_dim]. q, k and v
    are bf16 rows, which may be column ranges of a wider tensor; k_rows and v_rows a bf16 cache's rows."""
    T = _torch()
    nq, nk = tokens * n_heads * head_dim, tokens * n_kv_heads * head_dim
    rows, gammas, at = _heads_args(T, q, k, v, tokens, n_heads, n_kv_heads, head_dim, q_gamma, k_gamma, rope, positions)
    qp = vp = None
    if q is not None or q_out is not None:
        q_out, qp = _out16(T, q_out, "q_out", nq, k)
    k_rows, kp = _out16(T, k_rows, "k_rows", nk, k)
    if v is not None or v_rows is not None:
        v_rows, vp = _out16(T, v_rows, "v_rows", nk, k)
    _check(lib().reng_hip_head_norm_rope_bf16(*rows, tokens, n_heads, n_kv_heads, head_dim, *gammas, eps, *at, qp, kp, vp,
                                              T.stream()))
    return q_out, k_rows, v_rows


def head_norm_rope_mxfp4(q, k, v, tokens, n_heads, cache, first, q_gamma=None, k_gamma=None, eps=1e-6, rope=None,
                         positions=None, q_out=None):
    """q_out: head_norm_rope_bf16 with keys and values quantized into rows first .. first + tokens - 1 of an MxCache."""
    T = _torch()
    hd = cache.head_dim
    rows, gammas, at = _heads_args(T, q, k, v, tokens, n_heads, cache.n_kv_heads, hd, q_gamma, k_gamma, rope, positions)
    qp = None
    if q is not None or q_out is not None:
        q_out, qp = _out16(T, q_out, "q_out", tokens * n_heads * hd, k)
    _check(lib().reng_hip_head_norm_rope_mxfp4(*rows, tokens, n_heads, *gammas, eps, *at, qp, cache._here(), first, T.stream()))
    return q_out


def attention_mxfp4_workspace_bytes(n_heads, n_kv_heads, head_dim, length, tokens):
    """Device workspace attention_mxfp4 needs for up to `length` context rows and `tokens` tokens."""
    return lib().reng_hip_attention_mxfp4_workspace_bytes(n_heads, n_kv_heads, head_dim, length, tokens)


def attention_mxfp4(q, cache, n_heads, length, tokens, scale, mask=None, workspace=None, out=None):
    """bf16 out [tokens, n_heads * head_dim]: attention_tree over an MxCache, whose rows 0 .. length - 1 are
    context and the next `tokens` the tokens' own (mask as there; None: a chain). workspace: a device tensor of
    at least attention_mxfp4_workspace_bytes(...) bytes (allocated here when None)."""
    T = _torch()
    nq = tokens * n_heads * cache.head_dim
    out, op = _out16(T, out, "out", nq, q)
    if workspace is None:
        wb = attention_mxfp4_workspace_bytes(n_heads, cache.n_kv_heads, cache.head_dim, length, tokens)
        workspace = T.empty(wb, dtype=T.u8, device=q.device) if wb else None
    else:
        wb = workspace.numel() * workspace.element_size()
    if mask is not None and mask.dtype not in T.is32:
        raise ValueError(f"mask must hold 32-bit words, not {mask.dtype}")
    _check(lib().reng_hip_attention_mxfp4(
        _16bit(q, "q", nq), cache._here(), n_heads, length, tokens,
        None if mask is None else _at(mask, "mask", tokens * _nblocks(tokens, 32), 4), scale,
        None if workspace is None else _at(workspace, "workspace", 0, 1), wb, op, T.stream()))
    return out


# ---------------------------------------------------------------- decode step
# The non-GEMM steps of one Llama decoder layer at decode time (csrc/layer.hip);
# the C++ host path (host/fp8_decoder.hpp) strings them together with the GEMV.


def rms_norm_bf16(x, gamma, rows, cols, eps, out=None):
    """out[rows, cols] bf16 = x / sqrt(mean(x^2) + eps) * gamma, x f32 (ops.rs:49-72)."""
    import torch

    if out is None:
        out = torch.empty(rows * cols, dtype=torch.bfloat16, device=x.device)
    _check(lib().reng_hip_rms_norm_bf16(_dev(x, "x", 4 * rows * cols), _dev(gamma, "gamma", 4 * cols), rows, cols,
                                        eps, _dev(out, "out", 2 * rows * cols), _stream()))
    return out


def gemv_residual(x, codes, scales, n, k, fmt, residual, out=None):
    """f32 out[n] = residual + bf16(x . (decode(codes[n, k]) * scales)^T), x bf16 [k]."""
    import torch

    if out is None:
        out = torch.empty(n, dtype=torch.float32, device=x.device)
    _check(lib().reng_hip_gemv_w8a16_residual(_dev(x, "x", 2 * k), _dev(codes, "codes", n * k),
                                              _opt(scales, "scales", 4 * n), n, k, _fmt(fmt),
                                              _dev(residual, "residual", 4 * n), _dev(out, "out", 4 * n), _stream()))
    return out


def gemv_swiglu(x, codes, scales, n, k, fmt, out=None):
    """bf16 out[n / 2] = silu(gate) * up over codes whose rows alternate gate,
    up (row 2i gate row i, row 2i + 1 up row i)."""
    import torch

    if out is None:
        out = torch.empty(n // 2, dtype=torch.bfloat16, device=x.device)
    _check(lib().reng_hip_gemv_w8a16_swiglu(_dev(x, "x", 2 * k), _dev(codes, "codes", n * k),
                                            _opt(scales, "scales", 4 * n), n, k, _fmt(fmt),
                                            _dev(out, "out", 2 * (n // 2)), _stream()))
    return out


def gemv_rmsnorm(x, gamma, eps, codes, scales, n, k, fmt, swiglu=False, out=None):
    """bf16 out = W . bf16(rms_norm(x) * gamma), x f32 [k]; with swiglu the rows
    of codes alternate gate, up and out[n / 2] = silu(gate) * up."""
    import torch

    if out is None:
        out = torch.empty(n // 2 if swiglu else n, dtype=torch.bfloat16, device=x.device)
    fn = lib().reng_hip_gemv_w8a16_rmsnorm_swiglu if swiglu else lib().reng_hip_gemv_w8a16_rmsnorm
    _check(fn(_dev(x, "x", 4 * k), _dev(gamma, "gamma", 4 * k), eps, _dev(codes, "codes", n * k),
              _opt(scales, "scales", 4 * n), n, k, _fmt(fmt), _dev(out, "out", 2 * (n // 2 if swiglu else n)),
              _stream()))
    return out


def qkv_rope_row_order(n_heads, n_kv_heads, head_dim):
    """Source row (in [Wq; Wk; Wv] order) of each row of the rotation-pair
    order gemv_rmsnorm_qkv_rope takes."""
    import numpy as np

    half = head_dim // 2
    order = []
    for heads, base in ((n_heads, 0), (n_kv_heads, n_heads * head_dim)):
        for h in range(heads):
            for d in range(half):
                order += [base + h * head_dim + d, base + h * head_dim + d + half]
    order += list(range((n_heads + n_kv_heads) * head_dim, (n_heads + 2 * n_kv_heads) * head_dim))
    return np.asarray(order, dtype=np.int64)


def gemv_rmsnorm_qkv_rope(x, gamma, eps, codes, scales, n_heads, n_kv_heads, head_dim, k, fmt, sin_row, cos_row,
                          q, k_row, v_row):
    """Norm + [q | k | v] projection + RoPE + cache-row writes in one pass over
    codes in qkv_rope_row_order."""
    n = (n_heads + 2 * n_kv_heads) * head_dim
    _check(lib().reng_hip_gemv_w8a16_rmsnorm_qkv_rope(
        _dev(x, "x", 4 * k), _dev(gamma, "gamma", 4 * k), eps, _dev(codes, "codes", n * k),
        _opt(scales, "scales", 4 * n), n_heads, n_kv_heads, head_dim, k, _fmt(fmt),
        _dev(sin_row, "sin_row", 4 * head_dim), _dev(cos_row, "cos_row", 4 * head_dim),
        _dev(q, "q", 2 * n_heads * head_dim), _dev(k_row, "k_row", 2 * n_kv_heads * head_dim),
        _dev(v_row, "v_row", 2 * n_kv_heads * head_dim), _stream()))


def add_rms_norm_bf16(x, d, gamma, rows, cols, eps, h=None, out=None):
    """h = x + d (f32) and out = bf16(rms_norm(h) * gamma); returns (h, out)."""
    import torch

    if h is None:
        h = torch.empty(rows * cols, dtype=torch.float32, device=x.device)
    if out is None:
        out = torch.empty(rows * cols, dtype=torch.bfloat16, device=x.device)
    n = rows * cols
    _check(lib().reng_hip_add_rms_norm_bf16(_dev(x, "x", 4 * n), _dev(d, "d", 2 * n), _dev(gamma, "gamma", 4 * cols),
                                            rows, cols, eps, _dev(h, "h", 4 * n), _dev(out, "out", 2 * n),
                                            _stream()))
    return h, out


def rope_append(q, k, v, n_heads, n_kv_heads, head_dim, sin_row, cos_row, k_row, v_row):
    """Rotate-half RoPE of one position: q in place, k into k_row, v copied to v_row."""
    nq, nk = 2 * n_heads * head_dim, 2 * n_kv_heads * head_dim
    _check(lib().reng_hip_rope_append(_dev(q, "q", nq), _dev(k, "k", nk), _dev(v, "v", nk), n_heads, n_kv_heads,
                                      head_dim, _dev(sin_row, "sin_row", 4 * head_dim),
                                      _dev(cos_row, "cos_row", 4 * head_dim), _dev(k_row, "k_row", nk),
                                      _dev(v_row, "v_row", nk), _stream()))


def attention_decode(q, k_cache, v_cache, n_heads, n_kv_heads, head_dim, length, scale, out=None):
    """One query per head over cache rows 0 .. length - 1, bf16 out [n_heads * head_dim]."""
    import torch

    if out is None:
        out = torch.empty(n_heads * head_dim, dtype=torch.bfloat16, device=q.device)
    nq, nc = 2 * n_heads * head_dim, 2 * length * n_kv_heads * head_dim
    _check(lib().reng_hip_attention_decode(_dev(q, "q", nq), _dev(k_cache, "k_cache", nc),
                                           _dev(v_cache, "v_cache", nc), n_heads, n_kv_heads, head_dim, length, scale,
                                           _dev(out, "out", nq), _stream()))
    return out


def attention_workspace_bytes(n_heads, head_dim, length):
    """Device workspace attention_decode_split needs for caches of 1 .. length rows."""
    return lib().reng_hip_attention_workspace_bytes(n_heads, head_dim, length)


def attention_decode_split(q, k_cache, v_cache, n_heads, n_kv_heads, head_dim, length, scale, workspace=None,
                           out=None):
    """attention_decode with the cache split over workgroups and merged; workspace
    a device tensor of at least attention_workspace_bytes(...) bytes (allocated
    here when None)."""
    import torch

    if out is None:
        out = torch.empty(n_heads * head_dim, dtype=torch.bfloat16, device=q.device)
    if workspace is None:
        workspace = torch.empty(max(1, attention_workspace_bytes(n_heads, head_dim, length)), dtype=torch.uint8,
                                device=q.device)
    nq, nc = 2 * n_heads * head_dim, 2 * length * n_kv_heads * head_dim
    _check(lib().reng_hip_attention_decode_split(_dev(q, "q", nq), _dev(k_cache, "k_cache", nc),
                                                 _dev(v_cache, "v_cache", nc), n_heads, n_kv_heads, head_dim, length,
                                                 scale,
                                                 _dev(workspace, "workspace"),
                                                 workspace.numel() * workspace.element_size(),
                                                 _dev(out, "out", nq), _stream()))
    return out


def silu_mul_bf16(gate, up, n, out=None):
    import torch

    if out is None:
        out = torch.empty(n, dtype=torch.bfloat16, device=gate.device)
    _check(lib().reng_hip_silu_mul_bf16(_dev(gate, "gate", 2 * n), _dev(up, "up", 2 * n), n, _dev(out, "out", 2 * n),
                                        _stream()))
    return out


def add_bf16_f32(x, d, n, out=None):
    import torch

    if out is None:
        out = torch.empty(n, dtype=torch.float32, device=x.device)
    _check(lib().reng_hip_add_bf16_f32(_dev(x, "x", 4 * n), _dev(d, "d", 2 * n), n, _dev(out, "out", 4 * n),
                                       _stream()))
    return out


def stream_read(buf, nbytes, sink):
    """The read yardstick: read nbytes of buf once (a device tensor; sink a
    device tensor of at least stream_read_sink_bytes() bytes)."""
    _check(lib().reng_hip_stream_read(_dev(buf, "buf", nbytes), nbytes,
                                      _dev(sink, "sink", lib().reng_hip_stream_read_sink_bytes()), _stream()))


def stream_narrow(src, elems, dst):
    """The stream yardstick: the high byte of each of elems bf16 values of src
    into dst (device tensors)."""
    _check(lib().reng_hip_stream_narrow(_dev(src, "src", 2 * elems), elems, _dev(dst, "dst", elems), _stream()))


def stream_stage(x, codes, M, N, K, sink):
    """The copy yardstick of the 16 < M <= 64 skinny GEMM: its global -> LDS
    copy stream for x [M, K] and codes [N, K] with no arithmetic (device tensors;
    sink: a device tensor of at least 4 bytes)."""
    _check(lib().reng_hip_stream_stage(_dev(x, "x", 2 * M * K), _dev(codes, "codes", N * K), M, N, K,
                                       _dev(sink, "sink", 4), _stream()))


def stream_read_sink_bytes():
    return int(lib().reng_hip_stream_read_sink_bytes())


def verify_hw_convert(fmt):
    n = ctypes.c_uint64(0)
    first = ctypes.c_uint32(0)
    _check(lib().reng_hip_verify_hw_convert(_fmt(fmt), ctypes.byref(n), ctypes.byref(first)))
    return int(n.value), int(first.value)
