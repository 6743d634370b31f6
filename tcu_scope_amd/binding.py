"""ctypes binding of libtcu_scope_amd.so; every function takes torch CUDA tensors and
launches on torch's current stream unless told otherwise."""
import ctypes
import enum
import functools
import os
import subprocess

_HERE = os.path.dirname(os.path.abspath(__file__))
_LIB = os.environ.get("TCU_SCOPE_AMD_LIBRARY") or os.path.join(_HERE, "libtcu_scope_amd.so")
_CSRC = os.path.join(_HERE, "csrc")

EXPORTS = [
    "tcu_abi_version", "tcu_last_error", "tcu_init", "tcu_device_info", "tcu_set_option",
    "tcu_seg_reduce_f16", "tcu_seg_reduce_offsets_f16", "tcu_seg_scan_f16", "tcu_seg_scan_f16_noalloc", "tcu_seg_scan_offsets_f16", "tcu_seg_scan_by_key_f16", "tcu_seg_reduce_by_key_f16", "tcu_add_partial_sums_f16",
    "tcu_full_reduce_f16", "tcu_full_scan_f16", "tcu_gemv_f16_f32", "tcu_gemm_f16_f32", "tcu_gemv_f16_f16", "tcu_gemm_f16_f16", "tcu_gemv_col_major_f16_f32", "tcu_gemv_col_major_f16_f16",
    "tcu_gated_scan", "tcu_gated_scan_backward", "tcu_gated_scan_step", "tcu_fused_norm", "tcu_fused_norm_backward", "tcu_fused_gemm", "tcu_fused_gemm_backward",
    "tcu_fill_f16", "tcu_convert_f32_to_f16", "tcu_generate_f16", "tcu_stream_probe", "tcu_time_next_launch", "tcu_lane_probe", "tcu_temporary_allocations",
]


class Variant(enum.IntEnum):
    AUTO = 0
    MFMA_16 = 1
    MFMA_16N = 2
    MFMA_16N_BLOCK = 3
    MFMA_256 = 4
    MFMA_256N = 5
    MFMA_256N_BLOCK = 6
    WAVE_SHUFFLE = 7
    BLOCK_LDS = 8


VARIANTS = list(Variant)


class FullStrategy(enum.IntEnum):
    AUTO = 0
    SINGLE_PASS = 1
    MULTI_KERNEL = 2


# flag OR-ed onto a FullStrategy: the single-pass full-array kernels work on the matrix unit
FULL_MFMA = 0x100


class Dist(enum.IntEnum):
    UNIFORM = 0
    GRID = 1
    NORMAL = 2
    SMALLINT = 3


class Gate(enum.IntEnum):
    """How a gated scan reads its gate g: a = g, a = exp(g), or a = sigmoid(g) with the input weighted by 1 - a."""

    DECAY = 0
    LOG = 1
    SIGMOID = 2


class Activation(enum.IntEnum):
    """Activations of a gate and of a product's epilogue; GELU is the tanh form."""

    NONE = 0
    RELU = 1
    GELU = 2
    SILU = 3
    SIGMOID = 4


class Norm(enum.IntEnum):
    RMS = 0
    LAYER = 1


class NormOrder(enum.IntEnum):
    """ADD_NORM: the norm of residual + s x; NORM_ADD: residual + s times the (gated) norm of x."""

    ADD_NORM = 0
    NORM_ADD = 1


class GatedScanShape(ctypes.Structure):
    """tcu_gated_scan_shape."""

    _fields_ = [("dtype", ctypes.c_int), ("gate", ctypes.c_int), ("channels", ctypes.c_size_t), ("num_rows", ctypes.c_size_t), ("num_sequences", ctypes.c_size_t), ("sequence_length", ctypes.c_size_t),
                ("d_offsets", ctypes.c_void_p), ("offset_bits", ctypes.c_int), ("zero_outside", ctypes.c_int)]


class FusedNormShape(ctypes.Structure):
    """tcu_fused_norm_shape."""

    _fields_ = [("dtype", ctypes.c_int), ("norm", ctypes.c_int), ("order", ctypes.c_int), ("activation", ctypes.c_int), ("rows", ctypes.c_size_t), ("dim", ctypes.c_size_t), ("eps", ctypes.c_float),
                ("scale", ctypes.c_float)]


class FusedGemmShape(ctypes.Structure):
    """tcu_fused_gemm_shape."""

    _fields_ = [("dtype", ctypes.c_int), ("activation", ctypes.c_int), ("M", ctypes.c_size_t), ("N", ctypes.c_size_t), ("K", ctypes.c_size_t), ("beta", ctypes.c_float)]


class TcuError(RuntimeError):
    """A non-zero tcu_status; .status is 1 invalid argument, 2 unsupported, 3 runtime, 4 workspace."""

    def __init__(self, status, message):
        super().__init__(f"tcu_status {status}: {message}")
        self.status = status


def library_path():
    return _LIB


def build():
    """Compile the HIP sources for gfx950 into libtcu_scope_amd.so (needs hipcc, no GPU)."""
    subprocess.check_call(["make", "-C", _CSRC, "clean"], stdout=subprocess.DEVNULL)
    subprocess.check_call(["make", "-j4", "-C", _CSRC], stdout=subprocess.DEVNULL)
    return _LIB


_lib = None


def lib():
    """The loaded shared library.  Raises when it has not been built: there is no fallback."""
    global _lib
    if _lib is None:
        if not os.path.exists(_LIB):
            raise ImportError(f"{_LIB} is missing: build it with `make -C {_CSRC}` (python -c 'import __graft_entry__ as g; g.build()')")
        L = ctypes.CDLL(_LIB)
        c = ctypes
        vp, sz, ci, cf = c.c_void_p, c.c_size_t, c.c_int, c.c_float
        L.tcu_abi_version.restype = ci
        L.tcu_last_error.restype = c.c_char_p
        L.tcu_init.argtypes = [ci]
        L.tcu_device_info.argtypes = [c.POINTER(ci)] * 4
        L.tcu_set_option.argtypes = [c.c_char_p, ci]
        L.tcu_seg_reduce_f16.argtypes = [vp, vp, sz, sz, ci, ci, ci, vp]
        L.tcu_seg_reduce_offsets_f16.argtypes = [vp, vp, sz, vp, vp, ci, sz, vp]
        L.tcu_seg_scan_f16.argtypes = [vp, vp, vp, sz, sz, ci, ci, ci, vp]
        L.tcu_seg_scan_f16_noalloc.argtypes = [vp, vp, vp, sz, sz, ci, ci, ci, vp]
        L.tcu_seg_scan_offsets_f16.argtypes = [vp, vp, sz, vp, vp, ci, sz, vp]
        L.tcu_seg_scan_by_key_f16.argtypes = [vp, vp, vp, sz, ci, vp, c.POINTER(sz), vp]
        L.tcu_seg_reduce_by_key_f16.argtypes = [vp, vp, vp, vp, vp, sz, ci, vp, c.POINTER(sz), vp]
        L.tcu_add_partial_sums_f16.argtypes = [vp, vp, sz, sz, vp]
        L.tcu_full_reduce_f16.argtypes = [vp, vp, sz, vp, c.POINTER(sz), ci, sz, ci, vp]
        L.tcu_full_scan_f16.argtypes = [vp, vp, sz, vp, c.POINTER(sz), ci, sz, ci, vp]
        L.tcu_gemv_f16_f32.argtypes = [vp, vp, vp, sz, sz, cf, cf, ci, vp]
        L.tcu_gemm_f16_f32.argtypes = [vp, vp, vp, vp, sz, sz, sz, cf, cf, ci, vp]
        L.tcu_gemv_f16_f16.argtypes = [vp, vp, vp, sz, sz, cf, cf, ci, vp]
        L.tcu_gemv_col_major_f16_f32.argtypes = [vp, sz, vp, vp, sz, sz, cf, cf, vp]
        L.tcu_gemv_col_major_f16_f16.argtypes = [vp, sz, vp, vp, sz, sz, cf, cf, vp]
        L.tcu_gemm_f16_f16.argtypes = [vp, vp, vp, vp, sz, sz, sz, cf, cf, ci, vp]
        L.tcu_fill_f16.argtypes = [vp, cf, sz, vp]
        L.tcu_convert_f32_to_f16.argtypes = [vp, vp, sz, vp]
        L.tcu_generate_f16.argtypes = [vp, sz, c.c_uint64, ci, sz, vp]
        L.tcu_stream_probe.argtypes = [vp, vp, sz, ci, ci, ci, vp]
        L.tcu_lane_probe.argtypes = [vp, c.POINTER(sz), vp]
        L.tcu_time_next_launch.argtypes = [vp, vp]
        L.tcu_temporary_allocations.argtypes = []
        L.tcu_temporary_allocations.restype = c.c_ulong
        shape, psz = c.POINTER(GatedScanShape), c.POINTER(sz)
        L.tcu_gated_scan.argtypes = [shape, vp, sz, vp, sz, vp, sz, vp, vp, vp, psz, vp]
        L.tcu_gated_scan_backward.argtypes = [shape, vp, sz, vp, sz, vp, sz, vp, sz, vp, vp, vp, sz, vp, sz, vp, vp, psz, vp]
        L.tcu_gated_scan_step.argtypes = [ci, ci, sz, sz, vp, sz, vp, sz, vp, sz, vp, vp, sz, vp, ci, vp]
        norm, m = c.POINTER(FusedNormShape), [vp, sz]
        L.tcu_fused_norm.argtypes = [norm, *m * 3, vp, vp, vp, *m * 2, vp]
        L.tcu_fused_norm_backward.argtypes = [norm, *m * 3, vp, vp, vp, *m * 5, vp, vp, vp, vp, psz, vp]
        product = c.POINTER(FusedGemmShape)
        L.tcu_fused_gemm.argtypes = [product, *m * 2, vp, *m * 3, vp, psz, vp]
        L.tcu_fused_gemm_backward.argtypes = [product, *m * 6, vp, vp, psz, vp]
        for name in EXPORTS:
            if name not in ("tcu_last_error", "tcu_temporary_allocations"):
                getattr(L, name).restype = ci
        _lib = L
    return _lib


def _check(rc):
    if rc != 0:
        raise TcuError(rc, lib().tcu_last_error().decode())


_torch_module = None


def _torch():
    global _torch_module
    if _torch_module is None:
        import torch

        _torch_module = torch
    return _torch_module


def _stream(stream):
    torch = _torch()
    if stream is None:
        stream = torch.cuda.current_stream()
    return ctypes.c_void_p(stream.cuda_stream)


def _ptr(t):
    return ctypes.c_void_p(t.data_ptr()) if t is not None else None


def _need_f16(t, name):
    torch = _torch()
    if t.dtype != torch.float16 or not t.is_cuda or not t.is_contiguous():
        raise ValueError(f"{name} must be a contiguous CUDA float16 tensor")


def init(device_id=0):
    _check(lib().tcu_init(device_id))


def device_info():
    vals = [ctypes.c_int() for _ in range(4)]
    _check(lib().tcu_device_info(*[ctypes.byref(v) for v in vals]))
    return {"compute_units": vals[0].value, "wavefront_size": vals[1].value, "lds_bytes": vals[2].value, "is_gfx950": bool(vals[3].value)}


def set_option(name, value):
    _check(lib().tcu_set_option(name.encode(), int(value)))


def seg_reduce(x, segment_size, variant=Variant.AUTO, tiles_per_wave=0, waves_per_block=0, out=None, num_segments=None, stream=None):
    """out[j] = sum of x[j*S:(j+1)*S] (fp32 accumulate, fp16 result)."""
    torch = _torch()
    _need_f16(x, "x")
    nseg = (x.numel() // segment_size if segment_size > 0 else 1) if num_segments is None else num_segments
    if out is None:
        out = torch.empty(nseg, dtype=torch.float16, device=x.device)
    _check(lib().tcu_seg_reduce_f16(_ptr(x), _ptr(out), nseg, segment_size, int(variant), tiles_per_wave, waves_per_block, _stream(stream)))
    return out


def seg_reduce_offsets(x, begin, end, expected_segment_size=0, out=None, stream=None):
    """out[j] = sum of x[begin[j]:end[j]] (empty when end[j] <= begin[j]); begin/end are int32 or int64
    device tensors of equal length (two views of one offsets tensor are fine)."""
    torch = _torch()
    _need_f16(x, "x")
    if begin.dtype != end.dtype or begin.dtype not in (torch.int32, torch.int64) or begin.numel() != end.numel():
        raise ValueError("begin and end must be int32 or int64 tensors of the same length")
    if not (begin.is_contiguous() and end.is_contiguous()):
        raise ValueError("begin and end must be contiguous")
    nseg = begin.numel()
    if out is None:
        out = torch.empty(nseg, dtype=torch.float16, device=x.device)
    bits = 32 if begin.dtype == torch.int32 else 64
    _check(lib().tcu_seg_reduce_offsets_f16(_ptr(x), _ptr(out), nseg, _ptr(begin), _ptr(end), bits, expected_segment_size, _stream(stream)))
    return out


def seg_scan(x, segment_size, variant=Variant.AUTO, tiles_per_wave=0, waves_per_block=0, out=None, totals=None, num_segments=None, stream=None):
    """Inclusive prefix sum inside every segment; `totals` (optional tensor) receives the segment totals."""
    torch = _torch()
    _need_f16(x, "x")
    nseg = (x.numel() // segment_size if segment_size > 0 else 1) if num_segments is None else num_segments
    if out is None:
        out = torch.empty(nseg * max(segment_size, 0), dtype=torch.float16, device=x.device)
    _check(lib().tcu_seg_scan_f16(_ptr(x), _ptr(out), _ptr(totals), nseg, segment_size, int(variant), tiles_per_wave, waves_per_block, _stream(stream)))
    return out


def seg_scan_noalloc(x, segment_size, out, variant=Variant.AUTO, tiles_per_wave=0, waves_per_block=0, totals=None, num_segments=None, stream=None):
    """seg_scan through tcu_seg_scan_f16_noalloc: the caller brings `out`, nothing is allocated on the way
    (the look-back path keeps its partition descriptors in an array inside the library's device code)."""
    _need_f16(x, "x")
    _need_f16(out, "out")
    nseg = (x.numel() // segment_size if segment_size > 0 else 1) if num_segments is None else num_segments
    _check(lib().tcu_seg_scan_f16_noalloc(_ptr(x), _ptr(out), _ptr(totals), nseg, segment_size, int(variant), tiles_per_wave, waves_per_block, _stream(stream)))
    return out


def seg_scan_offsets(x, begin, end, expected_segment_size=0, out=None, stream=None):
    """Inclusive prefix sums inside every x[begin[j]:end[j]] (non-overlapping); the rest of `out` is not written."""
    torch = _torch()
    _need_f16(x, "x")
    if begin.dtype != end.dtype or begin.dtype not in (torch.int32, torch.int64) or begin.numel() != end.numel():
        raise ValueError("begin and end must be int32 or int64 tensors of the same length")
    if not (begin.is_contiguous() and end.is_contiguous()):
        raise ValueError("begin and end must be contiguous")
    if out is None:
        out = torch.zeros_like(x)
    bits = 32 if begin.dtype == torch.int32 else 64
    _check(lib().tcu_seg_scan_offsets_f16(_ptr(x), _ptr(out), begin.numel(), _ptr(begin), _ptr(end), bits, expected_segment_size, _stream(stream)))
    return out


def _key_bits(keys):
    torch = _torch()
    if keys.dtype not in (torch.int32, torch.int64) or not keys.is_cuda or not keys.is_contiguous():
        raise ValueError("keys must be a contiguous CUDA int32 or int64 tensor")
    return 32 if keys.dtype == torch.int32 else 64


def seg_scan_by_key(keys, x, out=None, workspace=None, stream=None):
    """Inclusive prefix sums inside runs of equal consecutive keys (thrust::inclusive_scan_by_key)."""
    torch = _torch()
    _need_f16(x, "x")
    bits = _key_bits(keys)
    n = x.numel()
    if keys.numel() != n:
        raise ValueError("keys and x must have the same length")
    if out is None:
        out = torch.empty_like(x)
    need = ctypes.c_size_t(0)
    _check(lib().tcu_seg_scan_by_key_f16(None, None, None, n, bits, None, ctypes.byref(need), None))
    if workspace is None:
        workspace = torch.empty(max(need.value, 256), dtype=torch.uint8, device=x.device)
    have = ctypes.c_size_t(_workspace_bytes(workspace, x.device, need.value))
    _check(lib().tcu_seg_scan_by_key_f16(_ptr(keys), _ptr(x), _ptr(out), n, bits, _ptr(workspace), ctypes.byref(have), _stream(stream)))
    return out


def seg_reduce_by_key(keys, x, workspace=None, stream=None):
    """One sum per run of equal consecutive keys (thrust::reduce_by_key): returns (keys_out, sums, num_runs tensor);
    the first two have room for x.numel() entries, of which the first num_runs.item() are written."""
    torch = _torch()
    _need_f16(x, "x")
    bits = _key_bits(keys)
    n = x.numel()
    if keys.numel() != n:
        raise ValueError("keys and x must have the same length")
    keys_out = torch.empty_like(keys)
    out = torch.empty_like(x)
    num_runs = torch.zeros(1, dtype=torch.int64, device=x.device)
    need = ctypes.c_size_t(0)
    _check(lib().tcu_seg_reduce_by_key_f16(None, None, None, None, None, n, bits, None, ctypes.byref(need), None))
    if workspace is None:
        workspace = torch.empty(max(need.value, 256), dtype=torch.uint8, device=x.device)
    have = ctypes.c_size_t(_workspace_bytes(workspace, x.device, need.value))
    _check(lib().tcu_seg_reduce_by_key_f16(_ptr(keys), _ptr(x), _ptr(keys_out), _ptr(out), _ptr(num_runs), n, bits, _ptr(workspace), ctypes.byref(have), _stream(stream)))
    return keys_out, out, num_runs


def _workspace_bytes(workspace, device, need):
    """Bytes of a workspace the caller gives.  An empty tensor has a null pointer, which the library takes as a question for the size: the
    call would return without having computed anything."""
    if workspace.device != device or not workspace.is_contiguous():
        raise ValueError(f"workspace must be a contiguous tensor on {device}")
    have = workspace.numel() * workspace.element_size()
    if have == 0 and need > 0:
        raise ValueError(f"workspace is empty; the call needs {need} bytes at least")
    return have


def add_partial_sums(out, partial_sums, segment_size, stream=None):
    _need_f16(out, "out")
    _need_f16(partial_sums, "partial_sums")
    _check(lib().tcu_add_partial_sums_f16(_ptr(out), _ptr(partial_sums), partial_sums.numel(), segment_size, _stream(stream)))
    return out


def _workspace(fn, x, out, n, strategy, segment_size, waves_per_block, workspace, stream):
    torch = _torch()
    need = ctypes.c_size_t(0)
    _check(fn(_ptr(x), None, n, None, ctypes.byref(need), int(strategy), segment_size, waves_per_block, _stream(stream)))
    if workspace is None:
        workspace = torch.empty(max(need.value, 256), dtype=torch.uint8, device=x.device)
    have = ctypes.c_size_t(_workspace_bytes(workspace, x.device, need.value))
    _check(fn(_ptr(x), _ptr(out), n, _ptr(workspace), ctypes.byref(have), int(strategy), segment_size, waves_per_block, _stream(stream)))
    return workspace


def full_reduce(x, strategy=FullStrategy.AUTO, segment_size=0, waves_per_block=0, out=None, workspace=None, stream=None):
    torch = _torch()
    _need_f16(x, "x")
    if out is None:
        out = torch.empty(1, dtype=torch.float16, device=x.device)
    _workspace(lib().tcu_full_reduce_f16, x, out, x.numel(), strategy, segment_size, waves_per_block, workspace, stream)
    return out


def full_scan(x, strategy=FullStrategy.AUTO, segment_size=0, waves_per_block=0, out=None, workspace=None, stream=None):
    torch = _torch()
    _need_f16(x, "x")
    if out is None:
        out = torch.empty_like(x)
    _workspace(lib().tcu_full_scan_f16, x, out, x.numel(), strategy, segment_size, waves_per_block, workspace, stream)
    return out


def full_workspace_bytes(kind, n, strategy=FullStrategy.AUTO, segment_size=0, waves_per_block=0):
    fn = lib().tcu_full_reduce_f16 if kind == "reduce" else lib().tcu_full_scan_f16
    need = ctypes.c_size_t(0)
    _check(fn(None, None, n, None, ctypes.byref(need), int(strategy), segment_size, waves_per_block, None))
    return need.value


def _out_entry(t, what, f32_entry, f16_entry):
    torch = _torch()
    if t.dtype == torch.float32:
        return f32_entry
    if t.dtype == torch.float16:
        return f16_entry
    raise TypeError(f"{what} must be a float32 or float16 tensor")


def gemv(A, x, alpha=1.0, beta=0.0, y=None, variant=Variant.AUTO, stream=None, out_dtype=None):
    """y = alpha*A@x + beta*y; A (M,K) row-major fp16, x (K,) fp16, y (M,) fp32 or fp16.

    The dtype of `y` (or `out_dtype` when y is None; default float32) selects
    tcu_gemv_f16_f32 or tcu_gemv_f16_f16."""
    torch = _torch()
    _need_f16(A, "A")
    _need_f16(x, "x")
    M, K = A.shape
    if y is None:
        y = torch.zeros(M, dtype=out_dtype or torch.float32, device=A.device)
    entry = _out_entry(y, "y", lib().tcu_gemv_f16_f32, lib().tcu_gemv_f16_f16)
    _check(entry(_ptr(A), _ptr(x), _ptr(y), M, K, alpha, beta, int(variant), _stream(stream)))
    return y


def gemv_col_major(At, x, alpha=1.0, beta=0.0, y=None, stream=None, out_dtype=None):
    """y = alpha*A@x + beta*y with A column-major: `At` is the (K, M) fp16 tensor whose row k is column k of A (rows may be
    further apart than M elements: lda = At.stride(0)); x (K,) fp16, y (M,) fp32 or fp16 (tcu_gemv_col_major_f16_f32 / _f16)."""
    torch = _torch()
    _need_f16(x, "x")
    if At.dtype != torch.float16 or not At.is_cuda or At.dim() != 2 or At.stride(1) != 1:
        raise ValueError("At must be a CUDA float16 matrix that holds the columns of A contiguously (stride 1 along its second dimension)")
    K, M = At.shape
    if y is None:
        y = torch.zeros(M, dtype=out_dtype or torch.float32, device=At.device)
    entry = _out_entry(y, "y", lib().tcu_gemv_col_major_f16_f32, lib().tcu_gemv_col_major_f16_f16)
    _check(entry(ctypes.c_void_p(At.data_ptr()), At.stride(0) if K > 1 else M, _ptr(x), _ptr(y), M, K, alpha, beta, _stream(stream)))
    return y


def gemm(A, Bt, alpha=1.0, beta=0.0, C=None, out=None, variant=Variant.AUTO, stream=None, out_dtype=None):
    """D = alpha*A@B + beta*C with A (M,K) fp16 and B given column-major, i.e. as Bt (N,K) fp16.

    C and D are float32 (tcu_gemm_f16_f32) or float16 (tcu_gemm_f16_f16): the dtype of `out`,
    else of `C`, else `out_dtype` (default float32)."""
    torch = _torch()
    _need_f16(A, "A")
    _need_f16(Bt, "Bt")
    M, K = A.shape
    N, K2 = Bt.shape
    if K != K2:
        raise ValueError("A and Bt disagree on K")
    if out is None:
        out = torch.empty(M, N, dtype=C.dtype if C is not None else (out_dtype or torch.float32), device=A.device)
    if C is not None and C.dtype != out.dtype:
        raise TypeError("C and out must have the same dtype")
    entry = _out_entry(out, "out", lib().tcu_gemm_f16_f32, lib().tcu_gemm_f16_f16)
    _check(entry(_ptr(A), _ptr(Bt), _ptr(C), _ptr(out), M, N, K, alpha, beta, int(variant), _stream(stream)))
    return out


# ---- recurrent blocks of language models ------------------------------------------------------------------------


_dtype_codes = {}


def _dtype_code(t, name):
    if not _dtype_codes:
        torch = _torch()
        _dtype_codes.update({torch.float16: 0, torch.bfloat16: 1, torch.float32: 2})
    code = _dtype_codes.get(t.dtype)
    if code is None:
        raise TypeError(f"{name} must be a float16, bfloat16 or float32 tensor")
    if not t.is_cuda:
        raise ValueError(f"{name} must be a CUDA tensor")
    return code


_enum_values = {}


def _enum(kind, value):
    """The number of a member of the enumeration `kind`, given the member, its number or its name in any case."""
    known = _enum_values.get((kind, value))
    if known is None:
        if isinstance(value, str):
            if value.upper() not in kind.__members__:
                raise ValueError(f"{value!r} is none of {', '.join(m.name.lower() for m in kind)}")
            known = int(kind[value.upper()])
        else:
            known = int(kind(value))
        _enum_values[(kind, value)] = known
    return known


def _matrix(t, name, like=None):
    """(pointer, rows, row stride) of a tensor whose leading dimensions can be read as one: rows of contiguous elements at an even distance."""
    sizes = t.shape
    if like is not None and not (sizes == like.shape and t.dtype is like.dtype and t.get_device() == like.get_device()):
        raise ValueError(f"{name} must have the shape, type and device of the other operands ({tuple(like.shape)}, {like.dtype}, {like.device}); got {tuple(sizes)}, {t.dtype}, {t.device}")
    if len(sizes) < 2:
        raise ValueError(f"{name} must have at least two dimensions")
    width = sizes[-1]
    if t.is_contiguous():
        return t.data_ptr(), sizes[0] if len(sizes) == 2 else sizes[:-1].numel(), width
    strides = t.stride()
    if width > 1 and strides[-1] != 1:
        raise ValueError(f"{name} must be contiguous along its last dimension")
    rows, stride, ok = 1, None, True
    for n, s in zip(reversed(sizes[:-1]), reversed(strides[:-1])):
        if n != 1:
            if stride is None:
                stride = s
            elif s != stride * rows:
                ok = False
            rows *= n
    if rows > 1 and not ok:
        raise ValueError(f"the rows of {name} are not evenly spaced: pass a contiguous tensor")
    return t.data_ptr(), rows, width if stride is None or rows <= 1 else stride


def _vector_f32(t, name, shape, device):
    if t is None:
        return None
    if not (t.dtype is _torch().float32 and t.shape == shape and t.is_contiguous() and t.device == device):
        raise ValueError(f"{name} must be a contiguous float32 tensor of shape {tuple(shape)} on {device}")
    return t.data_ptr()


_current = None


def _current_calls():
    """(current device, raw handle of a device's current stream), without the objects around them where this torch has such calls: 4 us less."""
    global _current
    if _current is None:
        torch = _torch()
        _current = (getattr(torch._C, "_cuda_getDevice", torch.cuda.current_device),
                    getattr(torch._C, "_cuda_getCurrentRawStream", lambda index: torch.cuda.current_stream(index).cuda_stream))
    return _current


def _launches(fn):
    """Runs a function whose `stream` is a raw handle on the stream asked for, or the current one of its first operand's device, with
    that device and stream current: what it allocates belongs to that stream."""
    first = fn.__code__.co_varnames[0]

    @functools.wraps(fn)
    def call(*args, stream=None, **kw):
        torch = _torch()
        operand = args[0] if args else kw.get(first)
        if not (isinstance(operand, torch.Tensor) and operand.is_cuda):
            raise ValueError(f"{first} must be a CUDA tensor")
        index = operand.get_device()
        if stream is not None:
            if stream.device != operand.device:
                raise ValueError(f"the stream belongs to {stream.device}, the tensors to {operand.device}")
            with torch.cuda.stream(stream):
                return fn(*args, stream=stream.cuda_stream, **kw)
        current_device, raw_stream = _current or _current_calls()
        if current_device() == index:
            return fn(*args, stream=raw_stream(index), **kw)
        with torch.cuda.device(index):
            return fn(*args, stream=raw_stream(index), **kw)

    return call


def _new(t):
    """An uninitialised contiguous tensor like t."""
    torch = _torch()
    return torch.empty_like(t) if t.is_contiguous() else t.new_empty(t.shape)


def _result(given, name, like):
    """(tensor, pointer, row stride): the tensor given for a result like `like`, or a new one."""
    if given is None:
        t = _new(like)
        return t, t.data_ptr(), like.shape[-1]
    p, _, stride = _matrix(given, name, like)
    return given, p, stride


def _new_f32(t, shape):
    return t.new_empty(shape, dtype=_torch().float32)


_untouched = {}


def _untouched_workspace(device):
    """256 bytes for the calls that ask for no more: they keep nothing there, so one piece of memory serves them all."""
    ws = _untouched.get(device)
    if ws is None:
        ws = _untouched[device] = _torch().empty(256, dtype=_torch().uint8, device=device)
    return ws


# Workspace sizes by entry point and sizes of the operands, so that the size is asked for once and not at every call.
_workspace_sizes = {}


def _call_with_workspace(fn, args, sizes, workspace, device, raw):
    """fn(*args, workspace, its size, stream) with the caller's workspace, or a new one of the size the call needs."""
    if workspace is not None:
        have = ctypes.c_size_t(_workspace_bytes(workspace, device, 256))
        _check(fn(*args, workspace.data_ptr(), ctypes.byref(have), raw))
        return
    torch = _torch()
    key = (fn.__name__, *sizes)
    size = _workspace_sizes.get(key, 0)
    have = ctypes.c_size_t(size)
    if size:
        ws = _untouched_workspace(device) if size == 256 else torch.empty(size, dtype=torch.uint8, device=device)
        rc = fn(*args, ws.data_ptr(), ctypes.byref(have), raw)
        if rc != 4:  # the size also goes by the operands' alignment: another one may need more
            return _check(rc)
    _check(fn(*args, None, ctypes.byref(have), None))
    if len(_workspace_sizes) >= 1024:
        _workspace_sizes.clear()
    _workspace_sizes[key] = have.value
    ws = torch.empty(have.value, dtype=torch.uint8, device=device)
    _check(fn(*args, ws.data_ptr(), ctypes.byref(have), raw))


def _scan_shape(x, gate, offsets, name="x"):
    torch = _torch()
    dtype = _dtype_code(x, name)
    s = GatedScanShape(dtype=dtype, gate=_enum(Gate, gate), channels=x.shape[-1])
    if offsets is not None:
        if x.dim() != 2:
            raise ValueError(f"with offsets {name} is a matrix of all rows")
        if offsets.dtype not in (torch.int32, torch.int64) or offsets.device != x.device or offsets.dim() != 1 or offsets.numel() < 1 or not offsets.is_contiguous():
            raise ValueError("offsets must be a contiguous int32 or int64 vector on the same device, one entry more than there are sequences")
        s.num_rows, s.num_sequences = x.shape[0], offsets.numel() - 1
        s.d_offsets, s.offset_bits = offsets.data_ptr(), 32 if offsets.dtype == torch.int32 else 64
    else:
        if x.dim() not in (2, 3):
            raise ValueError(f"{name} must be (sequences, tokens, channels), or (tokens, channels) of one sequence")
        s.num_sequences = x.shape[0] if x.dim() == 3 else 1
        s.sequence_length = x.shape[-2]
        s.num_rows = s.num_sequences * s.sequence_length
    return s


@_launches
def gated_scan(x, g, gate=Gate.SIGMOID, h0=None, offsets=None, out=None, h_last=None, workspace=None, *, stream=None):
    """h[t] = a[t] h[t-1] + b[t] along each sequence (tcu_gated_scan): returns (h, h_last).

    x, g: (sequences, tokens, channels) or (tokens, channels), float16, bfloat16 or float32, or with `offsets` (int32 or
    int64, one more than there are sequences, not decreasing) the rows of all sequences as one matrix.  gate: a Gate, or its
    name: "decay" (a = g, b = x), "log" (a = exp(g), b = x), "sigmoid" (a = sigmoid(g), b = (1 - a) x).  h0, h_last:
    (sequences, channels) float32, the states in front of and behind the sequences.  Rows outside all sequences
    are left as they are in `out`, and zero in a result this call allocates.  out may be x or g."""
    s = _scan_shape(x, gate, offsets)
    states = (s.num_sequences, s.channels)
    px, _, sx = _matrix(x, "x")
    pg, _, sg = _matrix(g, "g", x)
    p0 = _vector_f32(h0, "h0", states, x.device)
    s.zero_outside = out is None

    h, ph, sh = _result(out, "out", x)
    last = _new_f32(x, states) if h_last is None else h_last
    args = (ctypes.byref(s), px, sx, pg, sg, ph, sh, p0, _vector_f32(last, "h_last", states, x.device))
    _call_with_workspace(lib().tcu_gated_scan, args, (s.dtype, s.num_rows, s.channels, offsets is None), workspace, x.device, stream)
    return h, last


@_launches
def gated_scan_backward(dh, x, g, h, gate=Gate.SIGMOID, h0=None, dh_last=None, offsets=None, dx=None, dg=None, workspace=None, *, stream=None):
    """The gradient of gated_scan (tcu_gated_scan_backward): returns (dx, dg, dh0).

    dh, dh_last: gradients with respect to h and h_last (dh_last may be None); h: what gated_scan returned; x is read for
    the sigmoid gate only and may be None for the others.  dh0 is (sequences, channels) float32.  dx and dg may be given
    (both or neither), and be dh, x or g; rows outside all sequences are then left as they are, and otherwise zero."""
    s = _scan_shape(g, gate, offsets, "g")
    states = (s.num_sequences, s.channels)
    if x is None and s.gate == Gate.SIGMOID:
        raise ValueError("the sigmoid gate's gradient needs x")
    px, _, sx = _matrix(x, "x", g) if x is not None else (None, 0, 0)
    pg, _, sg = _matrix(g, "g")
    pd, _, sd = _matrix(dh, "dh", g)
    ph, _, sh = _matrix(h, "h", g)
    p0, pl = _vector_f32(h0, "h0", states, g.device), _vector_f32(dh_last, "dh_last", states, g.device)
    if (dx is None) != (dg is None):
        raise ValueError("dx and dg are given both or neither")
    s.zero_outside = dx is None

    (out_x, pox, sox), (out_g, pog, sog) = _result(dx, "dx", g), _result(dg, "dg", g)
    dh0 = _new_f32(g, states)
    args = (ctypes.byref(s), pd, sd, px, sx, pg, sg, ph, sh, p0, pl, pox, sox, pog, sog, dh0.data_ptr())
    _call_with_workspace(lib().tcu_gated_scan_backward, args, (s.dtype, s.num_rows, s.channels, offsets is None), workspace, g.device, stream)
    return out_x, out_g, dh0


@_launches
def gated_scan_step(x, g, state, gate=Gate.SIGMOID, slots=None, new_state=None, out=None, *, stream=None):
    """One token for each running sequence (tcu_gated_scan_step): returns h (rows, channels).

    x, g: (rows, channels); state: (slots, channels) float32; slots: int32, the slot of each row (None: row i uses slot i; a
    negative or too large one marks padding, whose row of `out` is left as it is, or zero in a result this call allocates).  The new states go to `new_state`, by
    default `state` itself; slots that no row names are not written."""
    torch = _torch()
    dtype = _dtype_code(x, "x")
    if x.dim() != 2:
        raise ValueError("x must be (rows, channels)")
    rows, channels = x.shape
    px, _, sx = _matrix(x, "x")
    pg, _, sg = _matrix(g, "g", x)
    if state.dim() != 2:
        raise ValueError("state must be (slots, channels)")
    shape = (state.shape[0], channels)
    ps = _vector_f32(state, "state", shape, x.device)
    pn = ps if new_state is None else _vector_f32(new_state, "new_state", shape, x.device)
    if slots is not None and (slots.dtype != torch.int32 or slots.device != x.device or tuple(slots.shape) != (rows,) or not slots.is_contiguous()):
        raise ValueError("slots must be a contiguous int32 vector with one entry per row, on the same device")

    h, ph, sh = _result(out, "out", x)
    _check(lib().tcu_gated_scan_step(dtype, _enum(Gate, gate), channels, rows, px, sx, pg, sg, ph, sh, ps, pn, shape[0], slots.data_ptr() if slots is not None else None, out is None, stream))
    return h


def _vector(t, name, n, like):
    """Pointer of a vector operand of `like`'s type with n entries (None: null)."""
    if t is None:
        return None
    if not (t.dtype is like.dtype and t.shape == (n,) and t.is_contiguous() and t.get_device() == like.get_device()):
        raise ValueError(f"{name} must be a contiguous vector of {n} entries of {like.dtype} on {like.device}")
    return t.data_ptr()


_ADD_NORM = int(NormOrder.ADD_NORM)


def _optional(t, name, like):
    return (None, 0) if t is None else _matrix(t, name, like)[::2]


def _norm_shape(x, gate, norm, order, activation, eps, scale, name):
    dtype = _dtype_code(x, name)
    if activation is None:
        activation = "none" if gate is None else "silu"
    p, rows, stride = _matrix(x, name)
    return p, stride, FusedNormShape(dtype=dtype, norm=_enum(Norm, norm), order=_enum(NormOrder, order), activation=_enum(Activation, activation), rows=rows, dim=x.shape[-1], eps=eps, scale=scale)


@_launches
def fused_norm(x, weight=None, bias=None, residual=None, gate=None, scale=1.0, channel_scale=None, norm=Norm.RMS, order=NormOrder.ADD_NORM, activation=None, eps=1e-6, out=None, residual_out=None, *, stream=None):
    """Norm of every row of x (..., dim), fused with a residual, its scale and a gate (tcu_fused_norm); s = scale * channel_scale.

    order "add_norm": z = residual + s x, returns (act(gate) y(z), z), or act(gate) y(x) alone without a residual.
    order "norm_add": returns residual + s act(gate) y(x).  y is the rms or layer norm times weight plus bias.
    activation: of the gate, by default silu.  weight, bias, channel_scale: vectors of x's type."""
    px, sx, s = _norm_shape(x, gate, norm, order, activation, eps, scale, "x")
    pr, pg = _optional(residual, "residual", x), _optional(gate, "gate", x)
    dim = x.shape[-1]
    vectors = _vector(weight, "weight", dim, x), _vector(bias, "bias", dim, x), _vector(channel_scale, "channel_scale", dim, x)
    keep = s.order == _ADD_NORM and residual is not None
    if residual_out is not None and not keep:
        raise ValueError("residual_out goes with the order add_norm and a residual")

    o, po, so = _result(out, "out", x)
    z, pz, sz = _result(residual_out, "residual_out", x) if keep else (None, None, 0)
    _check(lib().tcu_fused_norm(ctypes.byref(s), px, sx, *pr, *pg, *vectors, po, so, pz, sz, stream))
    return (o, z) if keep else o


@_launches
def fused_norm_backward(dout, z, weight=None, bias=None, gate=None, scale=1.0, channel_scale=None, x=None, dresidual_out=None, norm=Norm.RMS, order=NormOrder.ADD_NORM, activation=None, eps=1e-6, workspace=None, residual_gradient=None, *, stream=None):
    """The gradient of fused_norm (tcu_fused_norm_backward): a dict with "dx" and, where the operand is there, "dgate",
    "dweight", "dbias", "dscale" (of channel_scale) and "dresidual".

    z: what was normed: the residual_out of the forward call (order add_norm with a residual), else its x.  order add_norm:
    dresidual_out is the gradient with respect to residual_out (None: nothing came from it) and "dresidual" is returned if it is given, or as
    residual_gradient says; the gradient of channel_scale needs the forward call's x.  order norm_add: the residual's gradient is dout itself.  The vectors'
    gradients are float32."""
    pd, sd, s = _norm_shape(dout, gate, norm, order, activation, eps, scale, "dout")
    add_norm = s.order == _ADD_NORM
    pz, pg = _matrix(z, "z", dout)[::2], _optional(gate, "gate", dout)
    vectors = [_vector(t, n, s.dim, dout) for t, n in ((weight, "weight"), (bias, "bias"), (channel_scale, "channel_scale"))]
    ps = _optional(dresidual_out, "dresidual_out", dout)
    if add_norm and channel_scale is not None and x is None:
        raise ValueError("the gradient of channel_scale needs x")
    px = _optional(x if add_norm and channel_scale is not None else None, "x", dout)

    new = lambda: _new(dout)
    column = lambda: _new_f32(dout, s.dim)
    got = {"dx": new()}
    if gate is not None:
        got["dgate"] = new()
    if dresidual_out is not None if residual_gradient is None else residual_gradient:
        got["dresidual"] = new()
    for name, t in (("dweight", weight), ("dbias", bias), ("dscale", channel_scale)):
        if t is not None:
            got[name] = column()
    args = (ctypes.byref(s), pd, sd, *pz, *pg, *vectors, *px, *ps, *(v for n in ("dx", "dgate", "dresidual") for v in ((got[n].data_ptr(), s.dim) if n in got else (None, 0))),
            *(got[n].data_ptr() if n in got else None for n in ("dweight", "dbias", "dscale")))
    _call_with_workspace(lib().tcu_fused_norm_backward, args, (s.dtype, s.rows, s.dim, weight is None, bias is None, channel_scale is None), workspace, dout.device, stream)
    return got


def _operand(t, name, rows, columns, like):
    """(pointer, leading dimension) of a matrix operand of the fused product (None: null)."""
    if t is None:
        return None, 0
    if t.dtype is not like.dtype or t.get_device() != like.get_device():
        raise ValueError(f"{name} must have the type and device of the other operands ({like.dtype}, {like.device})")
    p, n, stride = _matrix(t, name)
    if n != rows or t.shape[-1] != columns:
        raise ValueError(f"{name} must be {rows} x {columns}; got {tuple(t.shape)}")
    return p, stride


@_launches
def fused_gemm(A, Bt, bias=None, activation=Activation.NONE, C=None, beta=1.0, out=None, preactivation=None, return_preactivation=False, workspace=None, *, stream=None):
    """D = act(A @ Bt.T + bias) + beta * C (tcu_fused_gemm): A (..., K), Bt (N, K), bias (N,), C and D (..., N), float16 or bfloat16.

    Returns D, or with return_preactivation or a `preactivation` tensor to fill (D, A @ Bt.T + bias); the second is what
    fused_gemm_backward wants as Z.  C is not read when beta is 0; out may be C."""
    dtype = _dtype_code(A, "A")
    pa, M, lda = _matrix(A, "A")
    if Bt.dim() != 2 or Bt.shape[-1] != A.shape[-1]:
        raise ValueError("Bt must be (N, K) with the K of A")
    N, K = Bt.shape
    s = FusedGemmShape(dtype=dtype, activation=_enum(Activation, activation), M=M, N=N, K=K, beta=beta if C is not None else 0.0)
    pb, pbias, pc = _operand(Bt, "Bt", N, K, A), _vector(bias, "bias", N, A), _operand(C, "C", M, N, A)

    def result(given, name):
        if given is not None:
            return (given, *_operand(given, name, M, N, A))
        t = A.new_empty((*A.shape[:-1], N))
        return t, t.data_ptr(), N

    D, *pd = result(out, "out")
    Z, *pz = result(preactivation, "preactivation") if return_preactivation or preactivation is not None else (None, None, 0)
    args = (ctypes.byref(s), pa, lda, *pb, pbias, *pc, *pd, *pz)
    _call_with_workspace(lib().tcu_fused_gemm, args, (M, N, K), workspace, A.device, stream)
    return D if Z is None else (D, Z)


@_launches
def fused_gemm_backward(dD, A, Bt, Z=None, activation=Activation.NONE, bias_gradient=True, input_gradient=True, weight_gradient=True, workspace=None, *, stream=None):
    """The gradient of fused_gemm (tcu_fused_gemm_backward): a dict with "dA" (like A), "dB" (like Bt) and "dbias" (float32),
    those that are asked for.  Z: what fused_gemm returned as the activation's argument; the gradient of C is beta * dD."""
    dtype = _dtype_code(A, "A")
    pa, M, lda = _matrix(A, "A")
    if Bt.dim() != 2 or Bt.shape[-1] != A.shape[-1]:
        raise ValueError("Bt must be (N, K) with the K of A")
    N, K = Bt.shape
    s = FusedGemmShape(dtype=dtype, activation=_enum(Activation, activation), M=M, N=N, K=K)
    pd, pb, pz = _operand(dD, "dD", M, N, A), _operand(Bt, "Bt", N, K, A), _operand(Z, "Z", M, N, A)

    got = {}
    if input_gradient:
        got["dA"] = _new(A)
    if weight_gradient:
        got["dB"] = _new(Bt)
    if bias_gradient:
        got["dbias"] = _new_f32(A, N)
    args = (ctypes.byref(s), *pd, pa, lda, *pb, *pz, *(v for n in ("dA", "dB") for v in ((got[n].data_ptr(), K) if n in got else (None, 0))), got["dbias"].data_ptr() if bias_gradient else None)
    _call_with_workspace(lib().tcu_fused_gemm_backward, args, (M, N, K, s.activation == 0, input_gradient, weight_gradient, bias_gradient), workspace, A.device, stream)
    return got


def fill(t, value, stream=None):
    _need_f16(t, "t")
    _check(lib().tcu_fill_f16(_ptr(t), value, t.numel(), _stream(stream)))
    return t


def convert_f32_to_f16(src, out=None, stream=None):
    torch = _torch()
    if out is None:
        out = torch.empty(src.shape, dtype=torch.float16, device=src.device)
    _check(lib().tcu_convert_f32_to_f16(_ptr(out), _ptr(src), src.numel(), _stream(stream)))
    return out


def generate(n, seed, dist=Dist.UNIFORM, first=0, out=None, device="cuda", stream=None):
    torch = _torch()
    if out is None:
        out = torch.empty(n, dtype=torch.float16, device=device)
    _check(lib().tcu_generate_f16(_ptr(out), n, seed & 0xFFFFFFFFFFFFFFFF, int(dist), first, _stream(stream)))
    return out


def stream_probe(dst, src, nbytes, mode, tiles_per_wave=0, waves_per_block=0, stream=None):
    _check(lib().tcu_stream_probe(_ptr(dst), _ptr(src), nbytes, mode, tiles_per_wave, waves_per_block, _stream(stream)))


def temporary_allocations():
    """How many times the library has taken temporary device memory since the process began."""
    return int(lib().tcu_temporary_allocations())


def time_next_launch(start, stop):
    """The next kernel launched through the library stamps the torch events `start` and `stop`
    (enable_timing=True, already recorded once so that their handles exist) with its own begin
    and end: start.elapsed_time(stop) is then the kernel's duration."""
    _check(lib().tcu_time_next_launch(start.cuda_event, stop.cuda_event))


def lane_probe(device="cuda", stream=None):
    torch = _torch()
    words = ctypes.c_size_t(0)
    _check(lib().tcu_lane_probe(None, ctypes.byref(words), None))
    out = torch.zeros(words.value, dtype=torch.int32, device=device)
    _check(lib().tcu_lane_probe(_ptr(out), ctypes.byref(words), _stream(stream)))
    return out
