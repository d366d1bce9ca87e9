"""ctypes binding of libgonngpu.so, the MI355X GEMM / SpMM backend (C ABI in
include/gonngpu.h).

This module only marshals arguments: every computation runs in the HIP library.
If the library is missing, importing works but the first call raises
GonngpuUnavailable; there is no CPU fallback.
"""
from __future__ import annotations

import ctypes
import functools
import os
import re
import threading

import numpy as np

PKG_DIR = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
REPO_DIR = os.path.dirname(PKG_DIR)
LIB_PATH = os.path.join(PKG_DIR, "lib", "libgonngpu.so")
HEADER_PATH = os.path.join(REPO_DIR, "include", "gonngpu.h")

GN_F32, GN_F16, GN_MXFP4 = 0, 1, 2
ROUND_NEAREST_EVEN, ROUND_TOWARD_ZERO = 0, 1
ACT_NONE, ACT_RELU, ACT_SIGMOID, ACT_TANH, ACT_LEAKY_RELU, ACT_ELU, ACT_SWISH, ACT_GELU = -1, 0, 1, 2, 4, 5, 6, 7


class GonngpuUnavailable(RuntimeError):
    pass


class GonngpuError(RuntimeError):
    def __init__(self, code, message):
        super().__init__(f"gonngpu error {code}: {message}")
        self.code = code
        self.message = message


class CError(ctypes.Structure):
    _fields_ = [("message", ctypes.c_void_p)]


_VP = ctypes.c_void_p
_L = ctypes.c_long
_I = ctypes.c_int
_F = ctypes.c_float
_SZ = ctypes.c_size_t
_U64 = ctypes.c_uint64
_ERR = ctypes.POINTER(CError)

SIGNATURES = {
    "create_gpu_buffer": (_I, [_VP, _L, ctypes.POINTER(_VP), ctypes.POINTER(_VP), _ERR]),
    "retrieve_gpu_buffer_data": (_I, [_VP, _VP, _L, _ERR]),
    "release_gpu_buffer": (_I, [_VP]),
    "perform_mps_matrix_multiplication": (_I, [_VP, _L, _L, _VP, _L, _L, _VP, _L, _L, _VP, _ERR]),
    "perform_mps_matrix_transpose": (_I, [_VP, _L, _L, _VP, _L, _L, _VP, _ERR]),
    "perform_optimized_gemm": (_I, [_VP, _VP, _VP, _L, _L, _L, _F, _F, _VP, _ERR]),
    "perform_batch_matmul_optimized": (_I, [_VP, _VP, _VP, _L, _L, _L, _L, _VP, _ERR]),
    "perform_fused_linear_activation": (_I, [_VP, _L, _L, _VP, _L, _VP, _I, _F, _VP, _VP, _ERR]),
    "perform_sparse_dense_matmul": (_I, [_VP, _VP, _L, _VP, _L, _L, _L, _L, _VP, _L, _L, _VP, _L, _L, _VP, _ERR]),
    "perform_sparse_matvec": (_I, [_VP, _VP, _L, _VP, _L, _L, _L, _L, _VP, _L, _VP, _L, _VP, _ERR]),
    "perform_sparse_sparse_matmul": (_I, [_VP, _VP, _L, _VP, _L, _L, _L, _L, _VP, _VP, _L, _VP, _L, _L, _L, _L, _VP,
                                          _L, _L, _VP, _ERR]),
    "perform_dense_sparse_matmul": (_I, [_VP, _L, _L, _VP, _VP, _L, _VP, _L, _L, _L, _L, _VP, _L, _L, _VP, _ERR]),
    "perform_sparse_add": (_I, [_VP, _VP, _L, _VP, _L, _L, _L, _L, _VP, _VP, _L, _VP, _L, _L, _L, _L, _VP, _VP, _VP,
                                ctypes.POINTER(_L), _L, _VP, _ERR]),
    "perform_sparse_scalar_multiply": (_I, [_VP, _VP, _L, _VP, _L, _L, _L, _L, _F, _VP, _ERR]),
    "perform_sparse_to_dense": (_I, [_VP, _VP, _L, _VP, _L, _L, _L, _L, _VP, _L, _L, _VP, _ERR]),
    "perform_dense_to_sparse": (_I, [_VP, _L, _L, _F, _VP, _VP, _VP, ctypes.POINTER(_L), _L, _VP, _ERR]),
    "free_c_error_message": (None, [_VP]),
    "gn_version": (ctypes.c_char_p, []),
    "gn_init": (_I, [_ERR]),
    "gn_stream": (_VP, []),
    "gn_device": (_I, []),
    "gn_buffer_device_ptr": (_VP, [_VP]),
    "gn_buffer_bytes": (_L, [_VP]),
    "gn_memory_stats": (None, [ctypes.POINTER(_L), ctypes.POINTER(_L), ctypes.POINTER(_L)]),
    "gn_malloc": (_I, [ctypes.POINTER(_VP), _SZ, _ERR]),
    "gn_free": (_I, [_VP]),
    "gn_free_async": (_I, [_VP, _VP]),
    "gn_csr_indices_changed": (_I, [_VP]),
    "gn_synchronize": (_I, [_VP, _ERR]),
    "gn_gemm": (_I, [_I, _I, _I, _L, _L, _L, _F, _VP, _L, _L, _VP, _L, _L, _F, _VP, _L, _L, _L, _VP, _I, _F, _VP,
                     _ERR]),
    "gn_cast_f32_f16": (_I, [_VP, _VP, _SZ, _I, _VP, _ERR]),
    "gn_cast_f16_f32": (_I, [_VP, _VP, _SZ, _VP, _ERR]),
    "gn_activation_backward": (_I, [_VP, _VP, _L, _L, _I, _F, _F, _VP, _VP, _VP, _ERR]),
    "gn_activation_backward_noalloc": (_I, [_VP, _VP, _L, _L, _I, _F, _F, _VP, _VP, _VP, _ERR]),
    "gn_transpose_f32": (_I, [_VP, _L, _L, _VP, _VP, _ERR]),
    "gn_activation_forward": (_I, [_VP, _VP, _L, _I, _F, _VP, _ERR]),
    "createMPSGraph": (_VP, []),
    "createMatMulNode": (_VP, [_VP, _VP, _VP]),
    "createReLUNode": (_VP, [_VP, _VP]),
    "compileGraph": (_VP, [_VP, _VP]),
    "executeCompiledGraph": (None, [_VP, _VP, ctypes.POINTER(_VP), _L, ctypes.POINTER(_VP), _L]),
    "gn_graph_placeholder": (_VP, [_VP, _L, _L, _I]),
    "gn_graph_matmul": (_VP, [_VP, _VP, _VP, _I, _I]),
    "gn_graph_activation": (_VP, [_VP, _VP, _I, _F]),
    "gn_graph_compile": (_I, [_VP, ctypes.POINTER(_VP), _L, ctypes.POINTER(_VP), _L, ctypes.POINTER(_VP), _ERR]),
    "gn_graph_execute": (_I, [_VP, _VP, ctypes.POINTER(_VP), _L, ctypes.POINTER(_VP), _L, _ERR]),
    "gn_graph_release": (None, [_VP]),
    "gn_softmax_rows": (_I, [_VP, _VP, _L, _L, _VP, _ERR]),
    "perform_activation_relu_forward": (_I, [_VP, _L, _VP, _VP, _ERR]),
    "perform_activation_sigmoid_forward": (_I, [_VP, _L, _VP, _VP, _ERR]),
    "perform_activation_tanh_forward": (_I, [_VP, _L, _VP, _VP, _ERR]),
    "perform_activation_softmax_1d_forward": (_I, [_VP, _L, _VP, _VP, _ERR]),
    "perform_activation_softmax_2d_forward": (_I, [_VP, _L, _L, _VP, _VP, _ERR]),
    "perform_activation_leaky_relu_forward": (_I, [_VP, _L, _F, _VP, _VP, _ERR]),
    "perform_activation_elu_forward": (_I, [_VP, _L, _F, _VP, _VP, _ERR]),
    "perform_activation_swish_forward": (_I, [_VP, _L, _VP, _VP, _ERR]),
    "perform_activation_gelu_forward": (_I, [_VP, _L, _VP, _VP, _ERR]),
    "gn_mxfp4_size": (_I, [_L, _L, ctypes.POINTER(_SZ), ctypes.POINTER(_SZ), _ERR]),
    "gn_mxfp4_quantize": (_I, [_I, _VP, _L, _L, _L, _VP, _VP, _VP, _ERR]),
    "gn_mxfp4_dequantize": (_I, [_VP, _VP, _L, _L, _I, _VP, _L, _VP, _ERR]),
    "gn_mxfp4_gemm": (_I, [_I, _L, _L, _L, _F, _VP, _L, _VP, _VP, _VP, _F, _VP, _L, _VP, _I, _F, _VP, _ERR]),
    "gn_logits_workspace": (_SZ, [_L, _L, _I]),
    "gn_token_logprobs": (_I, [_I, _VP, _L, _L, _L, _F, _VP, _VP, _VP, _VP, _I, _VP, _VP, _VP, _SZ, _VP, _ERR]),
    "gn_token_logprobs_backward": (_I, [_I, _VP, _L, _L, _L, _F, _VP, _VP, _VP, _VP, _VP, _VP, _L, _VP, _ERR]),
    "gn_distill_forward": (_I, [_I, _VP, _L, _L, _L, _F, _VP, _VP, _I, _VP, _VP, _VP, _SZ, _VP, _ERR]),
    "gn_distill_backward": (_I, [_I, _VP, _L, _L, _L, _F, _VP, _VP, _I, _VP, _VP, _VP, _L, _VP, _ERR]),
    "gn_spmm_csr": (_I, [_L, _L, _L, _L, _VP, _VP, _VP, _VP, _L, _VP, _L, _VP, _VP, _ERR]),
    "gn_spmv_csr": (_I, [_L, _L, _L, _VP, _VP, _VP, _VP, _VP, _VP, _VP, _ERR]),
    "gn_spmv_plan_create": (_I, [_L, _L, _L, _VP, _VP, ctypes.POINTER(_VP), _VP, _ERR]),
    "gn_spmv_plan_run": (_I, [_VP, _VP, _VP, _VP, _VP, _VP, _ERR]),
    "gn_spmv_plan_release": (None, [_VP, _VP]),
    "gn_fill_uniform_f32": (_I, [_VP, _SZ, _U64, _U64, _F, _F, _VP, _ERR]),
    "gn_fill_normal_f32": (_I, [_VP, _SZ, _U64, _U64, _F, _F, _VP, _ERR]),
    # Part 3: the other reference-bridge entries with a device implementation. The rest of
    # Part 3 (entries that report "not provided") has no Python binding.
    "perform_mps_matrix_add": (_I, [_VP, _L, _L, _VP, _L, _L, _VP, _L, _L, _VP, _ERR]),
    "perform_mps_matrix_add_broadcast": (_I, [_VP, _L, _L, _VP, _L, _L, _VP, _L, _L, _VP, _ERR]),
    "perform_mps_matrix_subtract": (_I, [_VP, _L, _L, _VP, _L, _L, _VP, _L, _L, _VP, _ERR]),
    "perform_mps_matrix_element_multiply": (_I, [_VP, _L, _L, _VP, _L, _L, _VP, _L, _L, _VP, _ERR]),
    "perform_mps_matrix_element_divide": (_I, [_VP, _L, _L, _VP, _L, _L, _VP, _L, _L, _VP, _ERR]),
    "perform_mps_matrix_scalar_add": (_I, [_VP, _L, _L, _F, _VP, _VP, _ERR]),
    "perform_mps_matrix_scalar_multiply": (_I, [_VP, _L, _L, _F, _VP, _VP, _ERR]),
    "perform_activation_relu_backward": (_I, [_VP, _VP, _L, _VP, _VP, _ERR]),
    "perform_activation_sigmoid_backward": (_I, [_VP, _VP, _L, _VP, _VP, _ERR]),
    "perform_activation_tanh_backward": (_I, [_VP, _VP, _L, _VP, _VP, _ERR]),
    "perform_activation_softmax_1d_backward": (_I, [_VP, _VP, _L, _VP, _VP, _ERR]),
    "perform_activation_softmax_2d_backward": (_I, [_VP, _VP, _L, _L, _VP, _VP, _ERR]),
    "perform_activation_leaky_relu_backward": (_I, [_VP, _VP, _L, _F, _VP, _VP, _ERR]),
    "perform_activation_elu_backward": (_I, [_VP, _VP, _L, _F, _VP, _VP, _ERR]),
    "perform_activation_swish_backward": (_I, [_VP, _VP, _L, _VP, _VP, _ERR]),
    "perform_activation_gelu_backward": (_I, [_VP, _VP, _L, _VP, _VP, _ERR]),
    "getGPUMemoryUsage": (None, [ctypes.POINTER(_L), ctypes.POINTER(_L)]),
}

_lib = None


def header_symbols(path=HEADER_PATH):
    """Function names declared in include/gonngpu.h."""
    text = open(path).read()
    text = re.sub(r"/\*.*?\*/", "", text, flags=re.S)
    return sorted(set(re.findall(r"^\s*(?:const\s+)?[A-Za-z_][\w\s\*]*?\b([A-Za-z_][A-Za-z0-9_]*)\s*\(", text, flags=re.M)))


def load(path=LIB_PATH):
    """Loads the library (no device work). Raises GonngpuUnavailable if it is not built."""
    global _lib
    if _lib is not None:
        return _lib
    if not os.path.exists(path):
        raise GonngpuUnavailable(f"{path} is not built; run __graft_entry__.build()")
    L = ctypes.CDLL(path)
    for name, (res, args) in SIGNATURES.items():
        fn = getattr(L, name)
        fn.restype = res
        fn.argtypes = args
    _lib = L
    return L


def _check(rc, err):
    if rc != 0:
        msg = ""
        if err.message:
            msg = ctypes.string_at(err.message).decode(errors="replace")
            _lib.free_c_error_message(err.message)
            err.message = None
        raise GonngpuError(rc, msg)


_errors = threading.local()


def call(name, *args):
    """Calls a C-ABI entry point whose last argument is CError*; raises GonngpuError on failure. The CError is the
    thread's own, kept for its next call (a new one takes 0.5 us)."""
    L = load()
    err = getattr(_errors, "err", None)
    if err is None:
        err = _errors.err = CError()
        _errors.ref = ctypes.byref(err)
    rc = getattr(L, name)(*args, _errors.ref)
    _check(rc, err)
    return rc


def call_rc(name, *args):
    """Like call() but returns (code, message) instead of raising."""
    L = load()
    err = CError()
    rc = getattr(L, name)(*args, ctypes.byref(err))
    msg = ""
    if err.message:
        msg = ctypes.string_at(err.message).decode(errors="replace")
        L.free_c_error_message(err.message)
    return rc, msg


def init():
    call("gn_init")


def stream():
    return load().gn_stream()


def library_device():
    """Number of the GPU that the library's stream is on."""
    return load().gn_device()


def memory_stats():
    cur, peak, n = _L(), _L(), _L()
    load().gn_memory_stats(ctypes.byref(cur), ctypes.byref(peak), ctypes.byref(n))
    return cur.value, peak.value, n.value


# --------------------------------------------------------------------------- GPUPtr handles
class Buffer:
    """A library-owned device buffer (the GPUPtr of the reference bridge)."""

    def __init__(self, nbytes=None, data=None):
        self.handle = _VP()
        dev = _VP()
        if data is not None:
            self._host = np.ascontiguousarray(data)
            nbytes = self._host.nbytes
            src = self._host.ctypes.data_as(_VP)
        else:
            src = None
        call("create_gpu_buffer", src, int(nbytes), ctypes.byref(self.handle), ctypes.byref(dev))
        self.nbytes = int(nbytes)
        self.device = dev.value
        self._host = None

    @classmethod
    def from_array(cls, arr):
        return cls(data=np.ascontiguousarray(arr, dtype=np.float32))

    def to_array(self, shape, dtype=np.float32):
        out = np.empty(shape, dtype=dtype)
        call("retrieve_gpu_buffer_data", self.handle, out.ctypes.data_as(_VP), out.nbytes)
        return out

    @property
    def device_ptr(self):
        return load().gn_buffer_device_ptr(self.handle)

    def release(self):
        if self.handle and self.handle.value:
            load().release_gpu_buffer(self.handle)
            self.handle = _VP()

    def __del__(self):
        try:
            self.release()
        except Exception:
            pass


# --------------------------------------------------------------------------- device-pointer API
def _current_stream(device=None):
    """Handle of torch's current stream (on the current device). Building torch's Stream object for it takes 2.7 us, a
    third of what a small call costs the host; asking for the handle takes 0.4 us. The function for
    that is not part of torch's public interface: without it, the Stream object is built."""
    import torch

    try:
        raw = torch._C._cuda_getCurrentRawStream
    except AttributeError:
        return torch.cuda.current_stream().cuda_stream
    return raw(torch.cuda.current_device() if device is None else device)


def _run_ordered(name, *args):
    """Runs a device-pointer entry point ordered with torch's current stream.

    The C ABI takes a stream argument (NULL = the library's own stream). Torch
    tensors are produced on torch's current stream, so the call is issued on that
    stream; if it is the legacy default stream (handle 0), the device is
    synchronized around a call on the library stream instead."""
    sp = _current_stream()
    if sp:
        return call(name, *args, sp)
    import torch

    torch.cuda.synchronize()
    call(name, *args, None)
    call("gn_synchronize", None)


def _ptr(t):
    """Device address of a torch tensor / int / None."""
    if t is None:
        return None
    if isinstance(t, int):
        return t
    return t.data_ptr()


def gemm(A, B, C, *, transA=False, transB=False, alpha=1.0, beta=0.0, bias=None, act=ACT_NONE, act_alpha=0.0,
         M=None, N=None, K=None, lda=None, ldb=None, ldc=None, batch=1, strideA=0, strideB=0, strideC=0,
         dtype=None, stream_ptr=None):
    """C = act(alpha*op(A)*op(B) + beta*C + bias) on torch device tensors (row-major, last two dims)."""
    import torch

    if dtype is None:
        dtype = GN_F16 if A.dtype == torch.float16 else GN_F32
    a_rows, a_cols = A.shape[-2], A.shape[-1]
    b_rows, b_cols = B.shape[-2], B.shape[-1]
    M = M if M is not None else (a_cols if transA else a_rows)
    K = K if K is not None else (a_rows if transA else a_cols)
    N = N if N is not None else (b_rows if transB else b_cols)
    lda = lda if lda is not None else A.stride(-2)
    ldb = ldb if ldb is not None else B.stride(-2)
    ldc = ldc if ldc is not None else C.stride(-2)
    _dispatch(stream_ptr, "gn_gemm", dtype, int(transA), int(transB), M, N, K, alpha, _ptr(A), lda, strideA, _ptr(B),
              ldb, strideB, beta, _ptr(C), ldc, strideC, batch, _ptr(bias), act, act_alpha)


def cast_f32_f16(x, out, round_mode=ROUND_NEAREST_EVEN, stream_ptr=None):
    _dispatch(stream_ptr, "gn_cast_f32_f16", _ptr(x), _ptr(out), x.numel(), round_mode)


def cast_f16_f32(x, out, stream_ptr=None):
    _dispatch(stream_ptr, "gn_cast_f16_f32", _ptr(x), _ptr(out), x.numel())


def activation_backward(grad_out, pre, act, grad_in, grad_bias=None, alpha=0.0, scale=1.0, stream_ptr=None):
    """grad_in = grad_out * act'(pre) * scale; grad_bias = column sums of grad_in (optional)."""
    rows, cols = pre.shape
    _dispatch(stream_ptr, "gn_activation_backward", _ptr(grad_out), _ptr(pre), rows, cols, act, alpha, scale,
              _ptr(grad_in), _ptr(grad_bias))


def activation_forward(x, out, act, alpha=0.0, stream_ptr=None):
    """out = act(x) element-wise (ActivationType code other than Softmax, or ACT_NONE)."""
    _dispatch(stream_ptr, "gn_activation_forward", _ptr(x), _ptr(out), x.numel(), act, alpha)


def softmax_rows(x, out, stream_ptr=None):
    """Row-wise softmax of a 2-D tensor (a 1-D tensor is one row)."""
    rows, cols = (1, x.shape[0]) if x.dim() == 1 else (x.shape[0], x.shape[1])
    _dispatch(stream_ptr, "gn_softmax_rows", _ptr(x), _ptr(out), rows, cols)


def transpose(x, out, stream_ptr=None):
    _dispatch(stream_ptr, "gn_transpose_f32", _ptr(x), x.shape[0], x.shape[1], _ptr(out))


def _refuse(message):
    raise GonngpuError(-1, message)


_torch = _current_device = None


def _types():
    """torch, imported once at the first call that needs it (asking the import system each time costs a call 0.3 us)."""
    global _torch, _current_device
    if _torch is None:
        import torch

        # The function behind current_device() is not part of torch's public interface; asking it takes 0.2 us less.
        _current_device = getattr(torch._C, "_cuda_getDevice", torch.cuda.current_device)
        _torch = torch
    return _torch


def _device_of(first, *others):
    """The tensors' common device, which has to be the current one: kernels start there."""
    device = first.get_device()
    for t in others:
        if t is not None and t.get_device() != device:
            _refuse(f"tensors on {first.device} and {t.device}")
    if device < 0 or device != _current_device():
        _refuse(f"a tensor on {first.device}: all have to be on the current GPU")
    return device


def _expect(what, t, dtype, n):
    """Checks an argument that is a dense array of n values of the given type. (numel and is_contiguous take 0.06 us each,
    a size 0.1, the shape 0.7.)"""
    if t.dtype is not dtype or t.numel() != n or not t.is_contiguous():
        _refuse(f"{what}: {n} contiguous values of {dtype} are needed, got {t.dtype} {tuple(t.shape)}")


def _expect_rows(what, t, dtype, rows, width):
    """The same of an array of rows x width."""
    if t.dtype is not dtype or t.dim() != 2 or t.size(0) != rows or t.numel() != rows * width or not t.is_contiguous():
        _refuse(f"{what}: {rows} x {width} contiguous values of {dtype} are needed, got {t.dtype} {tuple(t.shape)}")


def _matrix(what, t):
    """(GN_F32 or GN_F16, rows, cols, elements from row to row) of a matrix whose rows are dense."""
    T = _types()
    dtype = t.dtype
    if dtype is T.float32:
        dtype = GN_F32
    elif dtype is T.float16:
        dtype = GN_F16
    else:
        _refuse(f"{what}: float32 or float16 is needed, got {t.dtype}")
    strides = t.stride()
    if len(strides) == 2:
        rows, cols = t.size(0), t.size(1)
        if (strides[1] == 1 or cols <= 1) and (strides[0] >= cols or rows <= 1):
            return dtype, rows, cols, (strides[0] if rows > 1 else cols)
    _refuse(f"{what}: a matrix of dense rows is needed, got shape {tuple(t.shape)}, strides {strides}")


def _mxfp4_matrix(what, data, scales, rows, cols):
    """Checks the two arrays of a stored MXFP4 matrix."""
    u8, groups = _types().uint8, -(-cols // 128)
    _expect_rows(what, data, u8, rows, 64 * groups)
    _expect_rows(what, scales, u8, rows, 4 * groups)


def _width(t):
    """k of a rows x k array."""
    return t.size(1) if t.dim() == 2 else -1


def _dispatch_on(device, stream_ptr, name, *args):
    """_dispatch for arguments whose device is known to be the current one. The library's own stream is on one device only:
    it does not stand in for the default stream of another."""
    ordered = stream_ptr is None
    if ordered:
        stream_ptr = _current_stream(device)
    if not stream_ptr:
        if device != library_device():
            _refuse(f"the library's stream is on GPU {library_device()}, the tensors are on GPU {device}: a stream of theirs is needed")
        if ordered:
            return _run_ordered(name, *args)
    return call(name, *args, stream_ptr)


def mxfp4_empty(rows, cols, device="cuda"):
    """The two arrays (codes, scales) of a rows x cols MXFP4 matrix, not filled in."""
    T = _types()
    groups = -(-cols // 128)
    return (T.empty((rows, 64 * groups), dtype=T.uint8, device=device),
            T.empty((rows, 4 * groups), dtype=T.uint8, device=device))


def mxfp4_quantize(x, data, scales, stream_ptr=None):
    """A float32 or float16 matrix brought to MXFP4, into the arrays of mxfp4_empty(*x.shape)."""
    dt, rows, cols, ld = _matrix("mxfp4_quantize", x)
    _mxfp4_matrix("mxfp4_quantize: data, scales", data, scales, rows, cols)
    device = _device_of(x, data, scales)
    _dispatch_on(device, stream_ptr, "gn_mxfp4_quantize", dt, x.data_ptr(), rows, cols, ld, data.data_ptr(), scales.data_ptr())


def mxfp4_dequantize(data, scales, out, stream_ptr=None):
    """The values of a stored MXFP4 matrix, to a float32 or float16 matrix of its size."""
    dt, rows, cols, ld = _matrix("mxfp4_dequantize", out)
    _mxfp4_matrix("mxfp4_dequantize: data, scales", data, scales, rows, cols)
    device = _device_of(data, scales, out)
    _dispatch_on(device, stream_ptr, "gn_mxfp4_dequantize", data.data_ptr(), scales.data_ptr(), rows, cols, dt, out.data_ptr(), ld)


def mxfp4_gemm(A, B, C, *, alpha=1.0, beta=0.0, bias=None, act=ACT_NONE, act_alpha=0.0, K=None, stream_ptr=None):
    """C = act(alpha*A*B^T + beta*C + bias) with B = (codes, scales) of an outputs x inputs MXFP4 matrix. A is a float16
    matrix, or a pair like B; then K is the number of columns (the arrays hold it rounded up to 128)."""
    T = _types()
    dtc, M, N, ldc = _matrix("mxfp4_gemm: C", C)
    if dtc != GN_F32:
        _refuse("mxfp4_gemm: C is float32")
    if isinstance(A, (tuple, list)):
        a, a_scales = A
        if K is None:
            K = 2 * _width(a)
        dt, lda = GN_MXFP4, 0
        _mxfp4_matrix("mxfp4_gemm: A", a, a_scales, M, K)
    else:
        a, a_scales = A, None
        dt, rows, cols, lda = _matrix("mxfp4_gemm: A", a)
        if dt != GN_F16 or K not in (None, cols):
            _refuse(f"mxfp4_gemm: A is float16 with K columns or a pair of MXFP4 arrays, got {a.dtype}, K = {K}")
        if rows != M:
            _refuse(f"mxfp4_gemm: {rows} rows of A, {M} of C")
        K = cols
    _mxfp4_matrix("mxfp4_gemm: B", B[0], B[1], N, K)
    if bias is not None:
        _expect("mxfp4_gemm: bias", bias, T.float32, N)
    device = _device_of(a, a_scales, B[0], B[1], C, bias)
    _dispatch_on(device, stream_ptr, "gn_mxfp4_gemm", dt, M, N, K, alpha, a.data_ptr(), lda, _ptr(a_scales), B[0].data_ptr(),
                 B[1].data_ptr(), beta, C.data_ptr(), ldc, _ptr(bias), act, act_alpha)


@functools.lru_cache(maxsize=256)
def _logits_workspace_bytes(rows, cols, k):
    return load().gn_logits_workspace(rows, cols, k)


def _logits_workspace(logits, rows, cols, k, device, stream_ptr):
    """Scratch for one call, from torch's allocator (which keeps what a captured graph uses), of the pool of the stream
    that the call runs on: a block of another stream's pool may still be in use there. A handle of 0 asked for is the library's
    stream, whereas torch's default stream, whose handle is 0 too, is None asked for (the call is then waited for). Asked
    for in the logits' type (the bytes are a multiple of 8): naming a type and a device takes 1.3 us more."""
    T = _types()
    n = _logits_workspace_bytes(rows, cols, k)
    if n == 0:
        return None, 0
    size = n // (4 if logits.dtype is T.float32 else 2)
    if stream_ptr is None:
        return logits.new_empty((size,)), n
    stream_ptr = stream_ptr or stream()
    if stream_ptr == _current_stream(device):
        return logits.new_empty((size,)), n
    with T.cuda.stream(T.cuda.ExternalStream(stream_ptr, device=device)):
        return logits.new_empty((size,)), n


def token_logprobs(logits, targets, logprob, *, lse=None, entropy=None, top_ids=None, top_logprobs=None,
                   temperature=1.0, stream_ptr=None):
    """logprob[r] = log softmax(logits[r] / temperature)[targets[r]] (int64; below 0: no target, 0), log-sum-exp
    and entropy of each row (float32), and the columns (int64) and log-probabilities of its k largest
    logits, k the width of top_ids, at most 64. targets and logprob may be None together."""
    T = _types()
    dt, rows, cols, ld = _matrix("token_logprobs", logits)
    if (targets is None) != (logprob is None) or (top_ids is None) != (top_logprobs is None):
        _refuse("token_logprobs: targets and logprob, and top_ids and top_logprobs, are given together")
    k = 0
    if top_ids is not None:
        k = _width(top_ids)
        _expect_rows("token_logprobs: top_ids", top_ids, T.int64, rows, k)
        _expect_rows("token_logprobs: top_logprobs", top_logprobs, T.float32, rows, k)
    if targets is not None:
        _expect("token_logprobs: targets", targets, T.int64, rows)
    for what, t in (("logprob", logprob), ("lse", lse), ("entropy", entropy)):
        if t is not None:
            _expect("token_logprobs: " + what, t, T.float32, rows)
    device = _device_of(logits, targets, logprob, lse, entropy, top_ids, top_logprobs)
    ws, n = _logits_workspace(logits, rows, cols, k, device, stream_ptr)
    _dispatch_on(device, stream_ptr, "gn_token_logprobs", dt, logits.data_ptr(), rows, cols, ld, temperature,
                 _ptr(targets), _ptr(logprob), _ptr(lse), _ptr(entropy), k, _ptr(top_ids), _ptr(top_logprobs),
                 _ptr(ws), n)


def token_logprobs_backward(logits, targets, lse, grad_logprob, grad_logits, *, entropy=None, grad_entropy=None,
                            temperature=1.0, stream_ptr=None):
    """The gradient of the logits (their type; may be the logits themselves) from those of logprob and, with
    the forward's entropy, of the entropy."""
    T = _types()
    dt, rows, cols, ld = _matrix("token_logprobs_backward", logits)
    dg, grows, gcols, ldg = _matrix("token_logprobs_backward: grad_logits", grad_logits)
    if (dg, grows, gcols) != (dt, rows, cols):
        _refuse("token_logprobs_backward: grad_logits has the type and shape of logits")
    if (targets is None) != (grad_logprob is None) or (entropy is None) != (grad_entropy is None):
        _refuse("token_logprobs_backward: targets and grad_logprob, and entropy and grad_entropy, are given together")
    if targets is not None:
        _expect("token_logprobs_backward: targets", targets, T.int64, rows)
    for what, t in (("lse", lse), ("grad_logprob", grad_logprob), ("entropy", entropy), ("grad_entropy", grad_entropy)):
        if t is not None:
            _expect("token_logprobs_backward: " + what, t, T.float32, rows)
    device = _device_of(logits, targets, lse, grad_logprob, grad_logits, entropy, grad_entropy)
    _dispatch_on(device, stream_ptr, "gn_token_logprobs_backward", dt, logits.data_ptr(), rows, cols, ld, temperature,
                 _ptr(targets), _ptr(lse), _ptr(entropy), _ptr(grad_logprob), _ptr(grad_entropy), grad_logits.data_ptr(),
                 ldg)


def distill(logits, ids, teacher, loss, *, lse=None, temperature=1.0, stream_ptr=None):
    """loss[r] = temperature^2 KL(teacher || student) with the teacher's softmax over its entries ids[r] (int64, below 0:
    absent), teacher[r] (float32 logits or log-probabilities), at most 256 of them, and the student's
    over all columns of logits[r]; lse: the student's log-sum-exp."""
    T = _types()
    dt, rows, cols, ld = _matrix("distill", logits)
    k = _width(ids)
    _expect_rows("distill: ids", ids, T.int64, rows, k)
    _expect_rows("distill: teacher", teacher, T.float32, rows, k)
    for what, t in (("loss", loss), ("lse", lse)):
        if t is not None:
            _expect("distill: " + what, t, T.float32, rows)
    device = _device_of(logits, ids, teacher, loss, lse)
    ws, n = _logits_workspace(logits, rows, cols, 0, device, stream_ptr)
    _dispatch_on(device, stream_ptr, "gn_distill_forward", dt, logits.data_ptr(), rows, cols, ld, temperature, ids.data_ptr(),
                 teacher.data_ptr(), k, loss.data_ptr(), _ptr(lse), _ptr(ws), n)


def distill_backward(logits, ids, teacher, lse, grad_loss, grad_logits, *, temperature=1.0, stream_ptr=None):
    """The gradient of the logits (their type; may be the logits themselves) from that of distill's loss."""
    T = _types()
    dt, rows, cols, ld = _matrix("distill_backward", logits)
    dg, grows, gcols, ldg = _matrix("distill_backward: grad_logits", grad_logits)
    if (dg, grows, gcols) != (dt, rows, cols):
        _refuse("distill_backward: grad_logits has the type and shape of logits")
    k = _width(ids)
    _expect_rows("distill_backward: ids", ids, T.int64, rows, k)
    _expect_rows("distill_backward: teacher", teacher, T.float32, rows, k)
    _expect("distill_backward: lse", lse, T.float32, rows)
    _expect("distill_backward: grad_loss", grad_loss, T.float32, rows)
    device = _device_of(logits, ids, teacher, lse, grad_loss, grad_logits)
    _dispatch_on(device, stream_ptr, "gn_distill_backward", dt, logits.data_ptr(), rows, cols, ld, temperature, ids.data_ptr(),
                 teacher.data_ptr(), k, _ptr(lse), grad_loss.data_ptr(), grad_logits.data_ptr(), ldg)


def spmm_csr(M, N, K, nnz, rowptr, col, val, D, C, flags=None, ldd=None, ldc=None, stream_ptr=None):
    _dispatch(stream_ptr, "gn_spmm_csr", M, N, K, nnz, _ptr(rowptr), _ptr(col), _ptr(val), _ptr(D),
              ldd if ldd is not None else N, _ptr(C), ldc if ldc is not None else N, _ptr(flags))


def spmv_csr(M, K, nnz, rowptr, col, val, x, y, flags=None, stream_ptr=None):
    _dispatch(stream_ptr, "gn_spmv_csr", M, K, nnz, _ptr(rowptr), _ptr(col), _ptr(val), _ptr(x), _ptr(y), _ptr(flags))


class SpmvPlan:
    """A grouped-layout SpMV plan over device CSR arrays (gn_spmv_plan_*). The row pointer
    and column tensors must outlive the plan and stay unchanged."""

    def __init__(self, M, K, nnz, rowptr, col, stream_ptr=None):
        self.handle = _VP()
        self._keep = (rowptr, col)
        sp = stream_ptr if stream_ptr is not None else _current_stream()
        call("gn_spmv_plan_create", M, K, nnz, _ptr(rowptr), _ptr(col), ctypes.byref(self.handle), sp or None)
        self._stream = sp or None

    def run(self, val, x, y, flags=None, stream_ptr=None):
        _dispatch(stream_ptr, "gn_spmv_plan_run", self.handle, _ptr(val), _ptr(x), _ptr(y), _ptr(flags))

    def release(self, stream_ptr=None):
        if self.handle:
            load().gn_spmv_plan_release(self.handle, stream_ptr if stream_ptr is not None else self._stream)
            self.handle = _VP()


def fill_uniform(out, seed, stream_id, lo=-1.0, hi=1.0, stream_ptr=None):
    _dispatch(stream_ptr, "gn_fill_uniform_f32", _ptr(out), out.numel(), seed, stream_id, lo, hi)


def fill_normal(out, seed, stream_id, mean=0.0, std=1.0, stream_ptr=None):
    _dispatch(stream_ptr, "gn_fill_normal_f32", _ptr(out), out.numel(), seed, stream_id, mean, std)


def synchronize(stream_ptr=None):
    call("gn_synchronize", stream_ptr)


def _dispatch(stream_ptr, name, *args):
    """Explicit stream -> call on it; otherwise order with torch's current stream."""
    if stream_ptr is not None:
        return call(name, *args, stream_ptr)
    return _run_ordered(name, *args)
