"""Python mirror of the php-gpu-tensors matmul API over libgemm_sm100.so.

The PHP extension cannot be built here (no PHP toolchain), so this module
stands in for its user-facing surface on the matmul path, with the reference's
names, argument meaning and exceptions:

    CudaArray::matmul                stubs/cuda.stub.php:472
    CudaArray::transpose / fromFlatArray / fromBuffer / ones / full / toArray
    cuda_get_backend_info            src/cuda.c:131-153
    cuda_set_matmul_precision        src/cuda.c:155-209
    cuda_tune_matmul                 src/cuda.c:211-290
    PhpTensors\\InvalidArgumentException / RuntimeException

and, with no counterpart there, the feed-forward layers of
include/pt_feed_forward.h: CudaArray.layer_norm, linear and grouped_linear with
layer_norm_backward, linear_backward and grouped_linear_backward.

Every product computed here runs on the GPU through the C ABI of
include/gemm_sm100.h and include/pt_tensor.h (the C++ host layer
pt_tensor_matmul_into dispatches to the launchers).  PyTorch is used only for
device memory, host<->device copies and the current CUDA stream.  There is no
CPU fallback: if the library is missing, or no CUDA device is present, the
calls raise.
"""
import ctypes
import math
import os
import struct

import numpy as np

PKG_DIR = os.path.dirname(os.path.abspath(__file__))
LIB_PATH = os.path.join(PKG_DIR, "libgemm_sm100.so")

MAX_DIMS = 10
DTYPE_CODES = {"float32": 0, "float64": 1, "float16": 11, "bfloat16": 12}
ELEMENT_BYTES = {"float32": 4, "float64": 8, "float16": 2, "bfloat16": 2}
PT_OK, PT_INVALID_ARGUMENT, PT_RUNTIME, PT_WORKSPACE = 0, 1, 2, 3
PT_MATMUL_ALLOW_FLOAT64 = 1
EPILOGUES = {"none": 0, "tanh": 1, "relu": 2, "sigmoid": 3}
# activations of the linear layers
ACTIVATIONS = dict(EPILOGUES, gelu=4, gelu_tanh=5, silu=6)


class InvalidArgumentException(ValueError):
    """PhpTensors\\InvalidArgumentException."""


class RuntimeException(RuntimeError):
    """PhpTensors\\RuntimeException."""


class CudaBackendInfo(ctypes.Structure):
    """cuda_backend_info (src/backends/cuda/backend_info.h:7-14)."""
    _fields_ = [
        ("cublas", ctypes.c_int), ("cublas_lt", ctypes.c_int), ("cudnn", ctypes.c_int),
        ("blas_calls", ctypes.c_ulonglong), ("lt_calls", ctypes.c_ulonglong),
        ("builtin_matmul_calls", ctypes.c_ulonglong),
        ("cub_calls", ctypes.c_ulonglong), ("axis_calls", ctypes.c_ulonglong),
        ("generic_reduce_calls", ctypes.c_ulonglong),
        ("last_matmul", ctypes.c_char_p), ("precision", ctypes.c_char_p),
        ("last_blas_status", ctypes.c_int),
    ]


class TuningCandidate(ctypes.Structure):
    _fields_ = [("algorithm_id", ctypes.c_int), ("workspace_bytes", ctypes.c_size_t),
                ("median_ms", ctypes.c_double)]


class TuningResult(ctypes.Structure):
    _fields_ = [("candidate_count", ctypes.c_int), ("selected_candidate", ctypes.c_int),
                ("candidates", TuningCandidate * 8)]


class PtTensor(ctypes.Structure):
    """pt_tensor (include/pt_tensor.h)."""
    _fields_ = [("data", ctypes.c_void_p), ("dtype", ctypes.c_int), ("ndims", ctypes.c_int),
                ("shape", ctypes.c_int * MAX_DIMS), ("strides", ctypes.c_size_t * MAX_DIMS)]


_PT_TENSOR = struct.Struct("@Pii%di%dN" % (MAX_DIMS, MAX_DIMS))    # pt_tensor's layout
_PAD = [(0,) * (MAX_DIMS - n) for n in range(MAX_DIMS + 1)]

_LIB = None

_SIGNATURES = {
    "cuda_blas_shutdown": (None, []),
    "cuda_blas_set_precision": (ctypes.c_int, [ctypes.c_int]),
    "cuda_blas_precision_name": (ctypes.c_char_p, []),
    "cuda_blas_info": (None, [ctypes.POINTER(CudaBackendInfo)]),
    "cuda_blas_tune_matmul": (ctypes.c_int, [ctypes.c_void_p] * 3 + [ctypes.c_int] * 3 +
                              [ctypes.c_size_t] * 4 + [ctypes.c_void_p,
                                                       ctypes.POINTER(TuningResult)]),
    "cuda_matmul_launcher": (ctypes.c_int, [ctypes.c_void_p] * 3 + [ctypes.c_int] * 3 +
                             [ctypes.c_size_t] * 6 + [ctypes.c_void_p]),
    "cuda_batched_matmul_nd_launcher": (
        ctypes.c_int, [ctypes.c_void_p] * 3 +
        [ctypes.POINTER(ctypes.c_int), ctypes.POINTER(ctypes.c_size_t), ctypes.c_int] * 3 +
        [ctypes.c_void_p]),
    "cuda_low_precision_matmul_nd_launcher": (
        ctypes.c_int, [ctypes.c_void_p] * 3 + [ctypes.c_int] +
        [ctypes.POINTER(ctypes.c_int), ctypes.POINTER(ctypes.c_size_t), ctypes.c_int] * 3 +
        [ctypes.c_void_p]),
    "cuda_f64_matmul_nd_launcher": (
        ctypes.c_int, [ctypes.c_void_p] * 3 +
        [ctypes.POINTER(ctypes.c_int), ctypes.POINTER(ctypes.c_size_t), ctypes.c_int] * 3 +
        [ctypes.c_void_p]),
    "cuda_matmul_epilogue_nd_launcher": (
        ctypes.c_int, [ctypes.c_void_p] * 3 + [ctypes.c_int] +
        [ctypes.POINTER(ctypes.c_int), ctypes.POINTER(ctypes.c_size_t), ctypes.c_int] * 3 +
        [ctypes.c_void_p, ctypes.c_int, ctypes.c_void_p]),
    "cuda_mixed_matmul_nd_launcher": (
        ctypes.c_int, [ctypes.c_void_p, ctypes.c_int, ctypes.c_void_p, ctypes.c_int,
                       ctypes.c_void_p] +
        [ctypes.POINTER(ctypes.c_int), ctypes.POINTER(ctypes.c_size_t), ctypes.c_int] * 3 +
        [ctypes.c_void_p]),
    "gemm_sm100_last_kernel": (ctypes.c_char_p, []),
    "gemm_sm100_selftest_wait_timeout": (ctypes.c_int, [ctypes.c_void_p]),
    "gemm_sm100_set_path": (ctypes.c_int, [ctypes.c_int]),
    "gemm_sm100_last_launch": (None, [ctypes.POINTER(ctypes.c_int)] * 3),
    "gemm_sm100_device_status": (ctypes.c_int, [ctypes.c_int, ctypes.c_int]),
    "gemm_sm100_algorithm_name": (ctypes.c_char_p, [ctypes.c_int]),
    "gemm_sm100_version": (ctypes.c_int, []),
    "gemm_mgpu_unique_id": (ctypes.c_int, [ctypes.c_void_p]),
    "gemm_mgpu_comm_init": (ctypes.c_int, [ctypes.c_void_p, ctypes.c_int, ctypes.c_int,
                                           ctypes.POINTER(ctypes.c_void_p)]),
    "gemm_mgpu_comm_destroy": (None, [ctypes.c_void_p]),
    "gemm_mgpu_nsplit_workspace_bytes": (ctypes.c_size_t, [ctypes.c_int, ctypes.c_int,
                                                           ctypes.c_int, ctypes.c_int]),
    "gemm_mgpu_nsplit_matmul": (ctypes.c_int, [ctypes.c_void_p, ctypes.c_int, ctypes.c_void_p,
                                               ctypes.c_size_t, ctypes.c_size_t, ctypes.c_void_p,
                                               ctypes.c_size_t, ctypes.c_size_t, ctypes.c_void_p,
                                               ctypes.c_int, ctypes.c_int, ctypes.c_int,
                                               ctypes.c_void_p, ctypes.c_size_t, ctypes.c_void_p]),
    "gemm_mgpu_nsplit_matmul_noalloc": (ctypes.c_int, [ctypes.c_void_p, ctypes.c_int,
                                                       ctypes.c_void_p, ctypes.c_size_t,
                                                       ctypes.c_size_t, ctypes.c_void_p,
                                                       ctypes.c_size_t, ctypes.c_size_t,
                                                       ctypes.c_void_p, ctypes.c_int,
                                                       ctypes.c_int, ctypes.c_int,
                                                       ctypes.c_void_p]),
    "gemm_mgpu_window_create": (ctypes.c_int, [ctypes.c_void_p, ctypes.c_size_t,
                                               ctypes.POINTER(ctypes.c_void_p),
                                               ctypes.POINTER(ctypes.c_void_p)]),
    "gemm_mgpu_window_destroy": (None, [ctypes.c_void_p]),
    "gemm_mgpu_window_set_exchange": (ctypes.c_int, [ctypes.c_void_p, ctypes.c_int]),
    "gemm_mgpu_nsplit_matmul_fused": (ctypes.c_int, [ctypes.c_void_p, ctypes.c_int,
                                                     ctypes.c_void_p, ctypes.c_size_t,
                                                     ctypes.c_size_t, ctypes.c_void_p,
                                                     ctypes.c_size_t, ctypes.c_size_t,
                                                     ctypes.c_int, ctypes.c_int, ctypes.c_int,
                                                     ctypes.c_void_p]),
    "pt_host_matmul": (ctypes.c_int, [ctypes.c_void_p] * 3 + [ctypes.c_int] * 8),
    "pt_host_matmul_sharded": (ctypes.c_int, [ctypes.c_void_p] * 3 + [ctypes.c_int] * 6 +
                               [ctypes.POINTER(ctypes.c_int)] + [ctypes.c_int] * 3),
    "pt_host_release": (None, []),
    "pt_last_error": (ctypes.c_char_p, []),
    "pt_matmul_result_shape": (ctypes.c_int, [ctypes.POINTER(PtTensor)] * 2 +
                               [ctypes.POINTER(ctypes.c_int), ctypes.POINTER(ctypes.c_int)]),
    "pt_tensor_matmul_into": (ctypes.c_int, [ctypes.POINTER(PtTensor)] * 3 +
                              [ctypes.c_int, ctypes.c_void_p]),
    "pt_tensor_matmul": (ctypes.c_int, [ctypes.POINTER(PtTensor)] * 3 +
                         [ctypes.c_int, ctypes.c_void_p]),
    "pt_tensor_release": (None, [ctypes.POINTER(PtTensor), ctypes.c_void_p]),
    "pt_tensor_matmul_backward": (ctypes.c_int, [ctypes.POINTER(PtTensor)] * 5 +
                                  [ctypes.c_void_p]),
    "pt_layer_norm": (ctypes.c_int, [ctypes.c_void_p] * 3 + [ctypes.c_float] +
                      [ctypes.c_void_p] * 4),
    "pt_layer_norm_backward": (ctypes.c_int, [ctypes.c_void_p] * 11),
    "pt_linear": (ctypes.c_int, [ctypes.c_void_p] * 4 + [ctypes.c_int] + [ctypes.c_void_p] * 6),
    "pt_linear_backward": (ctypes.c_int, [ctypes.c_void_p] * 5 + [ctypes.c_int] +
                           [ctypes.c_void_p] * 6),
    "pt_layer_norm_backward_workspace": (ctypes.c_size_t, [ctypes.c_longlong, ctypes.c_int]),
}


def exported_symbols():
    """Names the C ABI headers declare (checked against the library by tests)."""
    return sorted(_SIGNATURES)


def library():
    """Loads libgemm_sm100.so (built in-tree); raises if it is missing."""
    global _LIB
    if _LIB is None:
        if not os.path.exists(LIB_PATH):
            raise RuntimeException(
                "libgemm_sm100.so is not built (%s); run php-gpu-tensors_b200/build.py" % LIB_PATH)
        lib = ctypes.CDLL(LIB_PATH)
        for name, (restype, argtypes) in _SIGNATURES.items():
            fn = getattr(lib, name)
            fn.restype = restype
            fn.argtypes = argtypes
        _LIB = lib
    return _LIB


_TORCH = None
_TORCH_DTYPES = {}     # name -> torch dtype, filled with _TORCH
_DTYPE_NAMES = {}


def _torch():
    global _TORCH
    if _TORCH is None:
        import torch
        if not torch.cuda.is_available():
            raise RuntimeException("CUDA device unavailable: CudaArray needs a B200 (sm_100a)")
        for name in DTYPE_CODES:
            _TORCH_DTYPES[name] = getattr(torch, name)
            _DTYPE_NAMES[getattr(torch, name)] = name
        _TORCH = torch
    return _TORCH


def _torch_dtype(dtype):
    _torch()
    return _TORCH_DTYPES[dtype]


def _check_dtype(dtype):
    if dtype not in DTYPE_CODES:
        raise InvalidArgumentException("Unsupported dtype '%s' for the matmul path" % dtype)


def _contiguous_strides(shape):
    strides, s = [], 1
    for d in reversed(shape):
        strides.insert(0, s)
        s *= d
    return strides


def current_stream():
    """Raw cudaStream_t of torch's current stream on the current device."""
    return ctypes.c_void_p(_torch().cuda.current_stream().cuda_stream)


def _raise_for(status):
    if status == PT_OK:
        return
    msg = library().pt_last_error().decode()
    if status == PT_INVALID_ARGUMENT:
        raise InvalidArgumentException(msg)
    raise RuntimeException(msg)


class CudaArray:
    """A device tensor view: flat storage + element offset, shape, strides.

    Mirrors the reference's tensor_t view model (src/tensor.h:49-79): strides
    are in elements, transpose() swaps the last two axes without copying.
    """

    def __init__(self, storage, shape, strides=None, offset=0, dtype="float32"):
        _check_dtype(dtype)
        self._flat = storage               # 1-D torch tensor of the dtype
        self._tensor = self._memory = None
        self._shape = [int(d) for d in shape]
        self._strides = [int(s) for s in (strides if strides is not None
                                          else _contiguous_strides(self._shape))]
        self._offset = int(offset)
        self._dtype = dtype

    def _same_memory(self):
        """Whether the wrapped tensor still has the memory that was wrapped."""
        return (self._memory is None
                or self._tensor.untyped_storage()._cdata == self._memory._cdata)

    def _wrapped(self):
        """A torch tensor of this array's memory, shape and strides: the wrapped
        one while it still has them, as its owner may give it others
        (`tensor.data = ...`, transpose_)."""
        t = self._tensor
        if self._memory is not None and not (
                self._same_memory() and t.storage_offset() == self._offset
                and list(t.shape) == self._shape and list(t.stride()) == self._strides):
            t = _torch().empty(0, dtype=_TORCH_DTYPES[self._dtype], device=self._memory.device)
            t.set_(self._memory, self._offset, self._shape, self._strides)
            self._tensor, self._memory = t, None
        return t

    @property
    def _storage(self):
        """The whole storage as a 1-D torch tensor (of a wrapped tensor made
        when it is first asked for)."""
        if self._flat is None:
            t = self._wrapped()
            n = t.untyped_storage().nbytes() // t.element_size()
            self._flat = _torch().as_strided(t, (n,), (1,), 0)
        return self._flat

    def _address(self):
        """Device address of the first element."""
        if self._memory is not None:
            return self._memory.data_ptr() + self._offset * ELEMENT_BYTES[self._dtype]
        if self._tensor is not None:
            return self._tensor.data_ptr()
        return self._flat.data_ptr() + self._offset * ELEMENT_BYTES[self._dtype]

    # ---------------------------------------------------------- constructors
    @classmethod
    def fromFlatArray(cls, values, shape, dtype="float32"):
        """Values are converted like the reference: double -> float -> dtype (RNE)."""
        torch = _torch()
        host = torch.tensor(np.asarray(values, dtype=np.float64).astype(
            np.float64 if dtype == "float64" else np.float32), dtype=torch.float64
            if dtype == "float64" else torch.float32)
        storage = host.to(_torch_dtype(dtype)).cuda().reshape(-1)
        return cls(storage, shape, dtype=dtype)

    @classmethod
    def fromBuffer(cls, buffer, shape, dtype="float32"):
        """Raw little-endian element bytes (PHP pack('g*'/'e*'...) / toBuffer())."""
        torch = _torch()
        raw = torch.frombuffer(bytearray(buffer), dtype=torch.uint8)
        storage = raw.view(_torch_dtype(dtype)).cuda()
        return cls(storage, shape, dtype=dtype)

    @classmethod
    def from_torch(cls, tensor, dtype=None):
        """Wraps a CUDA torch tensor view without copying (storage offset kept).
        The array keeps the memory, the shape and the strides of this moment,
        whatever the tensor object is given later."""
        if _TORCH is None:
            _torch()
        self = cls.__new__(cls)
        if dtype is None:
            self._dtype = _DTYPE_NAMES[tensor.dtype]
        else:
            _check_dtype(dtype)
            self._dtype = dtype
        self._tensor, self._flat, self._memory = tensor, None, tensor.untyped_storage()
        self._shape, self._strides = list(tensor.shape), list(tensor.stride())
        self._offset = tensor.storage_offset()
        return self

    @classmethod
    def full(cls, shape, value, dtype="float32"):
        n = int(np.prod(shape)) if len(shape) else 1
        storage = _torch().full((n,), float(value), dtype=_torch_dtype(dtype), device="cuda")
        return cls(storage, shape, dtype=dtype)

    @classmethod
    def ones(cls, shape, dtype="float32"):
        return cls.full(shape, 1.0, dtype)

    @classmethod
    def zeros(cls, shape, dtype="float32"):
        return cls.full(shape, 0.0, dtype)

    # ---------------------------------------------------------- views
    def transpose(self):
        if len(self._shape) < 2:
            raise InvalidArgumentException("transpose requires rank >= 2")
        shape, strides = list(self._shape), list(self._strides)
        shape[-2], shape[-1] = shape[-1], shape[-2]
        strides[-2], strides[-1] = strides[-1], strides[-2]
        return CudaArray(self._storage, shape, strides, self._offset, self._dtype)

    def view(self, shape, strides, offset):
        """An arbitrary strided view of the same storage (slices, broadcasts)."""
        return CudaArray(self._storage, shape, strides, offset, self._dtype)

    # ---------------------------------------------------------- metadata
    def dtype(self):
        return self._dtype

    def getShape(self):
        return list(self._shape)

    def getStrides(self):
        return list(self._strides)

    def _pt(self):
        t = PtTensor()
        t.data = self._address()
        t.dtype = DTYPE_CODES[self._dtype]
        t.ndims = len(self._shape)
        for i, (d, s) in enumerate(zip(self._shape, self._strides)):
            t.shape[i] = d
            t.strides[i] = s
        return t

    def _packed(self):
        """The pt_tensor as bytes, which a pointer argument takes as they are."""
        n = len(self._shape)
        if n > MAX_DIMS:
            raise InvalidArgumentException("tensors have at most %d axes" % MAX_DIMS)
        pad = _PAD[n]
        try:
            return _PT_TENSOR.pack(self._address(), DTYPE_CODES[self._dtype], n, *self._shape,
                                   *pad, *self._strides, *pad)
        except struct.error:
            raise InvalidArgumentException("extents must be 32-bit and strides not negative")

    # ---------------------------------------------------------- matmul
    def matmul(self, other, allow_float64=False):
        """C = self . other on the GPU (CudaArray::matmul)."""
        if not isinstance(other, CudaArray):
            raise InvalidArgumentException("Matrix multiplication operand must be a CudaArray")
        lib = library()
        a, b = self._pt(), other._pt()
        shape = (ctypes.c_int * MAX_DIMS)()
        nd = ctypes.c_int(0)
        if self._dtype != other._dtype or self._dtype not in DTYPE_CODES:
            raise InvalidArgumentException(
                "matmul requires matching float32, float16 or bfloat16 operands")
        _raise_for(lib.pt_matmul_result_shape(ctypes.byref(a), ctypes.byref(b), shape,
                                              ctypes.byref(nd)))
        out_shape = [shape[i] for i in range(nd.value)]
        n = int(np.prod(out_shape)) if out_shape else 1
        storage = _torch().empty(max(n, 1), dtype=_torch_dtype(self._dtype), device="cuda")
        result = CudaArray(storage, out_shape, dtype=self._dtype)
        r = result._pt()
        flags = PT_MATMUL_ALLOW_FLOAT64 if allow_float64 else 0
        _raise_for(lib.pt_tensor_matmul_into(ctypes.byref(a), ctypes.byref(b), ctypes.byref(r),
                                             flags, current_stream()))
        return result

    def matmul_epilogue(self, other, bias=None, activation="none"):
        """Fused native-matmul step: act(round(self . other) + bias)."""
        lib = library()
        if other._dtype != self._dtype:
            raise InvalidArgumentException(
                "matmul requires matching float32, float16 or bfloat16 operands")
        a, b = self._pt(), other._pt()
        shape = (ctypes.c_int * MAX_DIMS)()
        nd = ctypes.c_int(0)
        _raise_for(lib.pt_matmul_result_shape(ctypes.byref(a), ctypes.byref(b), shape,
                                              ctypes.byref(nd)))
        out_shape = [shape[i] for i in range(nd.value)]
        n = int(np.prod(out_shape)) if out_shape else 1
        storage = _torch().empty(max(n, 1), dtype=_torch_dtype(self._dtype), device="cuda")
        result = CudaArray(storage, out_shape, dtype=self._dtype)
        bias_ptr = None
        if bias is not None:
            if bias._dtype != self._dtype or bias.getShape() != [out_shape[-1]]:
                raise InvalidArgumentException("bias must be a [N] vector of the operand dtype")
            bias_ptr = ctypes.c_void_p(bias._storage.data_ptr() +
                                       bias._offset * ELEMENT_BYTES[self._dtype])
        arrays = [_shape_args(x) for x in (self, other, result)]
        ok = lib.cuda_matmul_epilogue_nd_launcher(
            a.data, b.data, result._pt().data, DTYPE_CODES[self._dtype],
            *arrays[0], *arrays[1], *arrays[2], bias_ptr, EPILOGUES[activation],
            current_stream())
        if not ok:
            info = cuda_get_backend_info()
            raise RuntimeException("Matmul backend submission failed (cuBLAS status %d)"
                                   % info["lastBlasStatus"])
        return result

    # ---------------------------------------------------------- feed-forward
    def layer_norm(self, gamma=None, beta=None, eps=1e-5, save_stats=False):
        """Layer norm over the last axis (pt_layer_norm); gamma and beta are
        [cols] arrays of this dtype or float32.  With save_stats the result is
        (y, mean, rstd), the float32 statistics layer_norm_backward takes."""
        _check_feed_forward("layer_norm", (), gamma, beta)
        y = _result_like(self)
        mean, rstd = _result_pair(self._shape[:-1]) if save_stats else (None, None)
        _raise_for(library().pt_layer_norm(
            _ref(self), _ref(gamma), _ref(beta), eps, _ref(y), _ptr(mean), _ptr(rstd),
            _raw_stream()))
        return (y, mean, rstd) if save_stats else y

    def linear(self, weight, bias=None, activation="none", residual=None, save_pre=False):
        """activation(self . weight + bias) + residual in one pass (pt_linear):
        self [..., K], weight [K, N], bias [N], residual [..., N]; activation
        one of ACTIVATIONS.  With save_pre the result is (y, pre), pre the
        pre-activation that linear_backward takes."""
        return _linear(self, weight, (), bias, activation, residual, save_pre)

    def grouped_linear(self, weight, ends, bias=None, activation="none", residual=None,
                       save_pre=False):
        """linear with an own weight [E, K, N] and bias [E, N] for each of E
        groups of consecutive rows of self [rows, K]; ends, an int32 torch
        tensor on the device, holds the row behind each group's last one."""
        return _linear(self, weight, (ends,), bias, activation, residual, save_pre)

    # ---------------------------------------------------------- export
    def to_torch(self):
        """A new torch view of this array (no copy)."""
        if self._tensor is not None:
            return self._wrapped()[...]
        return self._storage.as_strided(self._shape, self._strides, self._offset)

    def toArray(self):
        t = self.to_torch().float() if self._dtype in ("float16", "bfloat16") else self.to_torch()
        return t.cpu().tolist()

    def toBuffer(self):
        return self.to_torch().contiguous().cpu().view(-1).view(
            _torch().uint8).numpy().tobytes()

    def to_numpy(self):
        t = self.to_torch().contiguous().cpu()
        if self._dtype in ("float16", "bfloat16"):
            return t.view(_torch().int16).numpy().view(np.uint16)
        return t.numpy()


# ---------------------------------------------------------------- feed-forward
def _check_feed_forward(what, required, *optional):
    for a in required:
        if not isinstance(a, CudaArray):
            raise InvalidArgumentException("%s operands must be CudaArrays" % what)
    for a in optional:
        if a is not None and not isinstance(a, CudaArray):
            raise InvalidArgumentException("%s operands must be CudaArrays or None" % what)


def _result(shape, dtype, like=None):
    """An uninitialised contiguous array; `like`, an array of the same type,
    saves torch's own argument handling."""
    self = CudaArray.__new__(CudaArray)
    t = None if like is None else like._tensor
    if t is not None and like._same_memory() and t.dtype == _TORCH_DTYPES[dtype]:
        t = t.new_empty(shape)
    else:
        t = _torch().empty(shape, dtype=_TORCH_DTYPES[dtype], device="cuda")
    self._tensor, self._flat, self._memory, self._dtype, self._offset = t, None, None, dtype, 0
    self._shape, self._strides = list(shape), list(t.stride())
    return self


def _result_like(a):
    """An uninitialised contiguous array of the shape and type of `a`."""
    t = a._tensor
    if t is None or not a._same_memory() or list(t.shape) != a._shape or not t.is_contiguous():
        return _result(a._shape, a._dtype, a)
    self = CudaArray.__new__(CudaArray)
    self._tensor, self._flat, self._memory = _torch().empty_like(t), None, None
    self._dtype, self._offset = a._dtype, 0
    self._shape, self._strides = a._shape, a._strides
    return self


def _result_pair(shape):
    """Two uninitialised contiguous float32 arrays in one allocation."""
    n = math.prod(shape)
    flat = _torch().empty(2 * n, dtype=_TORCH_DTYPES["float32"], device="cuda")
    strides = _contiguous_strides(shape)
    pair = []
    for offset in (0, n):
        a = CudaArray.__new__(CudaArray)
        a._tensor, a._flat, a._memory = None, flat, None
        a._dtype, a._offset, a._shape, a._strides = "float32", offset, list(shape), strides
        pair.append(a)
    return pair


def _ref(a):
    """`a` as a pt_tensor argument; None as a null pointer."""
    return None if a is None else a._packed()


def _ptr(a):
    return None if a is None else a._address()


def _raw_stream():
    torch = _torch()
    return torch._C._cuda_getCurrentRawStream(torch.cuda.current_device())


def _workspace(nbytes):
    torch = _torch()
    return torch.empty(nbytes, dtype=torch.uint8, device="cuda")


def layer_norm_backward(grad, x, gamma, mean, rstd, params=True):
    """Gradients of CudaArray.layer_norm (pt_layer_norm_backward): (dx, dgamma,
    dbeta), the last two float32 sums over all rows (None without `params`).
    mean and rstd are the statistics layer_norm saved."""
    _check_feed_forward("layer_norm_backward", (grad, x, mean, rstd), gamma)
    lead, cols = x._shape[:-1], x._shape[-1] if x._shape else 0
    for s in (mean, rstd):
        if s._dtype != "float32" or s._shape != lead or s._strides != _contiguous_strides(lead):
            raise InvalidArgumentException(
                "layer norm statistics must be contiguous float32 arrays, one value a row")
    dx = _result_like(x)
    dgamma = dbeta = work = None
    lib = library()
    size = ctypes.c_size_t(0)
    if params:
        dgamma, dbeta = _result_pair([cols])
        size.value = lib.pt_layer_norm_backward_workspace(math.prod(lead), cols)
        work = _workspace(size.value)
    _raise_for(lib.pt_layer_norm_backward(
        _ref(grad), _ref(x), _ref(gamma), _ptr(mean), _ptr(rstd), _ref(dx), _ptr(dgamma),
        _ptr(dbeta), None if work is None else work.data_ptr(), ctypes.addressof(size),
        _raw_stream()))
    return dx, dgamma, dbeta


def _activation_code(activation):
    if activation not in ACTIVATIONS:
        raise InvalidArgumentException("Unknown activation %r" % (activation,))
    return ACTIVATIONS[activation]


def _check_ends(ends, weight):
    torch = _torch()
    if (not isinstance(ends, torch.Tensor) or ends.dtype != torch.int32 or not ends.is_cuda
            or ends.dim() != 1 or not ends.is_contiguous()):
        raise InvalidArgumentException(
            "ends must be a contiguous int32 vector on the device, one value a group")
    if weight._shape[:1] != [ends.numel()]:
        raise InvalidArgumentException("ends must have one value for each of the weight's groups")
    return ends.data_ptr()


def _with_workspace(call, args, stream):
    """call(*args, workspace, size, stream), and where it asks for a workspace
    again with one."""
    size = ctypes.c_size_t(0)
    status = call(*args, None, ctypes.addressof(size), stream)
    if status == PT_WORKSPACE:
        work = _workspace(size.value)
        status = call(*args, work.data_ptr(), ctypes.addressof(size), stream)
    if status != PT_OK:
        _raise_for(status)


def _linear(x, weight, ends, bias, activation, residual, save_pre):
    """ends: empty, or the one `ends` of a grouped layer."""
    _check_feed_forward("linear", (weight,), bias, residual)
    ends = _check_ends(*ends, weight) if ends else None
    if not x._shape or not weight._shape:
        raise InvalidArgumentException("linear layers require rows and a weight")
    code = _activation_code(activation)
    shape = x._shape[:-1] + weight._shape[-1:]
    y = _result(shape, x._dtype, x)
    pre = _result(shape, x._dtype, x) if save_pre else None
    _with_workspace(library().pt_linear,
                    (_ref(x), _ref(weight), ends, _ref(bias), code, _ref(residual), _ref(y),
                     _ref(pre)), _raw_stream())
    return (y, pre) if save_pre else y


def _linear_backward(grad, x, weight, ends, pre, activation, bias, inputs, weights,
                     weight_grad_dtype):
    _check_feed_forward("linear_backward", (grad, x, weight), pre)
    code = _activation_code(activation)
    if weight_grad_dtype is not None:
        _check_dtype(weight_grad_dtype)
    ends = _check_ends(*ends, weight) if ends else None
    dx = _result_like(x) if inputs else None
    dw = None
    if weights:
        dw = _result(weight._shape, weight_grad_dtype or x._dtype,
                     None if weight_grad_dtype else x)
    dbias = _result(weight._shape[:-2] + weight._shape[-1:], "float32") if bias else None
    _with_workspace(library().pt_linear_backward,
                    (_ref(grad), _ref(x), _ref(weight), ends, _ref(pre), code, _ref(dx), _ref(dw),
                     _ptr(dbias)), _raw_stream())
    return dx, dw, dbias


def linear_backward(grad, x, weight, pre=None, activation="none", bias=True, inputs=True,
                    weights=True, weight_grad_dtype=None):
    """Gradients of CudaArray.linear (pt_linear_backward): (dx, dw, dbias), each
    None where it is not wanted (inputs, weights, bias).  pre is what
    linear(save_pre=True) kept; dw has weight's type or float32, dbias is
    float32; the residual's gradient is grad itself."""
    return _linear_backward(grad, x, weight, (), pre, activation, bias, inputs, weights,
                            weight_grad_dtype)


def grouped_linear_backward(grad, x, weight, ends, pre=None, activation="none", bias=True,
                            inputs=True, weights=True, weight_grad_dtype=None):
    """Gradients of CudaArray.grouped_linear, as linear_backward."""
    return _linear_backward(grad, x, weight, (ends,), pre, activation, bias,
                            inputs, weights, weight_grad_dtype)


def host_matmul(a, b, c, chunks=8, allow_float64=False, devices=None):
    """Batched product between HOST torch tensors (pinned for overlap):
    a [batches, M, K], b [batches, K, N] or [K, N] (shared), c [batches, M, N]
    are filled through pt_host_matmul, whose copies and products overlap.
    devices=[d0, d1, ...] shards the batch over those GPUs of this process
    (pt_host_matmul_sharded), `chunks` pieces per device."""
    torch = _torch()
    rev = {torch.float32: "float32", torch.float64: "float64", torch.float16: "float16",
           torch.bfloat16: "bfloat16"}
    dt = rev[a.dtype]
    if not (a.is_contiguous() and b.is_contiguous() and c.is_contiguous()):
        raise InvalidArgumentException("host_matmul needs contiguous row-major host tensors")
    batches, M, K = a.shape
    shared = b.dim() == 2
    N = b.shape[-1]
    if (b.shape[-2] != K or list(c.shape) != [batches, M, N]
            or (not shared and b.shape[0] != batches)):
        raise InvalidArgumentException("Matrix multiplication failed - incompatible dimensions")
    flags = PT_MATMUL_ALLOW_FLOAT64 if allow_float64 else 0
    if devices is None:
        _raise_for(library().pt_host_matmul(
            a.data_ptr(), b.data_ptr(), c.data_ptr(), DTYPE_CODES[dt], batches, M, N, K,
            1 if shared else 0, chunks, flags))
    else:
        devs = (ctypes.c_int * len(devices))(*devices)
        _raise_for(library().pt_host_matmul_sharded(
            a.data_ptr(), b.data_ptr(), c.data_ptr(), DTYPE_CODES[dt], batches, M, N, K,
            1 if shared else 0, devs, len(devices), chunks, flags))
    return c


def _shape_args(x):
    nd = len(x._shape)
    shape = (ctypes.c_int * MAX_DIMS)(*x._shape)
    strides = (ctypes.c_size_t * MAX_DIMS)(*x._strides)
    return shape, strides, nd


def cuda_get_backend_info():
    """cuda_get_backend_info() matmul keys (src/cuda.c:131-153) + 'kernel'."""
    lib = library()
    info = CudaBackendInfo()
    lib.cuda_blas_info(ctypes.byref(info))
    return {
        "cublas": info.cublas, "cublasLt": info.cublas_lt,
        "blasCalls": info.blas_calls, "ltCalls": info.lt_calls,
        "builtinMatmulCalls": info.builtin_matmul_calls,
        "lastMatmul": info.last_matmul.decode(), "precision": info.precision.decode(),
        "lastBlasStatus": info.last_blas_status,
        "kernel": lib.gemm_sm100_last_kernel().decode(),
    }


def cuda_set_matmul_precision(precision):
    """src/cuda.c:155-209 (TF32 is supported by this backend)."""
    modes = {"fp32-strict": 0, "tf32": 1}
    if precision not in modes:
        raise InvalidArgumentException("Matmul precision must be 'fp32-strict' or 'tf32'")
    if not library().cuda_blas_set_precision(modes[precision]):
        raise RuntimeException("Failed to set matmul precision")


def cuda_tune_matmul(left, right):
    """src/cuda.c:211-290 over this library's own tile configurations."""
    if left.dtype() != "float32" or right.dtype() != "float32":
        raise InvalidArgumentException("Matmul autotuning currently requires valid float32 tensors")
    ls, rs = left.getShape(), right.getShape()
    if len(ls) != 2 or len(rs) != 2 or ls[1] != rs[0]:
        raise InvalidArgumentException("Matmul autotuning currently requires compatible 2D tensors")
    torch = _torch()
    out = torch.empty(ls[0] * rs[1], dtype=torch.float32, device="cuda")
    torch.cuda.synchronize()
    result = TuningResult()
    a, b = left._pt(), right._pt()
    status = library().cuda_blas_tune_matmul(
        a.data, b.data, out.data_ptr(), ls[0], ls[1], rs[1], left._strides[0], left._strides[1],
        right._strides[0], right._strides[1], current_stream(), ctypes.byref(result))
    if status < 0:
        raise RuntimeException("Matmul autotuning failed (cuBLAS status %d)"
                               % cuda_get_backend_info()["lastBlasStatus"])
    if status == 0:
        raise InvalidArgumentException(
            "Matmul autotuning requires compatible strides and at least 10 million operations")
    cands = []
    for i in range(result.candidate_count):
        c = result.candidates[i]
        cands.append({"algorithmId": c.algorithm_id, "workspaceBytes": c.workspace_bytes,
                      "medianMs": c.median_ms, "selected": i == result.selected_candidate,
                      "name": library().gemm_sm100_algorithm_name(c.algorithm_id).decode()})
    return {"backend": "builtin", "precision": library().cuda_blas_precision_name().decode(),
            "selectedCandidate": result.selected_candidate,
            "candidateCount": result.candidate_count, "candidates": cands,
            "product": CudaArray(out, [ls[0], rs[1]])}


def set_kernel_path(path):
    """0 automatic, 1 single-CTA tensor-core kernel whenever the layout allows,
    2 CUDA cores only, 3 2-CTA tensor-core kernel whenever allowed (16-bit,
    tf32, strict float32, float32 x bf16), 4 few-column split-K kernel
    whenever N <= 32 and K >= 128, 5 the 2-CTA 256 x 512 kernel for 16-bit
    products with a 16-bit result (other products as 3), 6 the same kernel
    running every tile as two 256-column halves.  The linear layers take 1 as
    their few-row kernel, 2 as their CUDA-core kernel, 3 as their pair kernel."""
    return library().gemm_sm100_set_path(
        {"auto": 0, "tensor-core": 1, "simt": 2, "tensor-core-pair": 3, "skinny": 4,
         "tensor-core-wide": 5, "tensor-core-wide-halves": 6}[path])


def last_launch():
    """(grid, block, cluster) of the last tensor-core, few-column or feed-forward
    launch on this thread."""
    g, b, c = ctypes.c_int(), ctypes.c_int(), ctypes.c_int()
    library().gemm_sm100_last_launch(ctypes.byref(g), ctypes.byref(b), ctypes.byref(c))
    return g.value, b.value, c.value


def device_status(device=0, clear=True):
    return library().gemm_sm100_device_status(device, 1 if clear else 0)


# ---------------------------------------------------------------- multi-GPU
class MgpuComm:
    """NCCL communicator of the library for one process per GPU.

    Rank 0 creates the id with gemm_mgpu_unique_id; it reaches the other ranks
    through the already-initialised torch.distributed process group (host
    plumbing only), and every rank joins on its current device.
    """

    def __init__(self, rank, world):
        import torch.distributed as dist
        lib = library()
        idbuf = (ctypes.c_ubyte * 128)()
        if rank == 0 and not lib.gemm_mgpu_unique_id(idbuf):
            raise RuntimeException("NCCL is unavailable for the multi-GPU entry points")
        obj = [bytes(idbuf)]
        if world > 1:
            dist.broadcast_object_list(obj, src=0)
        idbuf = (ctypes.c_ubyte * 128).from_buffer_copy(obj[0])
        handle = ctypes.c_void_p()
        if not lib.gemm_mgpu_comm_init(idbuf, world, rank, ctypes.byref(handle)):
            raise RuntimeException("gemm_mgpu_comm_init failed (status %d)"
                                   % cuda_get_backend_info()["lastBlasStatus"])
        self.handle, self.rank, self.world = handle, rank, world

    def close(self):
        if self.handle:
            library().gemm_mgpu_comm_destroy(self.handle)
            self.handle = None


def nsplit_columns(N, rank, world):
    """Column block [lo, hi) of rank `rank` in an N-split product."""
    if N % world:
        raise InvalidArgumentException("N-split needs N divisible by the number of ranks")
    nb = N // world
    return rank * nb, (rank + 1) * nb


def nsplit_matmul(comm, a, b_local, N, workspace=None):
    """C = A . B with B split along N: `b_local` is this rank's column block;
    every rank receives the whole row-major C (gemm_mgpu_nsplit_matmul)."""
    lib = library()
    torch = _torch()
    M, K = a.getShape()
    if b_local.getShape() != [K, N // comm.world] or a.dtype() != b_local.dtype():
        raise InvalidArgumentException("b_local must be this rank's [K, N / ranks] block")
    dt = a.dtype()
    need = lib.gemm_mgpu_nsplit_workspace_bytes(comm.world, DTYPE_CODES[dt], M, N)
    if need == 0 and M * N > 0:
        raise InvalidArgumentException("N-split needs N divisible by the number of ranks")
    if workspace is None:
        workspace = torch.empty(max(need, 16), dtype=torch.uint8, device="cuda")
    c = CudaArray(torch.empty(max(M * N, 1), dtype=_torch_dtype(dt), device="cuda"), [M, N],
                  dtype=dt)
    es = ELEMENT_BYTES[dt]
    ok = lib.gemm_mgpu_nsplit_matmul(
        comm.handle, DTYPE_CODES[dt], a._storage.data_ptr() + a._offset * es, a._strides[0],
        a._strides[1], b_local._storage.data_ptr() + b_local._offset * es, b_local._strides[0],
        b_local._strides[1], c._storage.data_ptr(), M, N, K, workspace.data_ptr(),
        workspace.numel(), current_stream())
    if not ok:
        raise RuntimeException("N-split matmul failed (status %d)"
                               % cuda_get_backend_info()["lastBlasStatus"])
    return c


class MgpuWindow:
    """An [M, N] float64 result buffer mapped into every rank (the fused
    N-split product writes into all of them)."""

    def __init__(self, comm, M, N):
        lib = library()
        h, local = ctypes.c_void_p(), ctypes.c_void_p()
        if not lib.gemm_mgpu_window_create(comm.handle, M * N * 8, ctypes.byref(h),
                                           ctypes.byref(local)):
            raise RuntimeException("gemm_mgpu_window_create failed (status %d)"
                                   % cuda_get_backend_info()["lastBlasStatus"])
        self.handle, self.local, self.comm, self.M, self.N = h, local.value, comm, M, N

    EXCHANGE = {"auto": 0, "store": 1, "overlap": 2}

    def set_exchange(self, mode):
        """'auto', 'store' (epilogue stores into every window) or 'overlap'
        (persistent kernel, copies under the next tile's math)."""
        if mode not in self.EXCHANGE or not library().gemm_mgpu_window_set_exchange(
                self.handle, self.EXCHANGE[mode]):
            raise InvalidArgumentException("unknown exchange mode %r" % (mode,))

    def result(self):
        """The window as a torch view (float64 [M, N]); valid after a fused call."""
        torch = _torch()
        n = self.M * self.N
        holder = _CudaPointer(self.local, n * 8)
        return torch.as_tensor(holder, device="cuda").view(torch.float64)[:n].view(self.M, self.N)

    def close(self):
        if self.handle:
            library().gemm_mgpu_window_destroy(self.handle)
            self.handle = None


class _CudaPointer:
    """__cuda_array_interface__ over raw device memory (bytes)."""

    def __init__(self, ptr, nbytes):
        self.__cuda_array_interface__ = {"shape": (nbytes,), "typestr": "|u1",
                                         "data": (ptr, False), "version": 3}


def nsplit_matmul_fused(window, a, b_local):
    """Fused N-split float64 product into `window` (every rank's copy)."""
    lib = library()
    M, K = a.getShape()
    es = 8
    ok = lib.gemm_mgpu_nsplit_matmul_fused(
        window.handle, DTYPE_CODES["float64"], a._storage.data_ptr() + a._offset * es,
        a._strides[0], a._strides[1], b_local._storage.data_ptr() + b_local._offset * es,
        b_local._strides[0], b_local._strides[1], M, window.N, K, current_stream())
    if not ok:
        raise RuntimeException("fused N-split matmul failed (status %d)"
                               % cuda_get_backend_info()["lastBlasStatus"])
    return window.result()
