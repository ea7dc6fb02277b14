"""ctypes binding of libaiter_b200.so.

Mirrors the reference's ctypes caller (aiter/jit/core.py:1457-1553): tensors go in as
`aiter_tensor_t*` (NULL for None), ints as C ints (-1 for None), strings as `const char*`
(NULL for None), bools as ints, floats as floats, and the current CUDA stream is appended as
the trailing `void*`.  A non-zero return raises RuntimeError("<name> failed: <message>").
There is no fallback: if the library is missing the import of this module fails.
"""
from __future__ import annotations

import ctypes
import importlib.machinery
import importlib.util
import os
import struct
import threading

import torch

from .dtypes import _torch_to_aiter_dtype as _DTYPE_IDS
from .dtypes import aiter_dtype_id, fp4x2, fp8, fp8_e8m0

# AITER_B200_LIBRARY points at another build of the library (comparing two builds on one machine)
LIB_PATH = os.environ.get("AITER_B200_LIBRARY") or os.path.join(os.path.dirname(os.path.abspath(__file__)), "csrc", "libaiter_b200.so")


class aiter_tensor_t(ctypes.Structure):
    _fields_ = [
        ("ptr", ctypes.c_void_p),
        ("numel_", ctypes.c_size_t),
        ("ndim", ctypes.c_int),
        ("shape", ctypes.c_int64 * 8),
        ("strides", ctypes.c_int64 * 8),
        ("dtype_", ctypes.c_int),
        ("device_id", ctypes.c_int),
    ]


assert ctypes.sizeof(aiter_tensor_t) == 160, "aiter_tensor_t layout drifted from include/aiter_b200.h"


def torch_to_aiter(t: torch.Tensor) -> aiter_tensor_t:
    shape, strides = t.shape, t.stride()
    ndim = len(shape)
    assert ndim <= 8, f"aiter_tensor_t supports at most 8 dims, got {ndim}"
    at = aiter_tensor_t()
    at.ptr = t.data_ptr()
    at.numel_ = t.numel()
    at.ndim = ndim
    at.shape[:ndim] = shape
    at.strides[:ndim] = strides
    at.dtype_ = aiter_dtype_id(t.dtype)
    idx = t.device.index
    at.device_id = -1 if (t.device.type != "cuda" or idx is None) else idx
    return at


def _load():
    if not os.path.exists(LIB_PATH):
        raise ImportError(
            f"{LIB_PATH} is missing: build it with `python aiter_b200/build.py` (needs nvcc). "
            "aiter_b200 has no CPU or PyTorch fallback."
        )
    return ctypes.CDLL(LIB_PATH)


_lib = _load()
if int(os.getenv("AITER_LOG_MORE", "0")) >= 1:
    import logging as _logging

    _logging.getLogger("aiter").info("loaded %s", LIB_PATH)
_lib.aiter_get_last_error.restype = ctypes.c_char_p
_lib.aiter_b200_kernel_list.restype = ctypes.c_char_p
_lib.aiter_b200_heuristic_name.restype = ctypes.c_char_p
_lib.aiter_b200_launch_count.restype = ctypes.c_ulonglong
if hasattr(_lib, "aiter_b200_gemm_a4w4_fused_workspace"):  # (a build from before the fused GEMMs has none)
    _lib.aiter_b200_gemm_a4w4_fused_workspace.restype = ctypes.c_longlong
assert _lib.aiter_ctypes_abi_version() == 2

T, I, S, F = "tensor", "int", "str", "float"
# name -> argument kinds (the stream is appended automatically)
SIGNATURES = {
    "gemm_a4w4_asm": (T, T, T, T, T, S, T, F, F, I, I),
    "gemm_a4w4_blockscale": (T, T, T, T, T, I, S),
    "gemm_a4w4_blockscale_tune": (T, T, T, T, T, I, I),
    "mxfp8_mxfp8_gemm_asm": (T, T, T, T, T, S, I),
    "mxfp8_mxfp4_gemm_asm": (T, T, T, T, T, S, I),
    "mxfp4_gemm_asm": (T, T, T, T, T, T, S, I),
    "nvfp4_gemm_asm": (T, T, T, T, F, F, T, T, S, I),
    "gemm_a16w16_asm": (T, T, T, T, T, I, S, I),
    "opus_gemm_a16w16_tune": (T, T, T, T, I, I),
    "opus_gemm": (T, T, T, T, T, T, T),
    "batched_gemm_bf16": (T, T, T, T, I),
    "batched_gemm_bf16_tune": (T, T, T, I, I),
    "dynamic_per_group_scaled_quant": (T, T, T, I, I, T, I),
    "gemm_a8w8_blockscale": (T, T, T, T, T, I, S),
    "gemm_a8w8_blockscale_tune": (T, T, T, T, T, I, I),
    "gemm_a8w8_blockscale_bpreshuffle": (T, T, T, T, T, I, S),
    "gemm_a8w8_blockscale_bpreshuffle_tune": (T, T, T, T, T, I, I),
    "gemm_a8w8_blockscale_cktile": (T, T, T, T, T, I, I, S),
    "gemm_a8w8_blockscale_cktile_tune": (T, T, T, T, T, I, I, I),
    "gemm_a8w8_blockscale_bpreshuffle_cktile": (T, T, T, T, T, I, S),
    "gemm_a8w8_blockscale_bpreshuffle_cktile_tune": (T, T, T, T, T, I, I, I),
    "flatmm_a8w8_blockscale_asm": (T, T, T, T, T),
    "gemm_a8w8_blockscale_bpreshuffle_asm": (T, T, T, T, T, T, I, S, I, T),
    "aiter_b200_gemm_a8w8_mxfp8_noalloc": (T, T, T, T, T, I, I),
    "aiter_b200_gemm_a16w16_fused": (T, T, T, T, T, I, I, S),
    "aiter_b200_gemm_a8w8_mxfp8_fused": (T, T, T, T, T, T, T, I, I, S),
    "aiter_b200_gemm_a4w4_fused": (T, T, T, T, T, T, T, T, I, I, S),
    "aiter_b200_gated_residual_norm": (T, T, T, T, T, T, T, T, T, T, F, F, F, I, I, I),
    "aiter_b200_act_and_mul": (T, T, T, I, I),
}
EXPORTS = sorted(
    list(SIGNATURES)
    + ["getPaddedM", "aiter_ctypes_abi_version", "aiter_get_last_error", "aiter_clear_last_error",
       "opus_gemm_workspace_init", "aiter_b200_device_status", "aiter_b200_kernel_list",
       "aiter_b200_heuristic_name", "aiter_b200_launch_count", "aiter_b200_noalloc_status",
       "aiter_b200_debug_wait_control", "aiter_b200_gemm_a4w4_fused_workspace"]
)


# aiter_tensor_t of an n-dimensional tensor as one packed byte string: filling the ctypes structure field by field took
# 3.7 us a tensor, half of a small call's host time; this takes 1.5
_PACKERS = [struct.Struct(f"@NNi4x{n}q{64 - 8 * n}x{n}q{64 - 8 * n}xii").pack for n in range(9)]
assert all(len(_PACKERS[n](*([0] * (2 * n + 5)))) == 160 for n in range(9)), "aiter_tensor_t layout drifted from include/aiter_b200.h"


def _pack_tensor(t):
    if t is None:
        return None
    shape = t.shape
    ndim = len(shape)
    dtype = _DTYPE_IDS.get(t.dtype)
    if dtype is None:
        dtype = aiter_dtype_id(t.dtype)  # raises, naming the type
    if ndim == 2:
        rows, cols = shape
        row_stride, col_stride = t.stride()
        return _pack_2d(t.data_ptr(), rows * cols, 2, rows, cols, row_stride, col_stride, dtype, t.get_device())
    assert ndim <= 8, f"aiter_tensor_t supports at most 8 dims, got {ndim}"
    return _PACKERS[ndim](t.data_ptr(), t.numel(), ndim, *shape, *t.stride(), dtype, t.get_device())


_pack_2d = _PACKERS[2]


def _int(value):
    return -1 if value is None else int(value)


def _str(value):
    return None if value is None else str(value).encode()


_CONVERT = {T: (_pack_tensor, ctypes.c_char_p), I: (_int, ctypes.c_int), S: (_str, ctypes.c_char_p), F: (float, ctypes.c_float)}
_FUNCS = {}
_raw_stream = getattr(torch._C, "_cuda_getCurrentRawStream", None)


def _bind(name: str):
    """The library function with its argument types, and how each Python argument is converted (tensors travel as the bytes of
    their descriptor, which the call reads before it returns)."""
    kinds = SIGNATURES[name]
    fn = getattr(_lib, name)
    fn.argtypes = [_CONVERT[k][1] for k in kinds] + [ctypes.c_void_p]
    _FUNCS[name] = bound = (fn, [_CONVERT[k][0] for k in kinds])
    return bound


# AITER_LOG_MORE=2 logs every call that crosses the C ABI with its arguments (tensors as shape / dtype / device), as
# the reference's ctypes caller does (aiter/jit/core.py:1466-1469); 1 logs the library path at load
AITER_LOG_MORE = int(os.getenv("AITER_LOG_MORE", "0"))


def _describe(a):
    if isinstance(a, torch.Tensor):
        return f"Tensor{tuple(a.shape)} {str(a.dtype).replace('torch.', '')} {a.device} stride{tuple(a.stride())}"
    return repr(a)


def call(name: str, *args):
    """Call an entry point on the current CUDA stream of the first tensor's device."""
    fn, convert = _FUNCS.get(name) or _bind(name)
    assert len(args) == len(convert), f"{name} takes {len(convert)} arguments, got {len(args)}"
    if AITER_LOG_MORE == 2:
        import logging

        logging.getLogger("aiter").info("calling %s(%s)", name, ", ".join(_describe(a) for a in args))
    stream = None
    for a in args:
        if isinstance(a, torch.Tensor) and a.is_cuda:
            stream = current_stream(a.get_device())
            break
    if fn(*[c(a) for c, a in zip(convert, args)], stream) != 0:
        _raise(name)


def _raise(name: str):
    msg = _lib.aiter_get_last_error()
    raise RuntimeError(f"{name} failed: {msg.decode() if msg else 'unknown error'}")


def current_stream(device: int):
    """The current stream of a GPU as the library takes it (device -1: none, the library refuses host tensors)."""
    if device < 0:
        return None
    return _raw_stream(device) if _raw_stream is not None else torch.cuda.current_stream(device).cuda_stream


HOST_PATH = os.path.join(os.path.dirname(os.path.abspath(__file__)), "csrc", "_aiter_b200_host.so")
_HOST_ENTRIES = ("gated_residual_norm", "act_and_mul", "gemm_a16w16_fused", "gemm_a8w8_mxfp8_fused", "gemm_a4w4_fused", "gemm_a4w4_fused_workspace")


class _Host:
    """The extension that allocates, fills descriptors and calls for the operators whose host time shows (see csrc/host.cpp).  It is loaded
    with the first of them: the other operators need neither the extension nor a library that has these."""

    _lock = threading.Lock()

    def __getattr__(self, name):  # (only until the functions are there)
        if name not in ("norm", "act", "gemm"):
            raise AttributeError(name)
        with self._lock:
            if name not in self.__dict__:
                self._load()
        return self.__dict__[name]

    def _load(self):
        if not os.path.exists(HOST_PATH):
            raise ImportError(f"{HOST_PATH} is missing: build it with `python aiter_b200/build.py`")
        missing = [n for n in _HOST_ENTRIES if not hasattr(_lib, f"aiter_b200_{n}")]
        if missing:
            raise ImportError(f"{LIB_PATH} has no aiter_b200_{missing[0]}: it was built before this operator")
        loader = importlib.machinery.ExtensionFileLoader("_aiter_b200_host", HOST_PATH)
        module = importlib.util.module_from_spec(importlib.util.spec_from_loader("_aiter_b200_host", loader))
        loader.exec_module(module)
        module.bind(*(ctypes.cast(getattr(_lib, f"aiter_b200_{n}"), ctypes.c_void_p).value for n in _HOST_ENTRIES), dict(_DTYPE_IDS), aiter_dtype_id, fp4x2, fp8, fp8_e8m0)
        self.__dict__.update(norm=module.norm, act=module.act, gemm=module.gemm)


host = _Host()


def call_host(name: str, function, *args):
    """A function of the extension: the entry point `name` on the stream that ends `args`; what it returns."""
    if AITER_LOG_MORE == 2:
        import logging

        logging.getLogger("aiter").info("calling %s(%s)", name, ", ".join(_describe(a) for a in args))
    result = function(*args)
    if result is None:
        _raise(name)
    return result


def get_padded_m(M: int, N: int, K: int, gl: int) -> int:
    return int(_lib.getPaddedM(int(M), int(N), int(K), int(gl)))


def device_status(device: int = 0):
    """(code, block, split, iteration) of the last expired in-kernel wait on `device`; zeros = healthy.
    Synchronises the device and clears the record."""
    words = (ctypes.c_uint * 4)()
    rc = _lib.aiter_b200_device_status(int(device), words)
    if rc != 0:
        msg = _lib.aiter_get_last_error()
        raise RuntimeError(f"aiter_b200_device_status failed: {msg.decode() if msg else ''}")
    return tuple(int(w) for w in words)


def noalloc_status(device: int = 0):
    """Same record for the allocation-free entry point, which keeps it in its own fixed array."""
    words = (ctypes.c_uint * 4)()
    rc = _lib.aiter_b200_noalloc_status(int(device), words)
    if rc != 0:
        msg = _lib.aiter_get_last_error()
        raise RuntimeError(f"aiter_b200_noalloc_status failed: {msg.decode() if msg else ''}")
    return tuple(int(w) for w in words)


def debug_wait_control(device: int = 0, limit_ns: int = 1_000_000_000, withhold_scales: bool = False) -> None:
    """Bound of the in-kernel waits on `device` and the switch that makes a GEMM's scale producer and the row loads of a
    streaming norm issue nothing (tests of the time-out path).  Call with no arguments to restore the defaults."""
    rc = _lib.aiter_b200_debug_wait_control(int(device), ctypes.c_ulonglong(int(limit_ns)), int(bool(withhold_scales)))
    if rc != 0:
        msg = _lib.aiter_get_last_error()
        raise RuntimeError(f"aiter_b200_debug_wait_control failed: {msg.decode() if msg else ''}")


def kernel_list() -> str:
    return _lib.aiter_b200_kernel_list().decode()


def heuristic_name(kind: int, M: int, N: int, K: int):
    l2 = ctypes.c_int(0)
    name = _lib.aiter_b200_heuristic_name(int(kind), int(M), int(N), int(K), ctypes.byref(l2))
    return name.decode(), int(l2.value)


def launch_count() -> int:
    return int(_lib.aiter_b200_launch_count())
