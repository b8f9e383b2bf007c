"""ctypes binding of libmvquant.so (declared in include/mvquant.h).

Every entry point takes one struct of 8-byte fields and a stream. The struct is
packed into an immutable bytes object for each call (one C call instead of a
marshalled argument each), so calls from several threads share nothing. As with
libmvdecode.so the library is loaded on first use and there is no fallback.

``binding()`` is the same entry points' usual calls as Python functions
(csrc/mvq_binding.cpp), which return None for every call that is not usual.
"""
import ctypes
import importlib.machinery
import importlib.util
import os
import struct
from functools import lru_cache
from pathlib import Path

from . import _native, _tensors

# MVQUANT_LIBRARY may name another build of the same library (e.g. a tuning variant).
LIB_PATH = Path(os.environ.get('MVQUANT_LIBRARY', Path(__file__).resolve().parent / 'lib' / 'libmvquant.so'))

BINDING_PATH = Path(__file__).resolve().parent / 'lib' / '_mvq_binding.so'

MVQ_ABI_VERSION = 1
DTYPE_F32, DTYPE_F16, DTYPE_BF16, DTYPE_I8, DTYPE_E4M3 = 0, 1, 2, 3, 4

# Field names of the argument structs, in order; 'eps' is a double, the rest 64-bit integers or pointers.
LINEAR_FIELDS = ('x', 'x_stride_row', 'x_scale', 'records', 'n', 'k', 'group', 'has_zeros', 'scale_dtype',
                 'bias', 'residual', 'residual_stride_row', 'out', 'out_stride_row', 'm', 'x_dtype', 'out_dtype')
DEQUANTIZE_FIELDS = ('records', 'n', 'k', 'group', 'has_zeros', 'scale_dtype', 'out', 'out_stride_row', 'out_dtype')
NORM_FIELDS = ('x', 'x_stride_row', 'residual', 'residual_stride_row', 'weight', 'out', 'out_stride_row', 'scales',
               'residual_out', 'residual_out_stride_row', 'rows', 'hidden', 'eps', 'dtype', 'out_dtype')
SILU_FIELDS = ('gate_up', 'stride_row', 'out', 'out_stride_row', 'scales', 'rows', 'width', 'dtype', 'out_dtype')


# The fields that describe a weight, the same in two structs.
pack_weight = struct.Struct('=6q').pack


def _packer(fields):
    return struct.Struct('=' + ''.join('d' if name == 'eps' else 'q' for name in fields)).pack


pack_linear = _packer(LINEAR_FIELDS)
pack_dequantize = _packer(DEQUANTIZE_FIELDS)
pack_norm = _packer(NORM_FIELDS)
pack_silu = _packer(SILU_FIELDS)

ENTRY_POINTS = ('mvq_w4_linear', 'mvq_w4_dequantize', 'mvq_add_rms_norm', 'mvq_silu_mul_quant')
EXPORTED_SYMBOLS = ENTRY_POINTS + ('mvq_abi_version', 'mvq_last_error', 'mvq_device_status',
                                   'mvq_clear_device_status', 'mvq_selftest_wait_timeout')
DEVICE_STATUS_WAIT_TIMEOUT = 1


@lru_cache(maxsize=1)
def library() -> ctypes.CDLL:
    """Load libmvquant.so once; raise if it is absent or incompatible."""
    if not LIB_PATH.exists():
        raise RuntimeError(
            f'{LIB_PATH} is not built: run `python -m micro_vllm_b200.build` '
            '(or __graft_entry__.build()) before using the CUDA kernels')
    lib = ctypes.CDLL(str(LIB_PATH))
    for name in ENTRY_POINTS:
        fn = getattr(lib, name)
        fn.restype = ctypes.c_int
        fn.argtypes = [ctypes.c_char_p, ctypes.c_void_p]
    lib.mvq_device_status.restype = lib.mvq_clear_device_status.restype = ctypes.c_int
    lib.mvq_device_status.argtypes = [ctypes.c_int32, ctypes.POINTER(ctypes.c_uint32)]
    lib.mvq_clear_device_status.argtypes = [ctypes.c_int32]
    lib.mvq_selftest_wait_timeout.restype = ctypes.c_int
    lib.mvq_selftest_wait_timeout.argtypes = [ctypes.c_uint64, ctypes.c_void_p]
    lib.mvq_abi_version.restype = ctypes.c_int
    lib.mvq_last_error.restype = ctypes.c_char_p
    version = lib.mvq_abi_version()
    if version != MVQ_ABI_VERSION:
        raise RuntimeError(f'libmvquant ABI {version}, expected {MVQ_ABI_VERSION}')
    return lib


@lru_cache(maxsize=1)
def binding():
    """Load _mvq_binding.so once and give it the library's entry points."""
    if not BINDING_PATH.exists():
        raise RuntimeError(
            f'{BINDING_PATH} is not built: run `python -m micro_vllm_b200.build` '
            '(or __graft_entry__.build()) before using the CUDA kernels')
    lib = library()
    loader = importlib.machinery.ExtensionFileLoader('_mvq_binding', str(BINDING_PATH))
    module = importlib.util.module_from_spec(importlib.util.spec_from_loader('_mvq_binding', loader))
    loader.exec_module(module)
    module.bind(*(ctypes.cast(getattr(lib, name), ctypes.c_void_p).value for name in ENTRY_POINTS))
    return module


def refuse_transforms(*tensors) -> None:
    """Raise where one of the tensors (or None) asks for what the kernels pass by (_tensors.refuse_transforms)."""
    if binding().any_transformed(*tensors):
        for t in tensors:
            if t is not None:
                _tensors.refuse_transforms(t, 'a tensor of this call')


def check(status: int) -> None:
    if status != _native.MV_OK:
        raise _native.NativeError(status, library().mvq_last_error().decode(errors='replace'))
