"""ctypes binding of ``libsq_b200.so`` (C ABI declared in ``include/sq_b200.h``).

There is no fallback: if the library has not been built, or no CUDA device is
present when a kernel is requested, the call raises.
"""
from __future__ import annotations

import ctypes
import importlib.machinery
import importlib.util
import struct
import warnings
from ctypes import c_char_p, c_float, c_int, c_int32, c_int64, c_size_t, c_void_p
from functools import lru_cache
from pathlib import Path

from .build import binding_path

LIB_PATH = Path(__file__).resolve().parent / "lib" / "libsq_b200.so"

# status codes of include/sq_b200.h
OK, ERR_NULL, ERR_SHAPE, ERR_ENUM, ERR_INDEX, ERR_DRIVER, ERR_WORKSPACE, ERR_DEVICE_WAIT = 0, -1, -2, -3, -4, -5, -6, -7
ERR_SCRATCH_LIMIT = -8
ERR_OVERLAP = -9
NOALLOC_SCRATCH_BYTES = 8 * 1024 * 1024 + 65536
BF16, FP16 = 0, 1
ACT_STATIC, ACT_TOKEN = 0, 1
CODES_NATURAL, CODES_EVEN_ODD = 0, 1
WEIGHTS_PREPACKED = 4  # OR-ed onto the weight-scale mode: weights are int8 [N, K] from sq_prepack_weights
CODES_INT4_RANGE = 2  # OR-ed onto the layout for sq_gemm: every code lies in [-8, 7]
WSCALE_CHANNEL_F32, WSCALE_GROUP_F16 = 0, 1
NORM_NONE, NORM_LAYER, NORM_RMS = 0, 1, 2
ROTARY_AXES = 4
ROTARY_INTERLEAVED, ROTARY_HALF = 0, 1
ROTARY_NORM_NONE, ROTARY_NORM_HEAD, ROTARY_NORM_TOKEN = 0, 1, 2
POS_INT32, POS_INT64, POS_FP32 = 0, 1, 2
ACT_FN_NONE, ACT_FN_GELU = 0, 1


class Param(ctypes.Structure):
    """``SqParam``: rows of parameters."""
    _fields_ = [("data", c_void_p), ("row_stride", c_int64), ("span", c_int64), ("is_fp32", c_int32), ("reserved", c_int32)]


class BlockNorm(ctypes.Structure):
    """``SqBlockNorm``."""
    _fields_ = [("x", c_void_p), ("branch", c_void_p),
                *((name, Param) for name in ("gate", "post_weight", "post_bias", "weight", "bias", "mod_scale", "mod_shift")),
                ("h_out", c_void_p), ("z_out", c_void_p), ("scales", c_void_p), ("scales_row_stride", c_int64),
                ("scales_group_stride", c_int64), ("rows", c_int64), ("width", c_int64), ("residual_scale", c_float),
                ("eps", c_float), ("dtype", c_int32), ("post_kind", c_int32), ("norm_kind", c_int32), ("reserved", c_int32)]


class Rotary(ctypes.Structure):
    """``SqRotary``."""
    _fields_ = [("q", c_void_p), ("k", c_void_p), ("q_out", c_void_p), ("k_out", c_void_p),
                *((name, c_int64 * 3) for name in ("q_strides", "k_strides", "q_out_strides", "k_out_strides")),
                ("q_weight", c_void_p), ("k_weight", c_void_p), ("positions", c_void_p),
                ("position_batch_stride", c_int64), ("position_token_stride", c_int64), ("inv_freq", c_void_p),
                ("batch", c_int64), ("length", c_int64), ("heads", c_int32), ("kv_heads", c_int32), ("dim", c_int32),
                ("axes", c_int32), ("sections", c_int32 * ROTARY_AXES), ("dtype", c_int32), ("layout", c_int32),
                ("norm", c_int32), ("position_type", c_int32), ("q_weight_fp32", c_int32), ("k_weight_fp32", c_int32),
                ("eps", c_float), ("reserved", c_int32)]


# the same two layouts by position, null pointers as 0: packing one takes a quarter of the time of filling the structure
BLOCK_NORM = struct.Struct("@PP" + 7 * "Pqqii" + "PPPqqqqffiiii")
ROTARY = struct.Struct("@PPPP12qPPPqqPqqiiii4iiiiiiifi")
assert BLOCK_NORM.size == ctypes.sizeof(BlockNorm) and ROTARY.size == ctypes.sizeof(Rotary)


_SIGNATURES = {
    "sq_prepass": (c_int, [c_void_p, c_int, c_int64, c_int64, c_int, c_int, c_void_p, c_void_p, c_int,
                           c_void_p, c_void_p, c_int64, c_int64, c_int64, c_int, c_int, c_void_p, c_void_p, c_void_p]),
    "sq_gemm": (c_int, [c_void_p, c_int, c_void_p, c_void_p, c_int, c_void_p, c_void_p, c_void_p, c_int,
                        c_int64, c_int64, c_int64, c_void_p, c_void_p]),
    "sq_gemm_split": (c_int, [c_void_p, c_int, c_void_p, c_void_p, c_int, c_void_p, c_void_p, c_void_p, c_int,
                              c_int64, c_int64, c_int64, c_void_p, c_void_p, c_size_t, c_void_p]),
    "sq_split_workspace_bytes": (c_size_t, [c_int64]),
    "sq_gemm_scatter": (c_int, [c_void_p, c_int, c_void_p, c_void_p, c_int, c_void_p, c_void_p, c_void_p, c_int, c_int64,
                                c_int64, c_int, c_int64, c_int64, c_int64, c_void_p]),
    "sq_gemm_check": (c_int, [c_void_p, c_int, c_void_p, c_void_p, c_int, c_void_p, c_void_p, c_void_p, c_int,
                              c_int64, c_int64, c_int64, c_void_p, c_void_p]),
    "sq_gemm_timeline": (c_int, [c_void_p, c_void_p, c_void_p, c_void_p, c_void_p, c_void_p, c_int64, c_int64, c_int64,
                                 c_void_p, c_void_p]),
    "sq_prepack_weights": (c_int, [c_void_p, c_int64, c_int64, c_void_p, c_void_p]),
    "sq_mma_rate": (c_int, [c_int, c_int, c_void_p, c_void_p]),
    "sq_workspace_bytes": (c_size_t, [c_int64, c_int64]),
    "sq_linear": (c_int, [c_void_p, c_int, c_int64, c_int64, c_int64, c_int, c_int, c_void_p, c_void_p, c_int,
                          c_void_p, c_void_p, c_int64, c_int64, c_int64, c_int64, c_int64,
                          c_void_p, c_void_p, c_int, c_void_p, c_void_p, c_void_p, c_size_t, c_void_p]),
    "sq_linear_fused": (c_int, [c_void_p, c_int, c_int64, c_int64, c_int64, c_int, c_int, c_void_p, c_void_p, c_int,
                                c_void_p, c_void_p, c_int64, c_int64, c_int64, c_int64, c_int64,
                                c_void_p, c_void_p, c_int, c_void_p,
                                c_int, c_int, c_float, c_void_p, c_void_p, c_void_p, c_int64, c_int64, c_int,
                                c_int, c_void_p, c_int64, c_int64, c_void_p,
                                c_void_p, c_void_p, c_size_t, c_void_p]),
    "sq_linear_scheduled": (c_int, [c_void_p, c_int, c_int64, c_int64, c_int64, c_int, c_int, c_void_p, c_void_p, c_int,
                                    c_void_p, c_void_p, c_int64, c_int64, c_void_p, c_int64, c_int64, c_int64,
                                    c_void_p, c_void_p, c_int, c_void_p,
                                    c_int, c_int, c_float, c_void_p, c_void_p, c_void_p, c_int64, c_int64, c_int,
                                    c_int, c_void_p, c_int64, c_int64, c_void_p,
                                    c_void_p, c_void_p, c_size_t, c_void_p]),
    "sq_prepass_composite": (c_int, [c_void_p, c_int, c_int64, c_int64, c_int, c_int, c_void_p, c_void_p, c_void_p, c_int,
                                     c_void_p, c_void_p, c_int64, c_int64, c_int64, c_int, c_int, c_void_p, c_void_p,
                                     c_void_p]),
    "sq_linear_composite": (c_int, [c_void_p, c_int, c_int64, c_int64, c_int64, c_int, c_int, c_void_p, c_void_p,
                                    c_void_p, c_int, c_void_p, c_void_p, c_int64, c_int64, c_void_p, c_int64, c_int64, c_int64,
                                    c_void_p, c_void_p, c_int, c_void_p, c_void_p, c_void_p, c_size_t, c_void_p]),
    "sq_linear_noalloc": (c_int, [c_void_p, c_int, c_int64, c_int64, c_int64, c_int, c_int, c_void_p, c_void_p, c_int,
                                  c_void_p, c_void_p, c_int64, c_int64, c_int64, c_int64, c_int64,
                                  c_void_p, c_void_p, c_int, c_void_p, c_void_p, c_void_p]),
    "sq_fp8_quantize": (c_int, [c_void_p, c_int, c_int64, c_int64, c_int, c_void_p, c_void_p, c_int64, c_int64, c_void_p]),
    "sq_fp8_gemm": (c_int, [c_void_p, c_void_p, c_int64, c_int64, c_void_p, c_void_p, c_void_p, c_void_p, c_int,
                            c_int64, c_int64, c_int64, c_void_p]),
    "sq_fp8_linear": (c_int, [c_void_p, c_int, c_int64, c_int64, c_int64, c_int, c_void_p, c_void_p, c_void_p, c_void_p,
                              c_void_p, c_size_t, c_void_p]),
    "sq_fp8_workspace_bytes": (c_size_t, [c_int64, c_int64]),
    "sq_block_norm": (c_int, [c_void_p, c_void_p]),
    "sq_rotary": (c_int, [c_void_p, c_void_p]),
    "sq_wait_probe": (c_int, [c_int64, c_void_p, c_void_p]),
    "sq_device_status": (c_int, []),
    "sq_status_string": (c_char_p, [c_int]),
    "sq_version": (c_char_p, []),
}

EXPORTED = tuple(_SIGNATURES)


@lru_cache(maxsize=1)
def load_library() -> ctypes.CDLL:
    if not LIB_PATH.exists():
        raise RuntimeError(
            f"{LIB_PATH} is missing: build it with `python {LIB_PATH.parents[1] / 'build.py'}` "
            "(needs nvcc). There is no fallback path.")
    lib = ctypes.CDLL(str(LIB_PATH))
    for name, (restype, argtypes) in _SIGNATURES.items():
        fn = getattr(lib, name)
        fn.restype = restype
        fn.argtypes = argtypes
    return lib


@lru_cache(maxsize=1)
def load_binding():
    """The binding (``csrc/sq_binding.cpp``), the short way into the library for ordinary calls of the block operators, or None:
    where none was built for this interpreter and PyTorch, or it does not load, the ctypes way serves every call."""
    path = binding_path()
    if path is None or not path.exists():
        return None
    load_library()
    import torch  # noqa: F401  (the module links its libraries)
    loader = importlib.machinery.ExtensionFileLoader("sq_binding", str(path))
    spec = importlib.util.spec_from_file_location("sq_binding", str(path), loader=loader)
    try:
        module = importlib.util.module_from_spec(spec)
        loader.exec_module(module)
    except ImportError as error:
        warnings.warn(f"{path.name} does not load, the block operators' calls go through ctypes: {error}")
        return None
    return module


def status_string(status: int) -> str:
    return load_library().sq_status_string(int(status)).decode()


def check(status: int, what: str) -> None:
    """Turn a non-zero status into the exception type the reference raises at the
    same place: argument errors found by its C++ checks are RuntimeError
    (TORCH_CHECK, kernels/w4a8/csrc/w4a8.cu:1079-1115).  Overlap, which only the block
    operators look for, is a ValueError like their other refusals."""
    if status == ERR_OVERLAP:
        raise ValueError(f"{what}: {status_string(status)}.")
    if status != OK:
        raise RuntimeError(f"{what}: {status_string(status)} (status {status})")
