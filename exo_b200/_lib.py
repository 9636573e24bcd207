"""Loads libexo_b200.so and declares the C prototypes of include/exo_b200.h.

The product path has no CPU implementation: if the CUDA library has not been
built (``python -m exo_b200.build``) importing this module raises."""
from __future__ import annotations

import ctypes
import os

HERE = os.path.dirname(os.path.abspath(__file__))
LIB_PATH = os.path.join(HERE, "libexo_b200.so")

i64 = ctypes.c_int64  # int_fast32_t is 8 bytes on glibc x86-64
vp = ctypes.c_void_p
cbool = ctypes.c_bool

_MM_INSTANCES = ("512x512x512", "4", "6", "14", "16", "27")
_CONV_INSTANCES = ("3", "17", "30")

# name -> argtypes; every compute entry point returns void
PROTOTYPES = {
    "sgemm_exo": [vp, i64, i64, i64, vp, vp, vp],
    "sgemm_exo_ffma": [vp, i64, i64, i64, vp, vp, vp],
    "sgemm_exo_3xtf32": [vp, i64, i64, i64, vp, vp, vp],
    "conv_specialized": [vp, vp, vp, vp, vp],
    "conv": [vp] + [i64] * 8 + [vp] * 4,
    "conv_nhwc_exo": [vp] + [i64] * 7 + [cbool] + [vp] * 4,
    "conv_nhwc_exo_3xtf32": [vp] + [i64] * 7 + [cbool] + [vp] * 4,
    "conv_nhwc_strided_exo": [vp] + [i64] * 8 + [cbool] + [vp] * 4,
    "matmul_on_cpu": [vp, i64, i64, i64, vp, cbool, vp, vp, vp],
    "conv_on_cpu_stride_1": [vp] + [i64] * 6 + [vp] * 4 + [cbool, vp],
    "gemm_bf16_exo": [vp, i64, i64, i64, vp, vp, vp],
    "matmul_on_cpu_static": [vp, i64, i64, i64, vp, cbool, vp, vp, vp],
    "ssyrk_exo": [vp, i64, i64, vp, vp],
    "ssyrk_exo_ffma": [vp, i64, i64, vp, vp],
    "ssyrk_exo_3xtf32": [vp, i64, i64, vp, vp],
    "quantize_rows_bf16_exo": [vp, i64, i64, vp, vp, vp],
    "quantize_rows_f32_exo": [vp, i64, i64, vp, vp, vp],
    "gemm_i8_scaled_bf16_exo": [vp, i64, i64, i64] + [vp] * 6,
    "gemm_i8_scaled_f32_exo": [vp, i64, i64, i64] + [vp] * 6,
    "linear_i8_bf16_exo": [vp, i64, i64, i64] + [vp] * 7,
    "linear_i8_f32_exo": [vp, i64, i64, i64] + [vp] * 7,
    "gated_bf16_exo": [vp, i64, i64, i64, i64] + [vp] * 6,
    "gated_bf16_backward_exo": [vp, i64, i64, i64, i64] + [vp] * 11,
    "gated_i8_bf16_exo": [vp, i64, i64, i64, i64] + [vp] * 7,
    # the Gemmini library's "auto" entry points (include/exo_b200_gemmini_shim.h)
    "tiled_matmul_auto": [ctypes.c_size_t] * 3 + [vp] * 4 + [ctypes.c_size_t] * 4 + [ctypes.c_float] * 3
                         + [ctypes.c_int, ctypes.c_float, ctypes.c_float] + [cbool] * 5 + [ctypes.c_uint8, ctypes.c_int],
    "tiled_conv_auto": [ctypes.c_int] * 12 + [cbool] * 5 + [vp] * 4 + [ctypes.c_int, ctypes.c_float]
                       + [ctypes.c_int] * 4,
}
for _n in _MM_INSTANCES:
    PROTOTYPES[f"cpu_matmul_{_n}"] = [vp, vp, cbool, vp, vp, vp]
    PROTOTYPES[f"matmul_{_n}"] = [vp, vp, cbool, vp, vp, vp]
for _n in _CONV_INSTANCES:
    PROTOTYPES[f"conv_{_n}_cpu"] = [vp, vp, vp, vp, vp, cbool, vp]
    PROTOTYPES[f"conv_{_n}"] = [vp, vp, vp, vp, vp, cbool, vp]

# Element type and shape (as names of the sizes) of every tensor of the feed-forward entry points, in order; "?"
# marks one that may be None, "=" one that is written.  The wrapper holds arrays and tensors against these before the
# call.
_LINEAR = "M N K", "{t} M K, i8 N K, f32 N, f32? N, =i8 M K, =f32 M, ={t} M N"
_SCALED = "M N K", "i8 M K, i8 N K, f32 M, f32 N, f32? N, ={t} M N"


def _signature(sizes, tensors, t=""):
    """(number of sizes, (element type, may be None, its sizes) of each tensor, positions of the ones that are written)"""
    specs, written = [], set()
    for at, spec in enumerate(tensors.format(t=t).split(",")):
        kind, *dims = spec.split()
        specs.append((kind.strip("=?"), kind.endswith("?"), tuple(sizes.split().index(d) for d in dims)))
        if kind.startswith("="):
            written.add(at)
    return len(sizes.split()), tuple(specs), frozenset(written)


SIGNATURES = {
    "quantize_rows_bf16_exo": _signature("M K", "bf16 M K, =i8 M K, =f32 M"),
    "quantize_rows_f32_exo": _signature("M K", "f32 M K, =i8 M K, =f32 M"),
    "gemm_i8_scaled_bf16_exo": _signature(*_SCALED, "bf16"),
    "gemm_i8_scaled_f32_exo": _signature(*_SCALED, "f32"),
    "linear_i8_bf16_exo": _signature(*_LINEAR, "bf16"),
    "linear_i8_f32_exo": _signature(*_LINEAR, "f32"),
    "gated_bf16_exo": _signature("act M F K", "bf16 M K, bf16 F K, bf16 F K, =bf16 M F, =bf16? M F, =bf16? M F"),
    "gated_bf16_backward_exo": _signature(
        "act M F K", "bf16 M K, bf16 F K, bf16 F K, bf16 M F, bf16 M F, bf16 M F, =bf16 M F, =bf16 M F, "
                     "=bf16? M K, =bf16? F K, =bf16? F K"),
    "gated_i8_bf16_exo": _signature("act M F K", "i8 M K, i8 F K, i8 F K, f32 M, f32 F, f32 F, =bf16 M F"),
}

SUPPORT = {
    "exo_b200_context_create": ([ctypes.c_int, vp], vp),
    "exo_b200_context_destroy": ([vp], None),
    "exo_b200_context_set_stream": ([vp, vp], None),
    "exo_b200_context_set_sgemm_path": ([vp, ctypes.c_int], None),
    "exo_b200_set_default_stream": ([vp], None),
    "exo_b200_context_cache_weights": ([vp, ctypes.c_int], None),
    "exo_b200_context_invalidate": ([vp], None),
    "exo_b200_context_trim": ([vp], None),
    "exo_b200_synchronize": ([vp], ctypes.c_int),
    "exo_b200_selftest_bounded_wait": ([vp, ctypes.c_int], ctypes.c_int),
    "exo_b200_measure_peak": ([ctypes.c_int, ctypes.c_int], ctypes.c_double),
    "exo_b200_sgemm_kernel_choice": ([i64, i64, i64], ctypes.c_int),
    "exo_b200_last_error": ([], ctypes.c_int),
    "exo_b200_last_error_string": ([], ctypes.c_char_p),
    "exo_b200_version": ([], ctypes.c_char_p),
}

_dll = None


def load() -> ctypes.CDLL:
    global _dll
    if _dll is not None:
        return _dll
    if not os.path.exists(LIB_PATH):
        raise ImportError(
            f"{LIB_PATH} is missing: build it with `python -m exo_b200.build` "
            "(needs nvcc; there is no CPU fallback)")
    dll = ctypes.CDLL(LIB_PATH)
    for name, argtypes in PROTOTYPES.items():
        f = getattr(dll, name)
        f.argtypes = argtypes
        f.restype = None
    for name, (argtypes, restype) in SUPPORT.items():
        f = getattr(dll, name)
        f.argtypes = argtypes
        f.restype = restype
    _dll = dll
    return dll
