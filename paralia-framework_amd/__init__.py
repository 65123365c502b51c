"""ctypes face of libparalia.so, the MI355X-native PARALiA runtime.

The product is the shared library (HIP kernels, C ABI, C++ scheduler and autotuner); this module only declares
its C signatures for Python callers such as the tests and the benchmark.  There is no Python or CPU fallback:
loading fails loudly when the library has not been built.
"""
from .binding import (LIB_PATH, PKG_DIR, ParaliaError, atc_info, build_library, check, epilogue, lib, load, plan_rows,
                      PL_ACT_GELU, PL_ACT_GELU_TANH, PL_ACT_NONE, PL_ACT_RELU, PL_ACT_SILU, PL_PLAN_ROW, PL_PLAN_MAX_WAITS,
                      PL_TYPE_BF16, PL_TYPE_F16, PL_TYPE_F32, PL_TYPE_F64)

__all__ = ["LIB_PATH", "PKG_DIR", "ParaliaError", "atc_info", "build_library", "check", "epilogue", "lib", "load", "plan_rows",
           "PL_ACT_GELU", "PL_ACT_GELU_TANH", "PL_ACT_NONE", "PL_ACT_RELU", "PL_ACT_SILU", "PL_PLAN_ROW", "PL_PLAN_MAX_WAITS",
           "PL_TYPE_BF16", "PL_TYPE_F16", "PL_TYPE_F32", "PL_TYPE_F64"]
