"""ctypes binding of the C ABI in ``include/bsgemm.h``.

The shared library is built in-tree by ``cutlass_b200/build.py`` (nvcc, sm_100a)
as ``cutlass_b200/lib/libbsgemm.so``.  There is no CPU fallback: if the library
is missing, loading raises.
"""
from __future__ import annotations

import ctypes as C
import importlib.machinery
import importlib.util
import os
import struct
import warnings

_HERE = os.path.dirname(os.path.abspath(__file__))
# BSG_PROFILE=1 selects the instrumented build (python -m cutlass_b200.build with the same variable set).
LIB_PATH = os.path.join(_HERE, "lib", "libbsgemm" + ("_profile" if os.environ.get("BSG_PROFILE") == "1" else "") + ".so")

BSG_OK = 0
STATUS_NAMES = {
    0: "BSG_OK",
    1: "BSG_ERR_MISALIGNED_OPERAND",
    2: "BSG_ERR_INVALID_PROBLEM",
    3: "BSG_ERR_NOT_SUPPORTED",
    4: "BSG_ERR_WORKSPACE_NULL",
    5: "BSG_ERR_INTERNAL",
    6: "BSG_ERR_ARCH_MISMATCH",
    7: "BSG_ERR_TIMEOUT",
    8: "BSG_ERR_CUDA",
}
KIND_NVFP4 = 0
KIND_MXFP8 = 1
KIND_MXFP4 = 2          # e2m1 data, ue8m0 scale per 32
KIND_MXFP8_MXFP4 = 3    # A e4m3, B e2m1, ue8m0 scale per 32
KIND_INT8 = 16          # signed 8-bit integers, fp32 scale per row of A and per row of B (no kind of bsg_gemm_args)
OUT_BF16 = 0
OUT_NVFP4 = 1
OUT_MXFP8 = 2
OUT_F16 = 3
OUT_F32 = 4
OUT_E4M3 = 5
OUT_E5M2 = 6
ACT_IDENTITY, ACT_RELU, ACT_GELU, ACT_SILU = 0, 1, 2, 3
BIAS_NONE, BIAS_PER_COLUMN, BIAS_PER_ROW = 0, 1, 2
MAX_GROUPS = 256
SCHED_STATIC, SCHED_DYNAMIC = 0, 1
LAYOUT_ROW_MAJOR, LAYOUT_COL_MAJOR = 0, 1
RS_WITH_ALLREDUCE = 1


class GemmArgs(C.Structure):
    _fields_ = [
        ("kind", C.c_int32), ("out_kind", C.c_int32), ("batch", C.c_int32), ("reserved0", C.c_int32),
        ("M", C.c_int64), ("N", C.c_int64), ("K", C.c_int64),
        ("A", C.c_void_p), ("B", C.c_void_p), ("SFA", C.c_void_p), ("SFB", C.c_void_p),
        ("C", C.c_void_p), ("D", C.c_void_p), ("SFD", C.c_void_p),
        ("ldc", C.c_int64), ("ldd", C.c_int64),
        ("alpha", C.c_float), ("beta", C.c_float),
        ("alpha_ptr", C.c_void_p), ("beta_ptr", C.c_void_p), ("norm_constant", C.c_void_p),
        ("tile_n", C.c_int32), ("cta_group", C.c_int32), ("sm_count", C.c_int32), ("raster_band", C.c_int32),
        ("bias", C.c_void_p), ("bias_mode", C.c_int32), ("activation", C.c_int32),
        ("lda", C.c_int64), ("ldb", C.c_int64),
        ("batch_stride_A", C.c_int64), ("batch_stride_B", C.c_int64), ("batch_stride_C", C.c_int64), ("batch_stride_D", C.c_int64),
        ("use_pdl", C.c_int32), ("scheduler", C.c_int32),
        ("cluster_m", C.c_int32), ("cluster_n", C.c_int32), ("cluster_fallback_m", C.c_int32), ("cluster_fallback_n", C.c_int32),
        ("out_layout", C.c_int32), ("reserved1", C.c_int32),
    ]


class GroupedArgs(C.Structure):
    _fields_ = [
        ("kind", C.c_int32), ("out_kind", C.c_int32), ("num_groups", C.c_int32), ("reserved0", C.c_int32),
        ("total_M", C.c_int64), ("N", C.c_int64), ("K", C.c_int64),
        ("A", C.c_void_p), ("B", C.c_void_p), ("SFA", C.c_void_p), ("SFB", C.c_void_p),
        ("C", C.c_void_p), ("D", C.c_void_p), ("offsets", C.c_void_p),
        ("ldc", C.c_int64), ("ldd", C.c_int64),
        ("alpha", C.c_float), ("beta", C.c_float),
        ("tile_n", C.c_int32), ("cta_group", C.c_int32), ("sm_count", C.c_int32), ("raster_band", C.c_int32),
        ("bias", C.c_void_p), ("reserved1", C.c_int32), ("activation", C.c_int32),
        ("alpha_array", C.c_void_p), ("beta_array", C.c_void_p),
        ("SFD", C.c_void_p), ("norm_constant", C.c_void_p), ("use_pdl", C.c_int32), ("scheduler", C.c_int32),
    ]


class Caps(C.Structure):
    _fields_ = [
        ("tile_m", C.c_int32), ("tile_n", C.c_int32), ("tile_k", C.c_int32), ("cta_group", C.c_int32),
        ("stages", C.c_int32), ("smem_bytes", C.c_int32), ("num_tiles", C.c_int64),
    ]


class PtrArrayArgs(C.Structure):
    """``bsg_ptr_array_args`` of include/bsgemm.h, field for field (the arrays are HOST arrays)."""
    _fields_ = [
        ("kind", C.c_int32), ("out_kind", C.c_int32), ("num_groups", C.c_int32), ("activation", C.c_int32),
        ("problem_sizes", C.c_void_p),
        ("A", C.c_void_p), ("B", C.c_void_p), ("SFA", C.c_void_p), ("SFB", C.c_void_p), ("C", C.c_void_p), ("D", C.c_void_p), ("SFD", C.c_void_p),
        ("lda", C.c_void_p), ("ldb", C.c_void_p), ("ldc", C.c_void_p), ("ldd", C.c_void_p),
        ("alpha", C.c_float), ("beta", C.c_float),
        ("alpha_array", C.c_void_p), ("beta_array", C.c_void_p), ("norm_constant", C.c_void_p),
        ("tile_n", C.c_int32), ("sm_count", C.c_int32), ("raster_band", C.c_int32), ("use_pdl", C.c_int32),
    ]


# name -> (restype, argtypes); every symbol include/bsgemm.h declares.
class QuantArgs(C.Structure):
    """``bsg_quant_args`` of include/bsgemm.h, field for field."""
    _fields_ = [("kind", C.c_int32), ("use_pdl", C.c_int32), ("rows", C.c_int64), ("K", C.c_int64), ("X", C.c_void_p),
                ("ldx", C.c_int64), ("Q", C.c_void_p), ("SF", C.c_void_p), ("norm_constant", C.c_void_p)]


INT8_LAYOUT = "4i4qPqPPqPPqqPPPPq4i"      # Int8Args, ActArgs and RouteArgs below as struct formats
ACT_LAYOUT = "4i2qPqPqPP"
ROUTE_LAYOUT = "4iqPq13Pq"


class Int8Args(C.Structure):
    """``bsg_int8_args`` of include/bsgemm.h, field for field."""
    _fields_ = [
        ("in_kind", C.c_int32), ("out_kind", C.c_int32), ("num_groups", C.c_int32), ("activation", C.c_int32),
        ("rows", C.c_int64), ("tokens", C.c_int64), ("N", C.c_int64), ("K", C.c_int64),
        ("X", C.c_void_p), ("ldx", C.c_int64), ("index", C.c_void_p), ("Q", C.c_void_p), ("ldq", C.c_int64), ("q_scale", C.c_void_p),
        ("W", C.c_void_p), ("ldw", C.c_int64), ("group_stride_w", C.c_int64), ("w_scale", C.c_void_p), ("bias", C.c_void_p),
        ("offsets", C.c_void_p), ("D", C.c_void_p), ("ldd", C.c_int64),
        ("kernel", C.c_int32), ("tile", C.c_int32), ("split", C.c_int32), ("reserved0", C.c_int32),
    ]


class ActArgs(C.Structure):
    """``bsg_act_args`` of include/bsgemm.h, field for field."""
    _fields_ = [
        ("type", C.c_int32), ("activation", C.c_int32), ("gated", C.c_int32), ("reserved0", C.c_int32), ("rows", C.c_int64), ("width", C.c_int64),
        ("in_", C.c_void_p), ("ld_in", C.c_int64), ("out", C.c_void_p), ("ld_out", C.c_int64), ("kept", C.c_void_p), ("kept_scale", C.c_void_p),
    ]


class RouteArgs(C.Structure):
    """``bsg_route_args`` of include/bsgemm.h, field for field."""
    _fields_ = [
        ("type", C.c_int32), ("experts", C.c_int32), ("k", C.c_int32), ("normalize", C.c_int32), ("tokens", C.c_int64),
        ("logits", C.c_void_p), ("ld", C.c_int64), ("mask", C.c_void_p),
        ("chosen", C.c_void_p), ("weights", C.c_void_p), ("counts", C.c_void_p), ("live", C.c_void_p), ("softmax", C.c_void_p),
        ("offsets", C.c_void_p), ("rows", C.c_void_p), ("positions", C.c_void_p), ("loss", C.c_void_p),
        ("grad_weights", C.c_void_p), ("grad_loss", C.c_void_p), ("grad_logits", C.c_void_p), ("ld_grad", C.c_int64),
    ]


SYMBOLS = {
    "bsg_version": (C.c_int32, []),
    "bsg_last_error_string": (C.c_char_p, []),
    "bsg_gemm_query": (C.c_int32, [C.POINTER(GemmArgs), C.POINTER(Caps)]),
    "bsg_grouped_query": (C.c_int32, [C.POINTER(GroupedArgs), C.POINTER(Caps)]),
    "bsg_gemm_workspace_size": (C.c_int32, [C.POINTER(GemmArgs), C.POINTER(C.c_size_t)]),
    "bsg_grouped_workspace_size": (C.c_int32, [C.POINTER(GroupedArgs), C.POINTER(C.c_size_t)]),
    "bsg_gemm_run": (C.c_int32, [C.POINTER(GemmArgs), C.c_void_p, C.c_size_t, C.c_void_p]),
    "bsg_grouped_run": (C.c_int32, [C.POINTER(GroupedArgs), C.c_void_p, C.c_size_t, C.c_void_p]),
    "bsg_workspace_init": (C.c_int32, [C.c_void_p, C.c_size_t, C.c_void_p]),
    "bsg_read_device_status": (C.c_int32, [C.c_void_p, C.c_void_p]),
    "bsg_gemm_run_static": (C.c_int32, [C.POINTER(GemmArgs), C.c_void_p, C.POINTER(C.c_uint32)]),
    "bsg_ptr_array_workspace_size": (C.c_int32, [C.POINTER(PtrArrayArgs), C.POINTER(C.c_size_t)]),
    "bsg_ptr_array_initialize": (C.c_int32, [C.POINTER(PtrArrayArgs), C.c_void_p, C.c_size_t, C.c_void_p]),
    "bsg_ptr_array_initialize_from_device": (C.c_int32, [C.POINTER(PtrArrayArgs), C.c_void_p, C.c_size_t, C.c_void_p]),
    "bsg_ptr_array_run": (C.c_int32, [C.POINTER(PtrArrayArgs), C.c_void_p, C.c_size_t, C.c_void_p]),
    "bsg_quantize": (C.c_int32, [C.POINTER(QuantArgs), C.c_void_p]),
    "bsg_int8_query": (C.c_int32, [C.POINTER(Int8Args), C.POINTER(Caps)]),
    "bsg_int8_scratch_rows": (C.c_int32, [C.POINTER(Int8Args), C.POINTER(C.c_int64)]),
    "bsg_int8_quantize": (C.c_int32, [C.POINTER(Int8Args), C.c_void_p]),
    "bsg_int8_gemm_run": (C.c_int32, [C.POINTER(Int8Args), C.c_void_p, C.c_size_t, C.c_void_p]),
    "bsg_int8_linear_run": (C.c_int32, [C.POINTER(Int8Args), C.c_void_p, C.c_size_t, C.c_void_p]),
    "bsg_act_forward": (C.c_int32, [C.POINTER(ActArgs), C.c_void_p]),
    "bsg_act_backward": (C.c_int32, [C.POINTER(ActArgs), C.c_void_p]),
    "bsg_route_scratch_size": (C.c_int32, [C.POINTER(RouteArgs), C.POINTER(C.c_size_t)]),
    "bsg_route_forward": (C.c_int32, [C.POINTER(RouteArgs), C.c_void_p, C.c_size_t, C.c_void_p]),
    "bsg_route_backward": (C.c_int32, [C.POINTER(RouteArgs), C.c_void_p]),
    "bsg_tp_create": (C.c_int32, [C.c_int32, C.c_int32, C.c_int32, C.c_int64, C.c_int64, C.POINTER(C.c_void_p), C.c_void_p]),
    "bsg_tp_connect": (C.c_int32, [C.c_void_p, C.c_void_p]),
    "bsg_tp_buffers": (C.c_int32, [C.c_void_p] + [C.POINTER(C.c_void_p)] * 4),
    "bsg_tp_gemm_run": (C.c_int32, [C.c_void_p, C.POINTER(GemmArgs), C.c_void_p, C.c_size_t, C.c_void_p]),
    "bsg_tp_set_mode": (C.c_int32, [C.c_void_p, C.c_int32]),
    "bsg_tp_destroy": (C.c_int32, [C.c_void_p]),
    "bsg_rs_create": (C.c_int32, [C.c_int32, C.c_int32, C.c_int64, C.c_int64, C.c_int32, C.POINTER(C.c_void_p), C.c_void_p]),
    "bsg_rs_connect": (C.c_int32, [C.c_void_p, C.c_void_p]),
    "bsg_rs_gemm_run": (C.c_int32, [C.c_void_p, C.POINTER(GemmArgs), C.c_void_p, C.c_size_t, C.c_void_p]),
    "bsg_rs_allreduce_run": (C.c_int32, [C.c_void_p, C.POINTER(GemmArgs), C.c_void_p, C.c_size_t, C.c_void_p, C.POINTER(C.c_void_p)]),
    "bsg_rs_destroy": (C.c_int32, [C.c_void_p]),
}

_lib = None
_direct: dict = {}
BINDING_PATH = os.path.join(_HERE, "lib", "_binding.so")
# What csrc/binding.cpp calls, in the order of its table.
BOUND = ("bsg_int8_linear_run", "bsg_int8_scratch_rows", "bsg_act_forward", "bsg_act_backward", "bsg_route_forward", "bsg_route_backward",
         "bsg_route_scratch_size", "bsg_last_error_string")
_binding = None


class _NoBinding:
    """Stands in for the binding: every call is left to the Python around it."""

    def __getattr__(self, name):
        return lambda *args: None


def _load_binding():
    if not os.path.exists(BINDING_PATH):
        raise ImportError(f"{BINDING_PATH} is missing")
    from .build import _binding_for
    loader = importlib.machinery.ExtensionFileLoader("_binding", BINDING_PATH)
    module = importlib.util.module_from_spec(importlib.util.spec_from_loader("_binding", loader))
    loader.exec_module(module)
    if module.made_for != _binding_for():
        raise ImportError(f"{BINDING_PATH} was made for {module.made_for}, this is {_binding_for()}")
    return module


def binding():
    """The module of ``csrc/binding.cpp``: whole calls with little host time.  Each of its functions returns None, having done
    nothing, for a call that is not the plain case; the Python around it then does the work or says what is wrong.  Where the module
    is missing, or was made for another Python or torch, that Python makes every call, and a warning says so once."""
    global _binding
    if _binding is None:
        lib = load()
        try:
            module = _load_binding()
        except ImportError as error:
            warnings.warn(f"{error}: calls take more host time without the binding; build it with `python -m cutlass_b200.build`", RuntimeWarning)
            _binding = _NoBinding()
            return _binding
        from .activation import ActivationCheckpoint
        from .arguments import ACTIVATIONS
        from .operator import _default_workspaces
        from .routing import Routing
        module.bind(check, ACTIVATIONS, _default_workspaces, ActivationCheckpoint, Routing, *(C.cast(getattr(lib, name), C.c_void_p).value for name in BOUND))
        _binding = module
    return _binding


def direct(name: str, layout: str):
    """(pack, call) of an entry point whose argument struct is passed as packed bytes: ``pack(*fields)`` lays the fields out as
    ``layout`` (native alignment) says, ``call(bytes, ...)`` takes the other arguments as integers.  A call through
    ``ctypes.Structure`` costs several microseconds more, which a kernel of a few microseconds does not hide."""
    found = _direct.get(name)
    if found is None:
        fn = load()[name]                    # a function object of its own: the prototypes of SYMBOLS stay as they are
        fn.restype = C.c_int32
        fn.argtypes = [C.c_char_p] + [C.c_void_p if t is not C.c_size_t else t for t in SYMBOLS[name][1][1:]]
        found = _direct[name] = (struct.Struct("@" + layout).pack, fn)
    return found


class BsgError(RuntimeError):
    def __init__(self, code: int, message: str):
        super().__init__(f"{STATUS_NAMES.get(code, code)}: {message}")
        self.code = code


def load() -> C.CDLL:
    """Load ``libbsgemm.so`` (once) and declare the prototypes."""
    global _lib
    if _lib is not None:
        return _lib
    if not os.path.exists(LIB_PATH):
        raise FileNotFoundError(
            f"{LIB_PATH} is missing: build it with `python -m cutlass_b200.build` (needs nvcc); "
            "there is no CPU fallback for the GEMM path")
    lib = C.CDLL(LIB_PATH)
    for name, (restype, argtypes) in SYMBOLS.items():
        fn = getattr(lib, name)
        fn.restype = restype
        fn.argtypes = argtypes
    _lib = lib
    return lib


def last_error() -> str:
    return load().bsg_last_error_string().decode("utf-8", "replace")


def check(code: int) -> None:
    if code != BSG_OK:
        raise BsgError(code, last_error())
