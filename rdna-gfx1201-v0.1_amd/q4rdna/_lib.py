"""ctypes binding of libq4rdna_gfx950.so (the C ABI in include/q4rdna.h).

The library is built in-tree (``make -C rdna-gfx1201-v0.1_amd``); importing
this module never falls back to anything else: a missing library raises.
"""
from __future__ import annotations

import ctypes
import os
import struct

HERE = os.path.dirname(os.path.abspath(__file__))
LIB_NAME = "libq4rdna_gfx950.so"
LIB_PATH = os.path.join(HERE, LIB_NAME)

OK = 0
NOT_APPLICABLE = 1
ERR_ARGUMENT = -1
ERR_FORMAT = -2
ERR_IO = -3
ERR_HIP = -4
ERR_MEMORY = -5

GROUP = 64
TILE_ROWS = 32
TILE_BYTES = 1088

ALGO_SIDECAR = 0
ALGO_ABSMAX = 1
ALGO_RANGE = 2
ALGO_MSE = 3

GLU_SWIGLU = 0
MAX_BATCH = 8
NOALLOC_SLOTS = 1 << 21

F32 = 0
F16 = 1
BF16 = 2
KV_BLOCK = 64
NORM_MAX_WIDTH = 16384

# Every symbol include/q4rdna.h declares.
EXPORTS = (
    "q4rdna_abi_version", "q4rdna_last_error", "q4rdna_sidecar_inspect", "q4rdna_sidecar_open",
    "q4rdna_sidecar_open_memory", "q4rdna_sidecar_close", "q4rdna_sidecar_count", "q4rdna_sidecar_entry",
    "q4rdna_find", "q4rdna_weight_from_device", "q4rdna_default_sidecar", "q4rdna_scope_allows",
    "q4rdna_mul_mat", "q4rdna_mul_mat_add", "q4rdna_mul_mat_glu", "q4rdna_mul_mat_ex", "q4rdna_mul_mat_batch",
    "q4rdna_policy_split_k", "q4rdna_mul_mat_ex_noalloc", "q4rdna_mul_mat_group", "q4rdna_plan_create", "q4rdna_plan_create_batch", "q4rdna_plan_launch",
    "q4rdna_plan_prepare",
    "q4rdna_plan_sweep", "q4rdna_plan_destroy",
    "q4rdna_plan_workgroups", "q4rdna_pack", "q4rdna_dequantize",
    "q4rdna_launch_count", "q4rdna_sidecar_hits", "q4rdna_report_stats",
    "q4rdna_kv_append", "q4rdna_kv_attend", "q4rdna_kv_read", "q4rdna_add_norm",
)


class Q4RdnaError(RuntimeError):
    """A negative status from the library."""

    def __init__(self, code: int, message: str):
        super().__init__(f"q4rdna error {code}: {message}")
        self.code = code


class Weight(ctypes.Structure):
    _fields_ = [("tiles", ctypes.c_void_p), ("rows", ctypes.c_uint32), ("columns", ctypes.c_uint32),
                ("device", ctypes.c_int32), ("reserved", ctypes.c_uint32)]


KERNEL_POLICY = 0
KERNEL_VALU = 1
KERNEL_SEQUENTIAL = 3
MAX_GROUP = 8


class LaunchOptions(ctypes.Structure):
    _fields_ = [("split_k", ctypes.c_uint32), ("kernel", ctypes.c_uint32), ("reserved", ctypes.c_uint32 * 6)]


class GroupDesc(ctypes.Structure):
    _fields_ = [("weight", Weight), ("gate_tiles", ctypes.c_void_p), ("add", ctypes.c_void_p), ("y", ctypes.c_void_p)]


class GemvDesc(ctypes.Structure):
    _fields_ = [("weight", Weight), ("gate_tiles", ctypes.c_void_p), ("x", ctypes.c_void_p),
                ("add", ctypes.c_void_p), ("y", ctypes.c_void_p)]


class CacheDesc(ctypes.Structure):
    _fields_ = [("pages", ctypes.c_void_p), ("scales", ctypes.c_void_p), ("open", ctypes.c_void_p),
                ("open_scales", ctypes.c_void_p), ("faults", ctypes.c_void_p), ("page_count", ctypes.c_uint32),
                ("slot_count", ctypes.c_uint32), ("kv_heads", ctypes.c_uint32), ("head_dim", ctypes.c_uint32),
                ("device", ctypes.c_int32), ("reserved", ctypes.c_uint32)]


class BatchDesc(ctypes.Structure):
    _fields_ = [("past", ctypes.c_void_p), ("cu_tokens", ctypes.c_void_p), ("table", ctypes.c_void_p),
                ("slots", ctypes.c_void_p), ("sequences", ctypes.c_uint32), ("tokens", ctypes.c_uint32),
                ("max_tokens", ctypes.c_uint32), ("table_width", ctypes.c_uint32)]


class Rows(ctypes.Structure):
    _fields_ = [("data", ctypes.c_void_p), ("token_stride", ctypes.c_int64), ("head_stride", ctypes.c_int64)]


class AppendDesc(ctypes.Structure):
    _fields_ = [("dtype", ctypes.c_uint32), ("q_heads", ctypes.c_uint32), ("k", Rows), ("v", Rows), ("q", Rows),
                ("q_out", Rows), ("cos", ctypes.c_void_p), ("sin", ctypes.c_void_p), ("positions", ctypes.c_uint32),
                ("rotary", ctypes.c_uint32), ("interleaved", ctypes.c_uint32), ("eps", ctypes.c_float),
                ("q_norm", ctypes.c_void_p), ("k_norm", ctypes.c_void_p)]


class AttendDesc(ctypes.Structure):
    _fields_ = [("dtype", ctypes.c_uint32), ("q_heads", ctypes.c_uint32), ("q", Rows), ("out", Rows),
                ("lse", ctypes.c_void_p), ("scale", ctypes.c_float), ("window", ctypes.c_uint32)]


class AddNormDesc(ctypes.Structure):
    _fields_ = [("dtype", ctypes.c_uint32), ("rows", ctypes.c_uint32), ("width", ctypes.c_uint32),
                ("scale", ctypes.c_float), ("eps", ctypes.c_float), ("reserved", ctypes.c_uint32),
                ("residual", ctypes.c_void_p), ("y", ctypes.c_void_p), ("gate", ctypes.c_void_p),
                ("h", ctypes.c_void_p), ("n", ctypes.c_void_p), ("residual_stride", ctypes.c_int64),
                ("y_stride", ctypes.c_int64), ("gate_stride", ctypes.c_int64), ("h_stride", ctypes.c_int64),
                ("n_stride", ctypes.c_int64), ("post_weight", ctypes.c_void_p), ("weight", ctypes.c_void_p)]


# The same structures as packers: one call fills a descriptor, where setting
# each field of a ctypes structure takes longer than the kernel's launch.
ROWS = struct.Struct("@Pqq")
APPEND = struct.Struct("@2I Pqq Pqq Pqq Pqq 2P 3If 2P")
ATTEND = struct.Struct("@2I Pqq Pqq P f I")
ADD_NORM = struct.Struct("@3I2fI 5P 5q 2P")

_lib = None


def load() -> ctypes.CDLL:
    """Load the library, declaring every prototype."""
    global _lib
    if _lib is not None:
        return _lib
    if not os.path.exists(LIB_PATH):
        raise RuntimeError(f"{LIB_PATH} is missing: build it with `make -C rdna-gfx1201-v0.1_amd` "
                           "(or __graft_entry__.build())")
    L = ctypes.CDLL(LIB_PATH)
    vp, u32, i32, i64, u64 = ctypes.c_void_p, ctypes.c_uint32, ctypes.c_int, ctypes.c_int64, ctypes.c_uint64
    WP = ctypes.POINTER(Weight)
    proto = {
        "q4rdna_abi_version": (i32, []),
        "q4rdna_last_error": (ctypes.c_char_p, []),
        "q4rdna_sidecar_inspect": (i32, [vp, u64, u64, ctypes.POINTER(u32)]),
        "q4rdna_sidecar_open": (i32, [ctypes.c_char_p, i32, ctypes.POINTER(vp)]),
        "q4rdna_sidecar_open_memory": (i32, [vp, u64, i32, ctypes.POINTER(vp)]),
        "q4rdna_sidecar_close": (None, [vp]),
        "q4rdna_sidecar_count": (u32, [vp]),
        "q4rdna_sidecar_entry": (i32, [vp, u32, ctypes.c_char_p, ctypes.POINTER(u32), ctypes.POINTER(u32),
                                       ctypes.POINTER(u64), ctypes.POINTER(u64)]),
        "q4rdna_find": (i32, [vp, ctypes.c_char_p, i64, i64, WP]),
        "q4rdna_weight_from_device": (i32, [vp, u32, u32, i32, WP]),
        "q4rdna_default_sidecar": (vp, [i32]),
        "q4rdna_scope_allows": (i32, [ctypes.c_char_p, ctypes.c_char_p]),
        "q4rdna_mul_mat": (i32, [WP, vp, i64, vp, i64, vp]),
        "q4rdna_mul_mat_add": (i32, [WP, vp, i64, vp, i64, vp, i64, vp]),
        "q4rdna_mul_mat_glu": (i32, [WP, WP, vp, i64, i32, vp, i64, vp]),
        "q4rdna_mul_mat_ex": (i32, [WP, WP, vp, vp, vp, ctypes.POINTER(LaunchOptions), vp]),
        "q4rdna_mul_mat_batch": (i32, [WP, WP, vp, u32, vp, vp, ctypes.POINTER(LaunchOptions), vp]),
        "q4rdna_policy_split_k": (u32, [u32, u32, i32]),
        "q4rdna_mul_mat_ex_noalloc": (i32, [WP, WP, vp, vp, vp, ctypes.POINTER(LaunchOptions), vp]),
        "q4rdna_mul_mat_group": (i32, [ctypes.POINTER(GroupDesc), u32, vp, i64, ctypes.POINTER(LaunchOptions), vp]),
        "q4rdna_plan_create": (i32, [ctypes.POINTER(GemvDesc), u32, i32, ctypes.POINTER(vp)]),
        "q4rdna_plan_create_batch": (i32, [ctypes.POINTER(GemvDesc), u32, u32, i32, ctypes.POINTER(vp)]),
        "q4rdna_plan_launch": (i32, [vp, vp]),
        "q4rdna_plan_prepare": (i32, [vp, vp]),
        "q4rdna_plan_sweep": (i32, [vp, vp]),
        "q4rdna_plan_destroy": (None, [vp]),
        "q4rdna_plan_workgroups": (u32, [vp]),
        "q4rdna_pack": (i32, [vp, u32, u32, i32, vp, vp]),
        "q4rdna_dequantize": (i32, [WP, vp, vp]),
        "q4rdna_launch_count": (u64, []),
        "q4rdna_sidecar_hits": (u64, [vp, u32]),
        "q4rdna_report_stats": (None, []),
        "q4rdna_kv_append": (i32, [vp, vp, vp, vp]),
        "q4rdna_kv_attend": (i32, [vp, vp, vp, vp]),
        "q4rdna_kv_read": (i32, [vp, vp, u32, vp, vp, vp]),
        "q4rdna_add_norm": (i32, [vp, vp]),
    }
    for name, (res, args) in proto.items():
        fn = getattr(L, name)
        fn.restype = res
        fn.argtypes = args
    _lib = L
    return L


def last_error() -> str:
    msg = load().q4rdna_last_error()
    return msg.decode() if msg else ""


def check(code: int) -> bool:
    """True for OK, False for NOT_APPLICABLE, raise on an error status."""
    if code == OK:
        return True
    if code == NOT_APPLICABLE:
        return False
    raise Q4RdnaError(code, last_error())
