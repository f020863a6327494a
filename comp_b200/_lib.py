"""ctypes binding of the C-ABI library `libcompb200.so` (declarations: include/comp_b200.h).

The library is loaded from this package directory only (built in-tree by `comp_b200.build`). There is no fallback:
if it is missing, every compute entry point raises.
"""

import ctypes
import os

HERE = os.path.dirname(os.path.abspath(__file__))
LIB_PATH = os.path.join(HERE, "libcompb200.so")

B2Q_OK = 0
ERRORS = {-1: "EINVAL", -2: "EALIGN", -3: "ECUDA", -4: "ERANGE", -5: "ETIMEOUT"}

P = ctypes.c_void_p
I64 = ctypes.c_int64
INT = ctypes.c_int


class KVCacheDesc(ctypes.Structure):
    """b2q_kv_cache (include/comp_b200.h)."""

    _fields_ = [("kq", P), ("ks", P), ("vq", P), ("vs", P), ("pages", I64), ("heads", ctypes.c_int32),
                ("page", ctypes.c_int32), ("dim", ctypes.c_int32), ("fmt", ctypes.c_int32)]


class AttentionArgs(ctypes.Structure):
    """b2q_attention_args (include/comp_b200.h)."""

    _fields_ = [*[(n, P) for n in ("q", "out", "lse", "table", "lens", "cu_q", "prefix", "starts", "slopes")],
                *[(n, I64) for n in ("q_st", "q_sh", "T", "batch", "table_stride", "table_pages", "max_q", "max_len")],
                *[(n, ctypes.c_int32) for n in ("q_heads", "dtype", "window")],
                ("scale", ctypes.c_float), ("softcap", ctypes.c_float)]


# The argument blocks of the MXFP4 and expert calls, field by field (include/comp_b200.h), as struct.Struct(...).pack makes them.
MX_LINEAR_ARGS = "@4P6q2i"
EXPERTS_ROUTE_ARGS = "@4P4q2i"
EXPERTS_LINEAR_ARGS = "@5P8q3i4x"
EXPERTS_COMBINE_ARGS = "@4P6qi4x"

# name -> (restype, argtypes); every symbol include/comp_b200.h declares
SIGNATURES = {
    "b2q_version": (ctypes.c_char_p, []),
    "b2q_last_error": (INT, [ctypes.c_char_p, ctypes.c_size_t]),
    "b2q_launch_count": (ctypes.c_longlong, []),
    "b2q_quant_q8_0": (INT, [P, I64, P, P, I64, I64, P]),
    "b2q_quant_q8_K": (INT, [P, I64, P, P, P, I64, I64, P]),
    "b2q_gemv_q4_0": (INT, [P, I64, P, P, P, P, P, I64, I64, I64, INT, P]),
    "b2q_gemv_tq2_0": (INT, [P, I64, P, P, P, P, P, I64, I64, I64, INT, P]),
    "b2q_gemv_q8_0": (INT, [P, I64, P, P, P, P, P, I64, I64, I64, INT, P]),
    "b2q_gemv_iq4_nl": (INT, [P, I64, P, P, P, P, P, I64, I64, I64, INT, P]),
    "b2q_gemv_q4_k": (INT, [P, I64, P, P, P, P, P, I64, I64, I64, INT, P]),
    "b2q_quant_gemv": (INT, [INT, P, I64, P, P, I64, P, P, P, I64, I64, I64, P]),
    "b2q_workspace_size": (ctypes.c_size_t, [INT, I64, I64, I64]),
    "b2q_pinned_workspace_size": (ctypes.c_size_t, [INT, I64, I64, I64]),
    "b2q_quant_gemv_pinned": (INT, [INT, P, I64, P, P, I64, P, I64, I64, I64, P, ctypes.c_size_t, P]),
    "b2q_host_device_pointer": (INT, [P, ctypes.POINTER(ctypes.c_void_p)]),
    "b2q_stage_pinned": (INT, [P, I64, P, I64, I64, P]),
    "b2q_split_blocks": (INT, [INT, P, I64, I64, P, I64, P, P]),
    "b2q_noalloc_scratch_bytes": (ctypes.c_size_t, []),
    "b2q_quant_gemv_splitk_noalloc": (INT, [INT, P, I64, P, P, I64, P, I64, I64, I64, INT, P]),
    "b2q_quant_gemv_ws": (INT, [INT, P, I64, P, P, I64, P, P, P, I64, I64, I64, P, ctypes.c_size_t, P]),
    "b2q_gemv_allgather": (INT, [INT, P, I64, P, P, I64, P, P, P, I64, P, P, I64, I64, I64, I64, I64, INT, INT,
                                 ctypes.c_longlong, P]),
    "b2q_kv_write": (INT, [P, INT, P, I64, I64, P, I64, I64, P, I64, P]),
    "b2q_kv_read": (INT, [P, INT, P, P, P, I64, P]),
    "b2q_attention_workspace_size": (ctypes.c_size_t, [P, P]),
    "b2q_attention": (INT, [P, P, P, ctypes.c_size_t, P]),
    "b2q_mx_bytes": (ctypes.c_size_t, [I64, I64, I64]),
    "b2q_mx_quantize": (INT, [INT, P, I64, I64, I64, I64, P, P]),
    "b2q_mx_dequantize": (INT, [P, I64, I64, I64, INT, P, I64, P]),
    "b2q_mx_pack": (INT, [P, P, I64, I64, I64, P, P]),
    "b2q_mx_matmul": (INT, [P, P, I64, I64, I64, INT, P, I64, P]),
    "b2q_mx_linear_workspace_size": (ctypes.c_size_t, [I64, I64, I64]),
    "b2q_mx_linear": (INT, [P, P]),
    "b2q_experts_plan_words": (ctypes.c_size_t, [I64, I64, I64]),
    "b2q_experts_route": (INT, [P, P]),
    "b2q_experts_sort": (INT, [P, I64, I64, I64, P, P]),
    "b2q_experts_linear_workspace_size": (ctypes.c_size_t, [I64, I64, I64, INT, I64, I64]),
    "b2q_experts_linear": (INT, [P, P]),
    "b2q_experts_combine": (INT, [P, P]),
    "b2q_set_tuning": (INT, [INT, INT, INT]),
    "b2q_set_pipeline": (INT, [INT, INT]),
    "b2q_set_warps": (INT, [INT]),
    "b2q_set_cluster": (INT, [INT]),
    "b2q_set_gemm_min_columns": (INT, [INT]),
    "b2q_set_gemm_schedule": (INT, [INT]),
    "b2q_set_splitk": (INT, [INT]),
    "b2q_device_error": (INT, [ctypes.POINTER(ctypes.c_int), INT]),
    "b2q_ipc_get_handle": (INT, [P, P, ctypes.POINTER(ctypes.c_uint64)]),
    "b2q_ipc_open_handle": (INT, [P, ctypes.POINTER(ctypes.c_void_p)]),
    "b2q_ipc_close_handle": (INT, [P]),
    "b2q_probe_dp4a": (INT, [P, P, P, P, I64, P]),
    "b2q_decode_q4_0": (INT, [P, P, I64, P]),
    "b2q_decode_tq2_0": (INT, [P, P, I64, P]),
}


class B2QError(RuntimeError):
    """A C-ABI call returned a nonzero status; `.code` holds it."""

    def __init__(self, code, msg):
        super().__init__(f"{ERRORS.get(code, code)}: {msg}")
        self.code = code


_lib = None


def load():
    """The loaded library (raises FileNotFoundError with the build command if it has not been built)."""
    global _lib
    if _lib is None:
        if not os.path.exists(LIB_PATH):
            raise FileNotFoundError(f"{LIB_PATH} is missing: build it with `python -m comp_b200.build` (needs nvcc)")
        lib = ctypes.CDLL(LIB_PATH)
        for name, (res, args) in SIGNATURES.items():
            fn = getattr(lib, name)
            fn.restype = res
            fn.argtypes = args
        _lib = lib
    return _lib


def last_error():
    buf = ctypes.create_string_buffer(512)
    load().b2q_last_error(buf, len(buf))
    return buf.value.decode(errors="replace")


def call(name, *args):
    """Calls a status-returning entry point; raises ValueError for argument errors, B2QError otherwise."""
    rc = getattr(load(), name)(*args)
    if rc != B2Q_OK:
        msg = last_error()
        if rc in (-1, -2, -4):
            raise ValueError(f"{name}: {msg}")
        raise B2QError(rc, msg)
    return rc


def launch_count():
    return int(load().b2q_launch_count())


def version():
    return load().b2q_version().decode()
