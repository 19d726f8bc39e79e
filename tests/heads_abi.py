"""ctypes view of the heads' part of the C ABI (include/volume_integration_b200.h)."""
import ctypes
import os

import torch

LIB = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "volume-integration_b200",
                   "volume_integration", "libvi_b200.so")
DTYPE = {torch.float32: 0, torch.float16: 1, torch.bfloat16: 2}


class Matrix(ctypes.Structure):
    _fields_ = [("data", ctypes.c_void_p), ("rows", ctypes.c_int64), ("cols", ctypes.c_int64),
                ("row_stride", ctypes.c_int64), ("col_stride", ctypes.c_int64)]


def matrix(t):
    return ctypes.byref(Matrix(t.data_ptr(), t.shape[0], t.shape[1], t.stride(0), t.stride(1)))


def load():
    lib = ctypes.CDLL(LIB)
    m, vp, i, i64, u64 = ctypes.POINTER(Matrix), ctypes.c_void_p, ctypes.c_int, ctypes.c_int64, ctypes.c_uint64
    lib.vi_last_error.restype = ctypes.c_char_p
    fwd = [i, i, m, m, vp, m, m, m]
    lib.vi_linear_act_forward_scratch_bytes.argtypes = fwd
    lib.vi_linear_act_forward.argtypes = fwd + [vp, u64, vp]
    bwd = [i, i, m, m, m, m, vp, m, m, vp]
    lib.vi_linear_act_backward_scratch_bytes.argtypes = bwd
    lib.vi_linear_act_keeps_dact.argtypes = [i, i, m, m]
    lib.vi_linear_act_backward.argtypes = bwd + [vp, u64, vp]
    lib.vi_linear_ce_forward_scratch_bytes.argtypes = [i, m, m, vp]
    lib.vi_linear_ce_forward.argtypes = [i, m, m, vp, vp, i64, i, vp, vp, vp, u64, vp]
    lib.vi_linear_ce_backward_scratch_bytes.argtypes = [i, m, m, vp, m, m, vp]
    lib.vi_linear_ce_backward.argtypes = [i, m, m, vp, vp, i64, i, vp, vp, m, m, vp, vp, u64, vp]
    for f in ("vi_linear_act_forward", "vi_linear_act_backward", "vi_linear_ce_forward", "vi_linear_ce_backward"):
        getattr(lib, f + "_scratch_bytes").restype = u64
    return lib
