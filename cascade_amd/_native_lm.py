"""ctypes bindings of the C ABI declared in include/cascade_lm.h.

There is no CPU fallback: if the HIP library has not been built, loading fails with an error that says so.
"""
import ctypes as C
import os

from ._native import CSA_OK, CascadeError

HERE = os.path.dirname(os.path.abspath(__file__))
LM_LIB_PATH = os.path.join(HERE, "libcascade_lm.so")

CSA_LM_BF16, CSA_LM_F16, CSA_LM_F32 = range(3)
CSA_LM_BACKWARD, CSA_LM_COPY_ROWS = 1, 2

# every symbol include/cascade_lm.h declares
EXPORTS = (
    "csa_lm_spans_workspace", "csa_lm_spans_u16_dev", "csa_lm_attention_forward_dev", "csa_lm_attention_workspace",
    "csa_lm_attention_backward_dev", "csa_lm_cross_entropy_workspace", "csa_lm_cross_entropy_forward_dev",
    "csa_lm_cross_entropy_backward_dev", "csa_lm_clip_workspace", "csa_lm_clip_dev", "csa_lm_last_error",
)


class CsaLmHeads(C.Structure):
    _fields_ = [("data", C.c_void_p), ("token_stride", C.c_int64), ("head_stride", C.c_int64)]


class CsaLmAttention(C.Structure):
    _fields_ = [
        ("type", C.c_int32), ("q_heads", C.c_uint32), ("kv_heads", C.c_uint32), ("head_dim", C.c_uint32), ("tokens", C.c_uint64),
        ("d_lo", C.c_void_p), ("d_hi", C.c_void_p), ("d_slope", C.c_void_p), ("scale", C.c_float), ("cap", C.c_float),
        ("q", CsaLmHeads), ("k", CsaLmHeads), ("v", CsaLmHeads),
    ]


class CsaLmValues(C.Structure):
    _fields_ = [("inp", C.c_void_p), ("out", C.c_void_p), ("n", C.c_uint64), ("type", C.c_int32)]


_lib = None


def load():
    """Loads libcascade_lm.so and declares its prototypes. Raises if the library is missing."""
    global _lib
    if _lib is not None:
        return _lib
    if not os.path.exists(LM_LIB_PATH):
        raise ImportError(f"{LM_LIB_PATH} is missing: build it with `python -m cascade_amd.build` (there is no CPU fallback)")
    lib = C.CDLL(LM_LIB_PATH)
    vp, u64, u32, i32, i64, f32 = C.c_void_p, C.c_uint64, C.c_uint32, C.c_int, C.c_int64, C.c_float
    lib.csa_lm_spans_workspace.restype = u64
    lib.csa_lm_spans_workspace.argtypes = [u64]
    lib.csa_lm_spans_u16_dev.restype = i32
    lib.csa_lm_spans_u16_dev.argtypes = [vp, u64, u32, vp, vp, vp, vp, u64, vp]
    lib.csa_lm_attention_forward_dev.restype = i32
    lib.csa_lm_attention_forward_dev.argtypes = [C.POINTER(CsaLmAttention), CsaLmHeads, vp, vp, u64, vp]
    lib.csa_lm_attention_workspace.restype = u64
    lib.csa_lm_attention_workspace.argtypes = [u64, u32, u32, u32, u32]
    lib.csa_lm_attention_backward_dev.restype = i32
    lib.csa_lm_attention_backward_dev.argtypes = [C.POINTER(CsaLmAttention), CsaLmHeads, vp, CsaLmHeads, CsaLmHeads, CsaLmHeads, CsaLmHeads, vp, u64, vp]
    lib.csa_lm_cross_entropy_workspace.restype = u64
    lib.csa_lm_cross_entropy_workspace.argtypes = [u64, u64, u64, u32]
    lib.csa_lm_cross_entropy_forward_dev.restype = i32
    lib.csa_lm_cross_entropy_forward_dev.argtypes = [i32, vp, i64, vp, i64, vp, u64, u64, u64, vp, vp, vp, u64, vp]
    lib.csa_lm_cross_entropy_backward_dev.restype = i32
    lib.csa_lm_cross_entropy_backward_dev.argtypes = [i32, vp, i64, vp, i64, vp, vp, vp, u64, u64, u64, vp, i64, vp, i64, vp, u64, vp]
    lib.csa_lm_clip_workspace.restype = u64
    lib.csa_lm_clip_workspace.argtypes = [u32]
    lib.csa_lm_clip_dev.restype = i32
    lib.csa_lm_clip_dev.argtypes = [vp, u32, f32, vp, vp, u64, vp]
    lib.csa_lm_last_error.restype = C.c_char_p
    lib.csa_lm_last_error.argtypes = []
    _lib = lib
    return lib


def check(status):
    if status != CSA_OK:
        raise CascadeError(status, load().csa_lm_last_error().decode())
