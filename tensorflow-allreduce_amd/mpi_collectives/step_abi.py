"""ctypes binding of the C ABI in include/step_abi.h (lib/libstep_hip.so): the
operators of a training step that stand next to the gradient exchange.

As with the ring's data path there is no CPU fallback: a missing library or a
failing entry point raises.
"""
import ctypes
import os

from .ring_abi import RingError

F32, I32, I64, BF16, F16 = 0, 1, 2, 3, 4

_PKG_ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
LIB_PATH = os.path.join(_PKG_ROOT, "lib", "libstep_hip.so")

# Every symbol include/step_abi.h declares.
EXPORTS = (
    "step_abi_version", "step_status_string", "step_last_hip_error",
    "step_embedding_lookup", "step_embedding_piece", "step_embedding_gradient_workspace", "step_embedding_gradient",
    "step_sum_slices_workspace", "step_sum_slices",
    "step_orthogonalize_side", "step_orthogonalize_workspace", "step_orthogonalize", "step_muon",
)


class Matrix(ctypes.Structure):
    """step_matrix: `count` contiguous matrices of rows x cols."""
    _fields_ = [("grad", ctypes.c_void_p), ("momentum", ctypes.c_void_p), ("out", ctypes.c_void_p),
                ("rows", ctypes.c_size_t), ("cols", ctypes.c_size_t), ("count", ctypes.c_size_t),
                ("rate", ctypes.c_float)]


class StepError(RingError):
    def __init__(self, status, where):
        self.status = status
        msg = "%s: %s (status %d" % (where, lib().step_status_string(status).decode(), status)
        if status == 3:
            msg += ", hipError %d" % lib().step_last_hip_error()
        RuntimeError.__init__(self, msg + ")")


_lib = None


def lib():
    """The loaded library; raises if it has not been built."""
    global _lib
    if _lib is None:
        if not os.path.exists(LIB_PATH):
            raise RuntimeError(
                "%s is missing: build it with `python tensorflow-allreduce_amd/build.py` "
                "(the step operators have no CPU fallback)" % LIB_PATH)
        L = ctypes.CDLL(LIB_PATH)
        ci, sz, vp, fl = ctypes.c_int, ctypes.c_size_t, ctypes.c_void_p, ctypes.c_float
        pm, pf = ctypes.POINTER(Matrix), ctypes.POINTER(fl)
        sig = {
            "step_abi_version": (ci, []),
            "step_status_string": (ctypes.c_char_p, [ci]),
            "step_last_hip_error": (ci, []),
            "step_embedding_lookup": (ci, [vp, ci, sz, vp, ci, sz, sz, sz, fl, vp, vp]),
            "step_embedding_piece": (sz, [sz]),
            "step_embedding_gradient_workspace": (sz, [sz, sz, sz]),
            "step_embedding_gradient": (ci, [vp, ci, sz, vp, ci, sz, sz, sz, fl, vp, vp, sz, vp]),
            "step_sum_slices_workspace": (sz, [sz, sz, sz]),
            "step_sum_slices": (ci, [vp, ci, sz, vp, ci, sz, sz, sz, fl, vp, vp, vp, vp, sz, vp]),
            "step_orthogonalize_side": (ci, [pm, sz, ci, ci]),
            "step_orthogonalize_workspace": (sz, [pm, sz, ci]),
            "step_orthogonalize": (ci, [pm, sz, ci, ci, ci, ci, pf, fl, vp, sz, vp]),
            "step_muon": (ci, [pm, sz, ci, ci, ci, pf, fl, fl, ci, fl, vp, sz, vp]),
        }
        for name in EXPORTS:
            fn = getattr(L, name)          # AttributeError if the symbol is missing
            fn.restype, fn.argtypes = sig[name]
        if L.step_abi_version() != 1:
            raise RuntimeError("libstep_hip.so has ABI version %d, expected 1" % L.step_abi_version())
        _lib = L
    return _lib


def check(status, where):
    if status != 0:
        raise StepError(status, where)
