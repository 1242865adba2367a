"""ctypes binding of ``libdsa_b200.so`` (the C ABI declared in ``include/dsa_b200.h``).

There is no fallback: if the library has not been built, or a call is made without a CUDA device,
the import / call raises.
"""
from __future__ import annotations

import ctypes
import os
from ctypes import c_char_p, c_float, c_int32, c_int64, c_size_t, c_void_p

_PKG = os.path.dirname(os.path.abspath(__file__))
LIB_PATH = os.path.join(_PKG, "libdsa_b200.so")

DTYPE_BF16, DTYPE_FP16 = 0, 1
IMPL_AUTO, IMPL_GENERIC, IMPL_TENSOR_CORE = 0, 1, 2



class RopeRows(ctypes.Structure):
    """``dsa_rope_rows`` of the C header."""
    _fields_ = [("x", c_void_p), ("stride_b", c_int64), ("stride_s", c_int64), ("stride_h", c_int64), ("heads", c_int32), ("norm", c_int32),
                ("weight", c_void_p), ("bias", c_void_p), ("params_fp32", c_int32), ("split", c_int32), ("y", c_void_p), ("y_tail", c_void_p),
                ("slots", c_void_p), ("y_slots", c_int64), ("slots_int64", c_int32), ("reserved", c_int32)]


class RopeGrads(ctypes.Structure):
    """``dsa_rope_grads`` of the C header."""
    _fields_ = [("rows", RopeRows), ("dy", c_void_p), ("dy_stride_b", c_int64), ("dy_stride_s", c_int64), ("dy_stride_h", c_int64),
                ("d_weight", c_void_p), ("d_bias", c_void_p)]


# name -> (restype, argtypes); must list every symbol include/dsa_b200.h declares
SIGNATURES = {
    "dsa_init": (c_int32, []),
    "dsa_get_last_error": (c_char_p, []),
    "dsa_kernel_status": (c_int32, [ctypes.POINTER(c_int32)]),
    "dsa_selftest_bounded_wait": (c_int32, [c_int64, c_void_p, c_void_p]),
    "dsa_topk_select": (c_int32, [c_void_p, c_int64, c_int64, c_int64, c_void_p, c_int32, c_void_p, c_void_p, c_void_p]),
    "dsa_topk_select_unordered": (c_int32, [c_void_p, c_int64, c_int64, c_int64, c_void_p, c_int32, c_void_p, c_void_p, c_void_p]),
    "dsa_lightning_indexer_unordered": (c_int32, [c_void_p, c_void_p, c_void_p, c_int32, c_int32, c_int32, c_int32, c_int32, c_int32,
                                                  c_int32, c_void_p, c_void_p, c_int32, c_void_p, c_void_p, c_void_p, c_size_t,
                                                  c_void_p]),
    "dsa_indexer_scores": (c_int32, [c_void_p, c_void_p, c_void_p, c_void_p, c_int32, c_int32, c_int32, c_int32, c_int32,
                                     c_int32, c_int32, c_void_p, c_void_p, c_void_p, c_int32, c_void_p]),
    "dsa_lightning_indexer_workspace_bytes": (c_size_t, [c_int32, c_int32, c_int32]),
    "dsa_lightning_indexer": (c_int32, [c_void_p, c_void_p, c_void_p, c_int32, c_int32, c_int32, c_int32, c_int32, c_int32,
                                        c_int32, c_void_p, c_void_p, c_int32, c_void_p, c_void_p, c_void_p, c_size_t,
                                        c_void_p]),
    "dsa_lightning_indexer_paged": (c_int32, [c_void_p, c_void_p, c_void_p, c_int32, c_int32, c_int32, c_int32, c_int32, c_int32,
                                              c_int32, c_void_p, c_void_p, c_void_p, c_int32, c_int32, c_int32, c_int32, c_void_p,
                                              c_void_p, c_void_p, c_size_t, c_void_p]),
    "dsa_lightning_indexer_noalloc_max_bytes": (c_size_t, []),
    "dsa_lightning_indexer_noalloc": (c_int32, [c_void_p, c_void_p, c_void_p, c_int32, c_int32, c_int32, c_int32, c_int32,
                                                c_int32, c_int32, c_void_p, c_void_p, c_int32, c_void_p, c_void_p, c_void_p,
                                                c_void_p]),
    "dsa_sparse_mla_fwd": (c_int32, [c_void_p, c_void_p, c_void_p, c_void_p, c_void_p, c_int32, c_int32, c_int32, c_int32,
                                     c_int32, c_int32, c_int32, c_float, c_int32, c_int32, c_int32, c_void_p, c_void_p,
                                     c_void_p, c_void_p, c_int32, c_int32, c_int32, c_void_p]),
    "dsa_sparse_mla_fwd_split_tail": (c_int32, [c_void_p, c_void_p, c_void_p, c_void_p, c_void_p, c_int32, c_int32, c_int32, c_int32,
                                                c_int32, c_int32, c_int32, c_float, c_int32, c_int32, c_int32, c_void_p, c_void_p, c_void_p,
                                                c_void_p, c_int32, c_int32, c_int32, c_int32, c_void_p, c_size_t, c_void_p]),
    "dsa_sparse_mla_fwd_two_part": (c_int32, [c_void_p, c_void_p, c_void_p, c_void_p, c_void_p, c_void_p, c_int32, c_int32, c_int32, c_int32,
                                              c_int32, c_int32, c_int32, c_float, c_int32, c_int32, c_int32, c_void_p, c_void_p, c_void_p,
                                              c_void_p, c_int32, c_int32, c_int32, c_void_p, c_size_t, c_void_p]),
    "dsa_sparse_mla_fwd_two_part_q": (c_int32, [c_void_p, c_void_p, c_void_p, c_void_p, c_void_p, c_void_p, c_void_p, c_int32, c_int32, c_int32, c_int32,
                                              c_int32, c_int32, c_int32, c_float, c_int32, c_int32, c_int32, c_void_p, c_void_p, c_void_p,
                                              c_void_p, c_int32, c_int32, c_int32, c_void_p, c_size_t, c_void_p]),
    "dsa_sparse_mla_fwd_splitkv_nsplit": (c_int32, [c_int32, c_int32, c_int32, c_int32]),
    "dsa_sparse_mla_fwd_splitkv_workspace_bytes": (c_size_t, [c_int32, c_int32, c_int32, c_int32, c_int32]),
    "dsa_sparse_mla_fwd_splitkv": (c_int32, [c_void_p, c_void_p, c_void_p, c_void_p, c_void_p, c_int32, c_int32, c_int32, c_int32,
                                             c_int32, c_int32, c_int32, c_float, c_int32, c_int32, c_int32, c_void_p, c_void_p,
                                             c_void_p, c_void_p, c_int32, c_int32, c_int32, c_void_p, c_size_t,
                                             c_void_p]),
    "dsa_sparse_mla_bwd": (c_int32, [c_void_p, c_void_p, c_void_p, c_void_p, c_void_p, c_void_p, c_void_p, c_void_p,
                                     c_int32, c_int32, c_int32, c_int32, c_int32, c_int32, c_int32, c_float, c_int32,
                                     c_int32, c_int32, c_void_p, c_void_p, c_void_p, c_void_p, c_int32, c_int32,
                                     c_void_p]),
    "dsa_block_sparse_logits": (c_int32, [c_void_p, c_void_p, c_void_p, c_void_p, c_void_p, c_void_p, c_void_p, c_int32, c_int32, c_int32,
                                          c_int32, c_int32, c_int32, c_int32, c_int32, c_int32, c_void_p, c_int32, c_int32, c_void_p]),
    "dsa_v4_build_indices": (c_int32, [c_void_p, c_void_p, c_void_p, c_void_p, c_void_p, c_void_p, c_void_p] + [c_int32] * 12 + [c_void_p]),
    "dsa_v4_build_joined_indices": (c_int32, [c_void_p] * 6 + [c_int32] * 14 + [c_void_p]),
    "dsa_v4_attention": (c_int32, [c_void_p] * 7 + [c_int32] * 5 + [c_float, c_int32, c_int32, c_void_p, c_size_t, c_void_p]),
    "dsa_sink_combine": (c_int32, [c_void_p, c_void_p, c_void_p, c_void_p, c_void_p, c_void_p, c_void_p, c_int64, c_int32, c_int32,
                                   c_int32, c_void_p]),
    "dsa_sparse_mla_bwd_tc_workspace_bytes": (c_size_t, [c_int32, c_int32, c_int32, c_int32, c_int32]),
    "dsa_sparse_mla_bwd_tc": (c_int32, [c_void_p, c_void_p, c_void_p, c_void_p, c_void_p, c_void_p, c_void_p, c_void_p,
                                        c_int32, c_int32, c_int32, c_int32, c_int32, c_int32, c_int32, c_float, c_int32,
                                        c_int32, c_int32, c_void_p, c_void_p, c_void_p, c_void_p, c_int32, c_int32,
                                        c_void_p, c_size_t, c_int32, c_void_p]),
    "dsa_norm_rope": (c_int32, [ctypes.POINTER(RopeRows), ctypes.POINTER(RopeRows), c_void_p, c_int32, c_void_p] + [c_int32] * 7
                      + [c_float, c_float, c_int32, c_void_p]),
    "dsa_norm_rope_bwd_workspace_bytes": (c_size_t, [c_int32]),
    "dsa_norm_rope_bwd": (c_int32, [ctypes.POINTER(RopeGrads), ctypes.POINTER(RopeGrads), c_void_p, c_int32, c_void_p] + [c_int32] * 7
                          + [c_float, c_float, c_void_p, c_size_t, c_int32, c_void_p]),
    "dsa_topk_distillation_workspace_bytes": (c_size_t, [c_int64, c_int32, c_int32, c_int32]),
    "dsa_topk_distillation": (c_int32, [c_void_p, c_int32, c_int64, c_void_p, c_int32, c_void_p, c_void_p, c_void_p, c_int64] + [c_int32] * 4
                              + [c_float, c_void_p, c_size_t, c_void_p]),
    "dsa_topk_distillation_bwd": (c_int32, [c_void_p, c_int32, c_int64, c_void_p, c_int32, c_void_p, c_void_p, c_void_p, c_void_p, c_int64]
                                  + [c_int32] * 4 + [c_float, c_void_p]),
    "dsa_sparse_mla_key_weights": (c_int32, [c_void_p] * 5 + [c_int32] * 6 + [c_float, c_int32, c_int32, c_int32, c_void_p]),
    "dsa_lightning_indexer_bwd_workspace_bytes": (c_size_t, [c_int32] * 7),
    "dsa_lightning_indexer_bwd": (c_int32, [c_void_p] * 8 + [c_int32] * 7 + [c_void_p, c_size_t, c_void_p]),
}

_lib = None


def load() -> ctypes.CDLL:
    """Load the library once; raise if it is missing (build it with ``python -m tilelang_ascend_b200.build``)."""
    global _lib
    if _lib is None:
        if not os.path.exists(LIB_PATH):
            raise RuntimeError(
                f"{LIB_PATH} is missing: build it with `python -m tilelang_ascend_b200.build` "
                "(there is no CPU or PyTorch fallback for these kernels)")
        lib = ctypes.CDLL(LIB_PATH)
        for name, (res, args) in SIGNATURES.items():
            fn = getattr(lib, name)
            fn.restype = res
            fn.argtypes = args
        _lib = lib
    return _lib


class DsaError(RuntimeError):
    pass


def check(rc: int) -> None:
    """Raise on a failed call.  With DSA_DEBUG_SYNC=1 in the environment every successful launch is also followed by a
    device synchronisation and a read of the kernels' status word, so that a bounded in-kernel wait that gave up raises
    at the call that caused it (a debugging aid: it serialises host and device)."""
    if rc != 0:
        raise DsaError(load().dsa_get_last_error().decode())
    if os.environ.get("DSA_DEBUG_SYNC") == "1":
        st = kernel_status()
        if st != 0:
            raise DsaError(f"kernel status word = {st}: a bounded in-kernel wait gave up; results of this call are not valid")


def kernel_status() -> int:
    """Synchronise the current device and return (and clear) the kernels' status word."""
    st = c_int32(0)
    check(load().dsa_kernel_status(ctypes.byref(st)))
    return st.value
