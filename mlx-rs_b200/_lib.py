"""ctypes binding of libmoe_b200.so (the C ABI in include/moe_b200.h).

The library is loaded from this package directory. If it is missing it is built
with nvcc (``build.py``); if that is impossible the import of any compute entry point
raises — there is no fallback implementation.
"""
from __future__ import annotations

import ctypes as C
import os
import threading

import torch

_HERE = os.path.dirname(os.path.abspath(__file__))
library_path = os.path.join(_HERE, "libmoe_b200.so")

MOE_OK = 0
MOE_ERR_INVALID = 1
MOE_ERR_UNSUPPORTED = 2
MOE_ERR_CUDA = 3
MOE_ERR_NO_MEMORY = 4
MOE_ERR_TIMEOUT = 5

SCORING_SOFTMAX = 0
SCORING_SOFTMAX_BIAS = 1
SCORING_SIGMOID_BIAS_SELECT = 2


class MlxError(RuntimeError):
    """Error::Mlx("<fn> failed (rc=N)") of crates/mlx-core/src/error.rs, plus the
    library's one-line reason."""

    def __init__(self, fn: str, rc: int, detail: str = ""):
        self.fn, self.rc, self.detail = fn, rc, detail
        msg = f"{fn} failed (rc={rc})"
        if detail:
            msg += f": {detail}"
        super().__init__(msg)


class QWeight(C.Structure):
    _fields_ = [("w", C.c_void_p), ("scales", C.c_void_p), ("biases", C.c_void_p)]


class BlockConfig(C.Structure):
    _fields_ = [(n, C.c_int32) for n in (
        "hidden", "num_experts", "top_k", "moe_inter", "shared_inter", "scoring",
        "norm_topk_prob", "has_shared_gate", "group_size", "bits")]


class BlockWeights(C.Structure):
    _fields_ = [("router", QWeight), ("expert_bias", C.c_void_p), ("gate", QWeight),
                ("up", QWeight), ("down", QWeight), ("shared_gate", QWeight),
                ("shared_up", QWeight), ("shared_down", QWeight),
                ("shared_expert_gate", QWeight)]


DTYPE_BF16, DTYPE_F16, DTYPE_F32 = 0, 1, 2
ACT_SILU, ACT_GELU = 0, 1


class FfnConfig(C.Structure):
    _fields_ = [(n, C.c_int32) for n in ("hidden", "inter", "activation", "group_size", "bits", "dtype")]


class FfnWeights(C.Structure):
    _fields_ = [("gate", QWeight), ("up", QWeight), ("down", QWeight)]


class RopeConfig(C.Structure):
    _fields_ = ([(n, C.c_int32) for n in ("dtype", "dims", "traditional", "inverse")] +
                [(n, C.c_double) for n in ("base", "scale", "mscale")])


_lib = None
_lock = threading.Lock()

# Every symbol include/moe_b200.h declares, with its ctypes signature.
SIGNATURES = {
    "moe_abi_version": (C.c_int, []),
    "moe_ctx_create": (C.c_int, [C.c_int, C.c_void_p, C.POINTER(C.c_void_p)]),
    "moe_ctx_destroy": (None, [C.c_void_p]),
    "moe_ctx_set_stream": (C.c_int, [C.c_void_p, C.c_void_p]),
    "moe_ctx_reserve": (C.c_int, [C.c_void_p, C.POINTER(BlockConfig), C.c_int64]),
    "moe_last_error": (C.c_char_p, [C.c_void_p]),
    "moe_quantized_matmul": (C.c_int, [C.c_void_p, C.c_void_p, C.c_int64, C.c_int64, C.c_void_p,
                                       C.c_void_p, C.c_void_p, C.c_int64, C.c_int, C.c_int,
                                       C.c_int, C.c_void_p]),
    "moe_gather_qmm": (C.c_int, [C.c_void_p, C.c_void_p, C.c_int64, C.c_int64, C.c_int64,
                                 C.c_void_p, C.c_void_p, C.c_void_p, C.c_void_p, C.c_int64,
                                 C.c_int64, C.c_void_p, C.c_int64, C.c_int, C.c_int, C.c_int,
                                 C.c_int, C.c_void_p]),
    "moe_gather_qmm_noalloc": (C.c_int, [C.c_void_p, C.c_void_p, C.c_int64, C.c_int64, C.c_int64,
                                         C.c_void_p, C.c_void_p, C.c_void_p, C.c_void_p, C.c_int64,
                                         C.c_int64, C.c_void_p, C.c_int64, C.c_int, C.c_int, C.c_int,
                                         C.c_int, C.c_void_p]),
    "moe_fast_rms_norm": (C.c_int, [C.c_void_p, C.c_void_p, C.c_void_p, C.c_float, C.c_int64,
                                    C.c_int64, C.c_void_p]),
    "moe_block_forward": (C.c_int, [C.c_void_p, C.POINTER(BlockConfig), C.POINTER(BlockWeights),
                                    C.c_void_p, C.c_int64, C.c_void_p]),
    "moe_layer_ffn_forward": (C.c_int, [C.c_void_p, C.POINTER(BlockConfig), C.POINTER(BlockWeights),
                                        C.c_void_p, C.c_int64, C.c_void_p, C.c_float, C.c_void_p,
                                        C.c_void_p]),
    "moe_gemma4_block_forward": (C.c_int, [C.c_void_p, C.POINTER(BlockConfig), C.POINTER(BlockWeights),
                                           C.c_void_p, C.c_void_p, C.c_void_p, C.c_int64, C.c_void_p,
                                           C.c_void_p, C.c_void_p]),
    "moe_block_profile": (C.c_int, [C.c_void_p, C.POINTER(BlockConfig), C.POINTER(BlockWeights),
                                    C.c_void_p, C.c_int64, C.c_void_p, C.POINTER(C.c_float),
                                    C.POINTER(C.c_int32)]),
    "moe_block_router_logits": (C.c_int, [C.c_void_p, C.POINTER(BlockConfig), C.POINTER(BlockWeights),
                                          C.c_void_p, C.c_int64, C.c_void_p]),
    "moe_block_route": (C.c_int, [C.c_void_p, C.POINTER(BlockConfig), C.POINTER(BlockWeights),
                                  C.c_void_p, C.c_int64, C.c_void_p, C.c_void_p, C.c_void_p,
                                  C.c_void_p]),
    "moe_ctx_status": (C.c_int, [C.c_void_p, C.POINTER(C.c_int32)]),
    "moe_ctx_expire_wait": (C.c_int, [C.c_void_p, C.c_int64]),
    "moe_ep_route": (C.c_int, [C.c_void_p, C.POINTER(BlockConfig), C.POINTER(BlockWeights),
                               C.c_void_p, C.c_int64, C.c_void_p]),
    "moe_ep_experts": (C.c_int, [C.c_void_p, C.POINTER(BlockConfig), C.POINTER(BlockWeights),
                                 C.c_void_p, C.c_int64, C.c_void_p, C.c_int32, C.c_int32,
                                 C.c_void_p]),
    "moe_ep_finish": (C.c_int, [C.c_void_p, C.c_void_p, C.c_int32, C.c_int64, C.c_int64,
                                C.c_void_p, C.c_void_p, C.c_float, C.c_void_p]),
    "moe_ep_experts_bf16": (C.c_int, [C.c_void_p, C.POINTER(BlockConfig), C.POINTER(BlockWeights),
                                      C.c_void_p, C.c_int64, C.c_void_p, C.c_int32, C.c_int32,
                                      C.c_void_p]),
    "moe_ep_finish_bf16": (C.c_int, [C.c_void_p, C.c_void_p, C.c_int32, C.c_int64, C.c_int64,
                                     C.c_void_p, C.c_void_p, C.c_float, C.c_void_p]),
    "moe_quantized_matmul_workspace": (C.c_int, [C.c_int, C.c_int64, C.c_int64, C.c_int64, C.c_int, C.c_int,
                                                 C.c_int, C.POINTER(C.c_size_t)]),
    "moe_quantized_matmul_ex": (C.c_int, [C.c_void_p, C.c_int, C.c_void_p, C.c_int64, C.c_int64, C.c_void_p,
                                          C.c_void_p, C.c_void_p, C.c_int64, C.c_int, C.c_int, C.c_int,
                                          C.c_void_p, C.c_void_p, C.c_size_t]),
    "moe_gated_ffn_workspace": (C.c_int, [C.POINTER(FfnConfig), C.c_int64, C.c_int, C.POINTER(C.c_size_t)]),
    "moe_gated_ffn_forward": (C.c_int, [C.c_void_p, C.POINTER(FfnConfig), C.POINTER(FfnWeights), C.c_void_p,
                                        C.c_int64, C.c_void_p, C.c_void_p, C.c_void_p, C.c_void_p, C.c_void_p,
                                        C.c_size_t]),
    "moe_gated_ffn_backward": (C.c_int, [C.c_void_p, C.POINTER(FfnConfig), C.POINTER(FfnWeights), C.c_void_p,
                                         C.c_void_p, C.c_void_p, C.c_int64, C.c_void_p, C.c_void_p, C.c_void_p,
                                         C.c_void_p, C.c_size_t]),
    "moe_fast_rope": (C.c_int, [C.c_void_p, C.POINTER(RopeConfig), C.c_void_p, C.POINTER(C.c_int64), C.c_int64,
                                C.c_int64, C.c_int64, C.c_int64, C.c_int64, C.c_void_p, C.c_int, C.c_void_p,
                                C.c_void_p, C.POINTER(C.c_int64)]),
}


def library():
    """Load (building first if needed) and return the ctypes handle."""
    global _lib
    if _lib is not None:
        return _lib
    with _lock:
        built = False
        if _lib is None:
            if not os.path.exists(library_path):
                from . import build as _build
                _build.build()
                built = True
            L = C.CDLL(library_path)
            for name, (res, args) in SIGNATURES.items():
                f = getattr(L, name)
                f.restype = res
                f.argtypes = args
            _lib = L
    if built:
        from . import ops
        ops.load_calls()
    return _lib


# Whether torch's current stream is being captured.
_capturing = getattr(torch._C, "_cuda_isCurrentStreamCapturing", lambda: False)


class Context:
    """A moe_ctx on one CUDA device, used by one thread; follows torch's current stream per call."""

    def __init__(self, device: int):
        self.device = device
        self.captured = False  # a graph may hold calls on it, and with them its scratch
        h = C.c_void_p()
        rc = library().moe_ctx_create(device, None, C.byref(h))
        if rc != MOE_OK:
            raise MlxError("moe_ctx_create", rc, f"device {device}")
        self.handle = h

    def bind_stream(self, stream_handle: int):
        library().moe_ctx_set_stream(self.handle, stream_handle)
        if not self.captured and _capturing():
            self.captured = True

    def check(self, fn: str, rc: int):
        if rc != MOE_OK:
            msg = library().moe_last_error(self.handle)
            raise MlxError(fn, rc, msg.decode() if msg else "")

    def close(self):
        if self.handle:
            library().moe_ctx_destroy(self.handle)
            self.handle = None

    def __del__(self):
        try:
            self.close()
        except Exception:
            pass


_kept: list[Context] = []  # contexts of ended threads whose scratch captured graphs may use


class _Contexts(dict):
    """One thread's contexts by device. They end with the thread (freeing the scratch waits for the
    work that uses it), except those that a graph captured there may still use."""

    def __del__(self):
        try:
            _kept.extend(c for c in self.values() if c.captured)
        except Exception:  # the interpreter is going
            pass


class _Thread(threading.local):
    def __init__(self):
        self.contexts = _Contexts()


_thread = _Thread()


def context_for(device_index: int) -> Context:
    """This thread's context of a device: a moe_ctx has one stream at a time and one scratch, so two
    threads may not share it."""
    contexts = _thread.contexts
    ctx = contexts.get(device_index)
    if ctx is None:
        ctx = contexts[device_index] = Context(device_index)
    return ctx
