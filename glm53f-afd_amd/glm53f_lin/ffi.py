"""Raw bindings of include/ext/glm53f_lin.h, one ctypes prototype per declaration. Pointers are device addresses passed
as integers; strides and offsets count elements; `stream` is a hipStream_t handle (0: the default stream). The entry
points live in the same shared library as the KDA kernels.
"""
import ctypes as C

from glm53f_kda import ffi as _kda

i32, i64, f32, ptr = C.c_int32, C.c_int64, C.c_float, C.c_void_p

_SHAPE = [i32, i32, i32, i32]                            # heads, qk_heads, key_dim, value_dim
_ROWS = [ptr, i64, ptr, i64, ptr, i64, ptr, f32]         # q, q_stride, k, k_stride, v, v_stride, log_decay, scale
_STATE = [ptr, ptr, ptr]                                 # state_in, state_out, state_off
_CHAIN = _SHAPE + [i32, ptr] + _ROWS + _STATE + [ptr, i64, ptr]
_ADVANCE = _SHAPE + [i32, i32, ptr, ptr, ptr, i64, i64, ptr, i64, i64, ptr, ptr, ptr, i64, ptr, ptr]
_PREFILL = _SHAPE + [i32, ptr, i32] + _ROWS + _STATE + [ptr, i64, ptr, i64, ptr]

PROTOTYPES = {
    "glm53f_lin_chain_batch": (i32, _CHAIN),
    "glm53f_lin_chain_batch_bf16state": (i32, _CHAIN),
    "glm53f_lin_advance_batch": (i32, _ADVANCE),
    "glm53f_lin_advance_batch_bf16state": (i32, _ADVANCE),
    "glm53f_lin_prefill_workspace_bytes": (i64, [i32, i32, i32, i32, i32]),
    "glm53f_lin_prefill_batch": (i32, _PREFILL),
    "glm53f_lin_prefill_batch_bf16state": (i32, _PREFILL),
}

_bound = False


def lib() -> C.CDLL:
    """The loaded library with these prototypes set. Raises if it has not been built."""
    global _bound
    handle = _kda.lib()
    if not _bound:
        for name, (res, args) in PROTOTYPES.items():
            fn = getattr(handle, name)
            fn.restype = res
            fn.argtypes = args
        _bound = True
    return handle


def __getattr__(name: str):
    if name in PROTOTYPES:
        return getattr(lib(), name)
    raise AttributeError(name)
