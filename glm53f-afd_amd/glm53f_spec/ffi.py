"""Raw bindings of include/ext/glm53f_spec.h, one ctypes prototype per declaration. Pointers are device addresses passed
as integers; strides count elements; `stream` is a hipStream_t handle (0: the default stream). The entry
points live in the same shared library as the KDA kernels.
"""
import ctypes as C

from glm53f_kda import ffi as _kda

i32, i64, ptr = C.c_int32, C.c_int64, C.c_void_p

PROTOTYPES = {
    "glm53f_spec_probs_workspace_bytes": (i64, [i32, i32]),
    "glm53f_spec_probs": (i32, [i32, i32, ptr, i32, i64, ptr, ptr, i64, ptr, i64, ptr]),
    "glm53f_spec_accept_workspace_bytes": (i64, [i32, i32]),
    "glm53f_spec_accept": (i32, [i32, i32, ptr, ptr, ptr, i64, ptr, i64, ptr, ptr, ptr, ptr, i64, ptr]),
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
