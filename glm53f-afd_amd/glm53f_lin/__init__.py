"""glm53f_lin: ctypes bindings of linear attention with one decay per head (include/ext/glm53f_lin.h). There is no CPU
fallback: using `ffi` without the built HIP library raises.
"""
