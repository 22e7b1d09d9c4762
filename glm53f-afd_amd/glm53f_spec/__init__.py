"""glm53f_spec: ctypes bindings of the two ends of a speculative round, probabilities of logits and the verification of
drafted tokens (include/ext/glm53f_spec.h). There is no CPU fallback: using `ffi` without the built HIP library raises.
"""
