"""The fused product is built with the kernels that calls reach, and with no others (no GPU)."""
import os

import fused_dispatch as fd

LIB = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "glm53f-afd_amd", "csrc", "libglm53f_kda.so")


def test_every_kernel_that_is_built_is_reached():
    built, reached = fd.built(LIB), fd.reached()
    assert len(built) > 30
    assert built == {k for k in reached if k[0] != "short"}, (sorted(built - reached), sorted(reached - built))
