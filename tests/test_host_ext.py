"""The C++ host layer over include/ext (glm53f-afd_amd/host/lin.hpp, spec.hpp, Gemm::fused) through its test program,
tests/host/ext_tests.cc: argument checks without a GPU, a speculative round against double arithmetic with one."""
import os
import subprocess

import pytest

HOST = os.path.join(os.path.dirname(os.path.abspath(__file__)), "host")
EXE = os.path.join(HOST, "ext_tests")


def _exe():
    if not os.path.exists(EXE):
        subprocess.run(["make", "-s", "-C", HOST, "ext_tests"], check=True)
    return EXE


def test_ext_argument_checks_without_a_gpu():
    r = subprocess.run([_exe(), "--cpu"], capture_output=True, text=True, timeout=120)
    assert r.returncode == 0, r.stdout + r.stderr


@pytest.mark.gpu
def test_ext_wrappers_run_a_round():
    r = subprocess.run([_exe(), "--gpu"], capture_output=True, text=True, timeout=300)
    print(r.stdout[-3000:])
    assert r.returncode == 0, r.stdout[-3000:] + r.stderr[-3000:]
