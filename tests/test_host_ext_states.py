"""Which states the C++ wrappers of the linear attention take together (tests/host/ext_state_tests.cc; no GPU)."""
import os
import subprocess

HOST = os.path.join(os.path.dirname(os.path.abspath(__file__)), "host")


def test_states_of_a_batch():
    exe = os.path.join(HOST, "ext_state_tests")
    if not os.path.exists(exe):
        subprocess.run(["make", "-s", "-C", HOST, "ext_state_tests"], check=True)
    r = subprocess.run([exe], capture_output=True, text=True, timeout=120)
    assert r.returncode == 0, r.stdout + r.stderr
