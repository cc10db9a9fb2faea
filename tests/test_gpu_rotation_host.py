"""Runs the host layer's tests of caches held in 4 bits, scaled rotations and prompt attention
(tests/cpp/host_rotation_tests.cc) on the device."""
import os
import subprocess

import pytest

BIN = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "chibillm_amd", "bin")


@pytest.mark.gpu
def test_host_rotations_gpu():
    path = os.path.join(BIN, "host_rotation_tests")
    if not os.path.exists(path):
        pytest.fail(f"{path} is not built: run __graft_entry__.build()")
    proc = subprocess.run([path], capture_output=True, text=True, timeout=100)
    print(proc.stdout[-4000:])
    assert proc.returncode == 0, proc.stdout[-4000:] + proc.stderr[-2000:]
    assert " 0 failed checks" in proc.stdout
