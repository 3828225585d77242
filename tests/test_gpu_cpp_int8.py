"""The INT8 plan and the layer operators from C++ (tests/cpp/int8_gpu_test.cu)."""

import subprocess

import pytest

pytestmark = pytest.mark.gpu


def test_int8_plan_from_cpp(engine):
    import __graft_entry__ as entry

    exe = entry.build_cpp_tests("int8_gpu_test")
    proc = subprocess.run([str(exe)], capture_output=True, text=True, timeout=300)
    assert proc.returncode == 0, proc.stdout + proc.stderr
    assert "all passed" in proc.stdout
