"""CPU: the library behind the C ABI is built by hipcc alone; only the Python package's helper needs torch's headers."""
import os
import subprocess
import sys

import pytest

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "neat_amd", "csrc")


def commands(*args):
    """What make would run, as if nothing were built."""
    r = subprocess.run(["make", "-C", CSRC, "-n", "-B", *args], capture_output=True, text=True)
    return r.returncode, r.stdout


@pytest.mark.parametrize("py", ["python3 -S -E", "/nonexistent/python"])     # no site-packages, so no torch; no Python at all
def test_the_library_needs_no_torch(py):
    for target in ((), ("lib",)):
        rc, out = commands(*target, f"PY={py}")
        assert rc == 0 and "-shared -fPIC -o ../libneat_hip.so" in out and "-c capi.hip" in out
        assert "host.cpp" not in out and "torch_python" not in out
    assert "left out" in commands(f"PY={py}")[1]
    rc, out = commands("CXX=/nonexistent/g++")
    assert rc == 0 and "host.cpp" not in out and "left out" in out


def test_both_are_built_where_torch_is():
    for target in ((), ("lib", "host")):
        rc, out = commands(*target, f"PY={sys.executable}")
        assert rc == 0 and "../libneat_hip.so" in out and "host.cpp" in out and "left out" not in out
