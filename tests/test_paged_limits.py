"""The paged entry points' refusals as the built library gives them, its launchers
included (tests/host/paged_limits_check.cpp, whose stand-ins for the HIP calls
count the launches)."""
import os
import subprocess
import tempfile

import pytest

from conftest import ROOT, load_package

LIB = load_package().vxfa.LIB_PATH


@pytest.mark.skipif(not os.path.exists(LIB), reason="libvxfa.so not built")
def test_what_is_refused_launches_nothing():
    with tempfile.TemporaryDirectory() as d:
        exe = os.path.join(d, "paged_limits_check")
        r = subprocess.run(["g++", "-O1", "-g", "-std=c++17", "-rdynamic", "-D__HIP_PLATFORM_AMD__", "-I/opt/rocm/include",
                            os.path.join(ROOT, "tests", "host", "paged_limits_check.cpp"), LIB,
                            "-Wl,-rpath," + os.path.dirname(LIB), "-Wl,-rpath-link,/opt/rocm/lib", "-o", exe],
                           capture_output=True, text=True, timeout=300)
        assert r.returncode == 0, r.stderr[-3000:]
        r = subprocess.run([exe], capture_output=True, text=True, timeout=120)
        assert r.returncode == 0 and r.stdout.endswith("ok\n"), (r.stdout + r.stderr)[-3000:]
