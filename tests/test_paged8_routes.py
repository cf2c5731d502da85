"""Which kernels the calls over pages of 8 bits and over chosen blocks take, by their sizes, without a GPU
(tests/host/paged8_routes.cpp, the built library over stand-ins for the HIP calls)."""
import os
import re
import subprocess

import pytest

from conftest import ROOT, load_package

LIB = load_package().vxfa.LIB_PATH
pytestmark = pytest.mark.skipif(not os.path.exists(LIB), reason="libvxfa.so not built")


@pytest.fixture(scope="module")
def routes(tmp_path_factory):
    """routes(op, sizes ..): launches as (kernel without its arguments, template's arguments, workgroups, threads, LDS)."""
    exe = str(tmp_path_factory.mktemp("routes") / "paged8_routes")
    r = subprocess.run(["g++", "-O1", "-g", "-std=c++17", "-rdynamic", "-D__HIP_PLATFORM_AMD__", "-I/opt/rocm/include",
                        os.path.join(ROOT, "tests", "host", "paged8_routes.cpp"), LIB, "-Wl,-rpath," + os.path.dirname(LIB),
                        "-Wl,-rpath-link,/opt/rocm/lib", "-o", exe], capture_output=True, text=True, timeout=300)
    assert r.returncode == 0, r.stderr[-3000:]

    def run(op, **sizes):
        r = subprocess.run([exe, op] + [f"{k}={v}" for k, v in sizes.items()], capture_output=True, text=True, timeout=60)
        assert r.returncode == 0, r.stdout + r.stderr
        out = []
        for line in r.stdout.splitlines():
            name, grid, block, lds = line.rsplit("|", 3)
            m = re.match(r"(?:void )?vxfa::(\w+)(?:<(.*?)>)?\(", name)
            out.append((m[1], tuple(x.strip() for x in (m[2] or "").split(",")), int(grid), int(block), int(lds)))
        return out

    return run


def heads_of_a_workgroup(launches):
    name, args = launches[0][:2]
    assert name == "paged_walk_kernel"
    return int(args[5])


@pytest.mark.parametrize("bound", [98304, 131072, 1 << 20])
def test_one_stream_of_128_keeps_a_head_a_workgroup(routes, bound):
    """However far the bound lies above its rows: a head's wavefronts share them, which is faster but for the longest
    streams, and there by a tenth only."""
    assert heads_of_a_workgroup(routes("attend", hq=32, hkv=8, hd=128, max_pages=bound // 64)) == 1
    assert heads_of_a_workgroup(routes("attend", hq=32, hkv=8, hd=64, max_pages=bound // 64)) == 4


def test_many_rows_take_four_heads_a_workgroup(routes):
    for hd in (64, 128):
        assert heads_of_a_workgroup(routes("attend", hq=32, hkv=8, hd=hd, streams=12, max_pages=8192 // 64)) == 4
        assert heads_of_a_workgroup(routes("attend", hq=32, hkv=8, hd=hd, streams=2, max_pages=65536 // 64)) == 4
        assert heads_of_a_workgroup(routes("attend", hq=32, hkv=8, hd=hd, streams=11, max_pages=8192 // 64)) == 1
        assert heads_of_a_workgroup(routes("attend", hq=6, hkv=6, hd=hd, streams=32, max_pages=8192 // 64)) == 1
