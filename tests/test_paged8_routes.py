"""Which kernels the calls over pages of 8 bits and over chosen blocks take, by their sizes, without a GPU
(tests/host/paged8_routes.cpp, the built library over stand-ins for the HIP calls)."""
import os
import re
import subprocess

import pytest

from conftest import ROOT, load_package
from paged8_choices import LONG

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


@pytest.mark.parametrize("name", LONG)
def test_long_choices_take_the_search_of_a_team(routes, name):
    """The calls of test_gpu_paged_choice.py run the kernels that they are there for."""
    c, (threads, seg, segs, join) = LONG[name]
    hkv, t = c.get("hkv", 8), max(t for _, t in c["sizes"])
    group = c.get("hq", 8) // hkv
    tile = min(16 // min(1 << (group - 1).bit_length(), 16), t)
    got = routes("choose", hq=c.get("hq", 8), hkv=hkv, hd=c.get("hd", 64), streams=len(c["sizes"]), nq=t, tokens=sum(t for _, t in c["sizes"]),
                 page=4096, block=16, top=c["top"], window=c.get("window", 0), max_pages=-(-max(n for n, _ in c["sizes"]) // 4096),
                 max_nkv=max(n for n, _ in c["sizes"]))
    assert got[0][:2] == ("paged_select_blocks", (str(c.get("hd", 64)), str(threads // 64))) and got[0][3] == threads
    assert got[0][4] == 4 * tile * seg and got[0][2] % (hkv * segs) == 0
    assert seg > 512 and (join > 1 or hkv * got[0][2] >= 128)
    if join:
        assert [x[:2] for x in got[1:]] == [("paged_select_join", (str(join),))]
        assert min(c["top"], seg) * segs > 1024 or join == 1
    else:
        assert len(got) == 1


def test_four_heads_a_workgroup_with_and_without_options(routes):
    """The calls of test_gpu_paged_q8_routes.py run the kernels that they are there for."""
    for (hq, hkv, hd), streams in [((32, 8, 128), 12), ((8, 8, 128), 12), ((8, 4, 64), 24), ((24, 8, 64), 12)]:
        for cap in (0, 30):
            got = routes("attend", hq=hq, hkv=hkv, hd=hd, streams=streams, max_pages=128, cap=cap)
            assert got[0][:2] == ("paged_walk_kernel", (str(hd), "true", "false", "4", "false" if cap else "true", "4"))
    assert heads_of_a_workgroup(routes("attend", hq=64, hkv=64, hd=64, streams=8, max_pages=131)) == 4
