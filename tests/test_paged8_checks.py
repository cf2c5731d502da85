"""Pages of 8 bits and chosen blocks without a GPU: structure layouts, view builders, the refusals of the
built library with its launchers (tests/host/paged8_check.cpp, whose stand-ins for the HIP calls
count the launches and look at their grids), and the references that the GPU tests go by against plain ones."""
import ctypes
import math
import os
import subprocess
import tempfile

import numpy as np
import pytest

import paged8_util as p8
from conftest import ROOT, load_package
from paged8_util import Batch8
from paged_util import Batch
from paged_util import reference as all_rows

vxfa = load_package().vxfa
views = load_package().views


def test_struct_layouts_match_the_header():
    assert ctypes.sizeof(vxfa.VxfaBlocks) == 24 and vxfa.VxfaBlocks.block.offset == 8 and vxfa.VxfaBlocks.n_recent.offset == 20
    assert vxfa.I8 == 24


def test_views():
    assert views.kv_pages(7, 64, 8, 128, 1) == ((128, 64, 8, 7), (1, 1024, 128, 65536))
    assert views.scale_pages(7, 64, 8) == ((4, 8, 7, 1), (4, 16, 128, 896))
    assert views.scale_pages(7, 64, 8, 32) == ((2, 8, 7, 1), (4, 8, 64, 448))
    assert views.bound_pages(7, 64, 8, 128, 32) == ((256, 2, 8, 7), (1, 256, 512, 4096))


@pytest.mark.skipif(not os.path.exists(vxfa.LIB_PATH), reason="libvxfa.so not built")
def test_what_is_refused_launches_nothing():
    with tempfile.TemporaryDirectory() as d:
        exe = os.path.join(d, "paged8_check")
        r = subprocess.run(["g++", "-O1", "-g", "-std=c++17", "-rdynamic", "-D__HIP_PLATFORM_AMD__", "-I/opt/rocm/include",
                            os.path.join(ROOT, "tests", "host", "paged8_check.cpp"), vxfa.LIB_PATH,
                            "-Wl,-rpath," + os.path.dirname(vxfa.LIB_PATH), "-Wl,-rpath-link,/opt/rocm/lib", "-o", exe],
                           capture_output=True, text=True, timeout=300)
        assert r.returncode == 0, r.stderr[-3000:]
        r = subprocess.run([exe], capture_output=True, text=True, timeout=120)
        assert r.returncode == 0 and r.stdout.endswith("ok\n"), (r.stdout + r.stderr)[-3000:]


def test_exponents():
    for x, e in ((0, -64), (127, 0), (np.nextafter(127, 200), 1), (128, 1), (254, 1), (255, 2), (63.5, -1), (1e-30, -64), (1e38, 64), (math.inf, 64)):
        assert p8.exponent(x) == e


def test_the_reference_over_lists_of_all_blocks_is_the_one_over_all_rows():
    c = Batch([(40, 3), (100, 1)], seed=2)
    lists = np.broadcast_to(np.arange(8, dtype=np.int32), (c.T, c.hkv, 8))
    for opt in (dict(), dict(window=20, cap=5.0, bias=4.0)):
        want = all_rows(c, 0.1, **opt)[0]
        assert np.abs(p8.reference(c, 0.1, **opt)[0] - want).max() < 1e-12
        assert np.abs(p8.reference(c, 0.1, lists=lists, **opt)[0] - want).max() < 1e-12
    # one listed twice: as if its rows were there twice
    twice = np.array([[[0, 1, 1]] * c.hkv] * c.T, np.int32)
    got = p8.reference(c, 0.1, lists=twice)[0][3]
    k, v = c.rows(1, 0, c.k)[0], c.rows(1, 0, c.v)[0]
    r = np.r_[0:16, 16:32, 16:32]
    e = np.exp(0.1 * (k[r] @ c.q[3, 0].astype(np.float64)))
    assert np.abs(got[0] - e @ v[r] / e.sum()).max() < 1e-12


def test_appended_values_stay_near():
    """A value is off by at most half a step of its block's scale for its own rounding."""
    c = Batch8([(20, 20)], hd=64, seed=3)
    new = np.random.default_rng(0).standard_normal((20, c.hkv, 64)).astype(np.float32)
    c.k, c.ks = p8.append(c, c.k, c.ks, new)
    for h in range(c.hkv):
        x, _ = c.rows(0, h, c.k)
        step = c.ks[c.table[0, np.arange(20) // 16], h, 0]
        assert (np.abs(x - new[:, h]) <= 0.5 * step[:, None]).all() and (np.abs(new[:, h]).max() <= 127 * step.max())


def test_bounds_hold_every_product():
    """No key of a block has a larger product with a query than the block's score says (queries that 8 bits hold)."""
    c = Batch8([(200, 200)], 4, 2, 64, 32, seed=4)
    b, bs = p8.bounds(c, 32, np.zeros((c.n_pages, 2, 1, 128), np.int8), np.ones((c.n_pages, 2, 1), np.float32))
    q = np.random.default_rng(1).integers(-127, 128, (50, 64)).astype(np.float64)
    for h in range(2):
        k, _ = c.rows(0, h, c.k)
        for i in range(7):
            p = c.table[0, i]
            hi, lo = b[p, h, 0, :64] * np.float64(bs[p, h, 0]), b[p, h, 0, 64:] * np.float64(bs[p, h, 0])
            assert ((q @ k[32 * i:32 * i + 32].T).max(1) <= np.where(q > 0, q * hi, q * lo).sum(1) + 1e-9).all()
