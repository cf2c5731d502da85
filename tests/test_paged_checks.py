"""The paged entry points without a GPU: structure layouts, the checks of
arguments (tests/host/paged_check.cpp, linked with
voxtral.cpp_amd/csrc/vxfa_paged.cpp, under AddressSanitizer and
UndefinedBehaviorSanitizer on the host side), view builders, and the 64-bit
reference that the GPU tests go by against torch's attention."""
import ctypes
import math
import os
import subprocess
import tempfile

import numpy as np
import pytest

from conftest import ROOT, load_package
from paged_util import Batch, reference, slopes

vxfa = load_package().vxfa
views = load_package().views
HIPCC = "/opt/rocm/bin/hipcc"


def test_struct_layouts_match_the_header():
    assert ctypes.sizeof(vxfa.VxfaPaged) == 48 and vxfa.VxfaPaged.n_streams.offset == 24 and vxfa.VxfaPaged.window.offset == 40
    assert ctypes.sizeof(vxfa.VxfaEvict) == 40 and vxfa.VxfaEvict.budget.offset == 12 and vxfa.VxfaEvict.kept.offset == 24


def test_views():
    ne, nb = views.kv_pages(7, 16, 8, 128)
    assert ne == (128, 16, 8, 7) and nb == (2, 2048, 256, 32768)
    ne, nb = views.weight_pages(7, 16, 8)
    assert ne == (16, 8, 7, 1) and nb == (4, 64, 512, 3584)
    assert views.dst(64, 4, 5) == ((64, 4, 5, 1), (4, 256, 1024, 5120))
    assert views.dst(64, 4, 3, elt=2) == ((64, 4, 3, 1), (2, 128, 512, 1536))


@pytest.mark.skipif(not os.path.exists(HIPCC), reason="hipcc not installed")
def test_arguments_are_checked_and_grids_hold_the_parts():
    with tempfile.TemporaryDirectory() as d:
        exe = os.path.join(d, "paged_check")
        r = subprocess.run([HIPCC, "--offload-arch=gfx950", "-O1", "-g", "-std=c++17",
                            "-Xarch_host", "-fsanitize=address", "-Xarch_host", "-fsanitize=undefined",
                            "-Xarch_host", "-fno-sanitize-recover=all",
                            "-Xclang", "-target-feature", "-Xclang", "-packed-fp32-ops",
                            "-x", "hip", os.path.join(ROOT, "tests", "host", "paged_check.cpp"),
                            os.path.join(ROOT, "voxtral.cpp_amd", "csrc", "vxfa_paged.cpp"), "-o", exe],
                           capture_output=True, text=True, timeout=600)
        assert r.returncode == 0, r.stderr[-3000:]
        r = subprocess.run([exe], capture_output=True, text=True, timeout=300, env=dict(os.environ, ASAN_OPTIONS="detect_leaks=0"))
        assert r.returncode == 0 and r.stdout.endswith("ok\n"), (r.stdout + r.stderr)[-3000:]


def test_slopes():
    # 8 heads, max_bias 8: 2^-1 .. 2^-8; of 12 heads the last four lie between
    assert slopes(8, 8.0) == [2.0 ** -(h + 1) for h in range(8)]
    s = slopes(12, 8.0)
    assert s[:8] == slopes(8, 8.0) and np.allclose(s[8:], [2.0 ** -0.5, 2.0 ** -1.5, 2.0 ** -2.5, 2.0 ** -3.5])
    assert slopes(5, 0.0) == [0.0] * 5


def test_reference_against_torch():
    import torch
    c = Batch([(50, 7), (33, 33), (20, 1)], 6, 2, 64, seed=1)
    out, add, err, _ = reference(c, 0.125)
    for s, (n, t) in enumerate(c.sizes):
        q = torch.from_numpy(c.q[c.q_start[s]:c.q_start[s] + t].astype(np.float64)).permute(1, 0, 2)
        k, v = (torch.from_numpy(np.stack([c.rows(s, h, x)[0] for h in range(2)])).repeat_interleave(3, 0) for x in (c.k, c.v))
        mask = torch.arange(n)[None] <= (n - t + torch.arange(t))[:, None]
        want = torch.nn.functional.scaled_dot_product_attention(q, k, v, attn_mask=mask, scale=0.125).permute(1, 0, 2)
        assert np.abs(out[c.q_start[s]:c.q_start[s] + t] - want.numpy()).max() < 1e-12
        # every token spreads a weight of 1 over the rows
        assert math.isclose(sum(add[s, h].sum() for h in range(2)), 6 * t, rel_tol=1e-12)
    # a cap far above the scores and a window of all rows change little or nothing
    assert np.abs(reference(c, 0.125, window=50)[0] - out).max() == 0
    assert np.abs(reference(c, 0.125, cap=1e4)[0] - out).max() < 1e-6
    # a planted mistake (one row's V) is far outside the bounds
    c.v[c.table[1, 0], 3] *= np.float16(1.5)
    assert (np.abs(reference(c, 0.125)[0] - out) > err).any()
