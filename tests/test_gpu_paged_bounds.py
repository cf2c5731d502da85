"""Bounds of blocks' keys on the GPU: keys that are no numbers."""
import numpy as np
import pytest

import paged8_util as p8
from paged8_util import Device8
from paged_util import Batch

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def ctx():
    from gpu_util import vxfa
    c = vxfa.Context(0)
    yield c
    c.close()


@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("block", [16, 64])
def test_dims_without_a_number(ctx, hd, block):
    """NaN is passed over, also where all of a block's keys have one in a dim: the dim's bounds are 0, and neither the
    block's scale nor its other dims are touched. A block of one row, whole blocks, all dims."""
    import torch
    c = Batch([(1, 1), (40, 40), (64, 64), (5, 5)], 2, 2, hd, 64, seed=hd)
    dims = {0: [3], 1: [0, 9, hd - 1], 2: [hd // 2], 3: list(range(hd))}
    for s, (n, _) in enumerate(c.sizes):
        c.k[c.table[s, 0], :n, 0][:, dims[s]] = np.nan
    d = Device8(c, block=block)
    ctx.paged_bounds(d.k, None, d.batch, d.b, d.bs, stream=torch.cuda.current_stream().cuda_stream)
    torch.cuda.synchronize()
    got, gots = d.bounds()
    # as if the elements were 0
    for s, (n, _) in enumerate(c.sizes):
        c.k[c.table[s, 0], :n, 0][:, dims[s]] = 0
    want, wants = p8.bounds(c, block, d.b_np, d.bs_np)
    assert np.array_equal(gots, wants), np.argwhere(gots != wants)[0]
    assert np.array_equal(got, want), np.argwhere(got != want)[0]
    d.check_guards()


def test_some_rows_without_a_number(ctx):
    """Rows of NaN among others leave the others' bounds."""
    import torch
    c = Batch([(50, 50)], 2, 2, 64, 64, seed=1)
    p = c.table[0, 0]
    c.k[p, :50] = np.abs(c.k[p, :50]) + np.float16(1)     # (0 is no bound of theirs)
    c.k[p, [0, 7, 16, 48, 49]] = np.nan
    d = Device8(c, block=16)
    ctx.paged_bounds(d.k, None, d.batch, d.b, d.bs, stream=torch.cuda.current_stream().cuda_stream)
    torch.cuda.synchronize()
    got, gots = d.bounds()
    for i in range(3):
        k = c.k[p, 16 * i:16 * i + 16].astype(np.float64)
        k = k[~np.isnan(k[:, 0, 0])]
        for h in range(2):
            e = p8.exponent(np.abs(k[:, h]).max())
            assert gots[p, h, i] == 2.0 ** e
            assert np.array_equal(got[p, h, i], np.concatenate([np.ceil(k[:, h].max(0) / 2.0 ** e), np.floor(k[:, h].min(0) / 2.0 ** e)]))
    assert (got[p, :, 3] == 0).all() and (gots[p, :, 3] == 2.0 ** -64).all()
