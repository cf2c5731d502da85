"""Streams that share pages (a common prefix): their outputs, and what accumulated
weights of shared rows hold. In one call that is the old value plus the sum of one
stream, or of some of them, which is left open; in calls one after another, in place,
all sums add up, the same bits every time."""
import itertools
import math

import numpy as np
import pytest

from paged_util import Batch, Device, check_out, reference

pytestmark = pytest.mark.gpu

SIZES = [(100, 0), (90, 0), (81, 0)]
SHARED = 3          # pages of 16 rows that all streams begin with


@pytest.fixture(scope="module")
def ctx():
    from gpu_util import vxfa
    c = vxfa.Context(0)
    yield c
    c.close()


def batch(t, hq, hkv, hd):
    c = Batch([(n, t) for n, _ in SIZES], hq, hkv, hd, seed=51)
    c.table[1:, :SHARED] = c.table[0, :SHARED]
    return c


def wanted(c, streams):
    """Weights after these streams' sums, and the bound of their errors: [page][kv head][row]; and the rows they have."""
    scale = 1 / math.sqrt(c.hd)
    _, add, _, adderr = reference(c, scale)
    want, tol, mine = c.w.astype(np.float64), np.zeros(c.w.shape), np.zeros(c.w.shape, bool)
    for s in streams:
        r = np.arange(c.sizes[s][0])
        p = c.table[s, r // c.page]
        for h in range(c.hkv):
            want[p, h, r % c.page] += add[s, h]
            tol[p, h, r % c.page] += adderr[s, h] + 2.0 ** -23 * np.abs(want[p, h, r % c.page])
            mine[p, h, r % c.page] = True
    return want, tol, mine


@pytest.mark.parametrize("hq,hkv,hd", [(8, 2, 128), (4, 4, 64)])
@pytest.mark.parametrize("t", [1, 40])
def test_one_call(ctx, hq, hkv, hd, t):
    import torch
    c = batch(t, hq, hkv, hd)
    d = Device(c)
    ctx.flash_attn_ext_paged(d.q, d.k, d.v, d.batch, d.dst, 1 / math.sqrt(hd), weights_in=d.w, weights=d.w)
    torch.cuda.synchronize()
    out, _, err, _ = reference(c, 1 / math.sqrt(hd))
    check_out(d.out(), out, err, True)
    d.check_guards()
    got = d.weights()
    # rows of one stream: its sum
    want, tol, mine = wanted(c, range(3))
    shared = np.zeros(c.w.shape, bool)
    shared[c.table[0, :SHARED]] = True
    alone = mine & ~shared
    assert (np.abs(got - want)[alone] <= tol[alone]).all()
    # shared rows: some of the streams' sums, one at least
    ok = np.zeros(c.w.shape, bool)
    for n in (1, 2, 3):
        for some in itertools.combinations(range(3), n):
            want, tol, _ = wanted(c, some)
            ok |= np.abs(got - want) <= tol
    assert ok[shared].all()
    # rows of none: as they were
    assert np.array_equal(got[~mine], c.w[~mine], equal_nan=True)


@pytest.mark.parametrize("hq,hkv,hd", [(8, 2, 128), (4, 4, 64)])
@pytest.mark.parametrize("t", [1, 40])
def test_a_call_for_each_stream(ctx, hq, hkv, hd, t):
    import torch
    c = batch(t, hq, hkv, hd)
    want, tol, _ = wanted(c, range(3))
    bits = None
    for _ in range(3):
        d = Device(c)
        starts = torch.tensor([0, t], dtype=torch.int32, device="cuda")
        for s in range(3):
            q = d.vxfa.desc(d.qt.data_ptr() + s * t * hq * hd * 2, d.q.type, (hd, t, hq, 1), d.q.nb)
            dst = d.vxfa.desc(d.dst.data + s * t * hq * hd * 2, d.dst.type, (hd, hq, t, 1), d.dst.nb)
            b = d.vxfa.paged(d.table.data_ptr() + 4 * c.max_pages * s, d.n_kv.data_ptr() + 4 * s, starts.data_ptr(), 1, c.max_pages, t)
            ctx.flash_attn_ext_paged(q, d.k, d.v, b, dst, 1 / math.sqrt(hd), weights_in=d.w, weights=d.w)
        torch.cuda.synchronize()
        got = d.weights().copy()
        known = ~np.isnan(want)
        assert (np.abs(got - want)[known] <= tol[known]).all()
        out, _, err, _ = reference(c, 1 / math.sqrt(hd))
        check_out(d.out(), out, err, True)
        assert bits is None or np.array_equal(bits.view(np.uint32), got.view(np.uint32))
        bits = got


@pytest.mark.parametrize("hkv,hd", [(2, 128), (4, 64)])
def test_eviction_of_streams_that_share_pages(ctx, hkv, hd):
    """Each stream's choice among the shared rows is its own; the shared pages stay as they were."""
    from test_gpu_paged import evict
    c = Batch([(n, 0) for n, _ in SIZES], 2 * hkv, hkv, hd, seed=52, spare=3 * 3 + 1)
    c.table[1:, :SHARED] = c.table[0, :SHARED]
    evict(ctx, c, 40, 4, 8)
    evict(ctx, c, 40, 0, 0, with_kept=False)
