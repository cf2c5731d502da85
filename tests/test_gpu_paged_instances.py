"""Paged attention's kernels by what chooses them: hd 64 chunks of more than 256
workgroups (one group of wavefronts a piece, where smaller calls take two), and
F32 queries with caps, slopes, windows and weights at both head dims."""
import pytest

from paged_util import Batch
from test_gpu_paged import attend

pytestmark = pytest.mark.gpu

# 20 heads, 128 tokens a workgroup: two tiles a stream by the bounds, 320 workgroups
MANY = [(700, 250), (650, 131), (300, 200), (250, 250), (900, 129), (129, 129), (400, 160), (500, 240)]
OPTIONS = [dict(), dict(window=90), dict(bias=8.0), dict(cap=30.0), dict(cap=50.0, bias=8.0, window=200)]


@pytest.fixture(scope="module")
def ctx():
    from gpu_util import vxfa
    c = vxfa.Context(0)
    yield c
    c.close()


@pytest.mark.parametrize("opt", OPTIONS, ids=str)
@pytest.mark.parametrize("q", ["f16", "f32"])
@pytest.mark.parametrize("weights", [None, "on top"])
def test_hd64_chunks_of_many_workgroups(ctx, opt, q, weights):
    attend(ctx, Batch(MANY, 20, 20, 64, page=32, q_type=q, seed=41), dst="f32", weights=weights, **opt)


@pytest.mark.parametrize("opt", [dict(), dict(cap=50.0, bias=8.0, window=200)], ids=str)
def test_hd64_chunks_of_many_workgroups_with_absent_pages(ctx, opt):
    absent = [(0, i) for i in (0, 1, 9, 21)] + [(2, 9)] + [(5, i) for i in range(5)]
    attend(ctx, Batch(MANY, 20, 20, 64, page=32, absent=absent, seed=42), weights="in place", **opt)


@pytest.mark.parametrize("opt", OPTIONS, ids=str)
@pytest.mark.parametrize("hq,hkv,hd", [(8, 2, 128), (5, 1, 128), (6, 2, 64), (8, 1, 64)])
@pytest.mark.parametrize("t", [1, 50])
def test_f32_queries(ctx, opt, hq, hkv, hd, t):
    attend(ctx, Batch([(t, t), (200, t), (431, t)], hq, hkv, hd, q_type="f32", seed=43), **opt)


@pytest.mark.parametrize("opt", OPTIONS, ids=str)
@pytest.mark.parametrize("hq,hkv,hd", [(8, 2, 128), (3, 3, 128), (6, 2, 64)])
@pytest.mark.parametrize("t", [1, 60])
def test_f32_queries_with_weights(ctx, opt, hq, hkv, hd, t):
    attend(ctx, Batch([(t, t), (300, t), (700, t)], hq, hkv, hd, q_type="f32", seed=44), weights="in place", **opt)
