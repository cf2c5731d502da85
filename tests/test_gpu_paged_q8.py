"""Pages of 8 bits, bounds of blocks, their choice and attention over chosen blocks on the
GPU against a plain implementation in 64 bits (paged8_util.py, which derives the bounds): appends, bounds
and choices number for number."""
import math

import numpy as np
import pytest

import paged8_util as p8
from paged8_util import Batch8, Device8
from paged_util import Batch, HALF, check_out

pytestmark = pytest.mark.gpu

EDGES = [1, 2, 15, 16, 17, 31, 32, 33, 63, 64, 65, 127, 128, 129, 255, 257]
HEADS = [(8, 2, 128), (4, 4, 128), (16, 1, 128), (6, 2, 128), (5, 1, 128), (32, 1, 128), (7, 7, 64), (12, 3, 64), (8, 1, 64), (40, 2, 64)]


@pytest.fixture(scope="module")
def ctx():
    from gpu_util import vxfa
    c = vxfa.Context(0)
    yield c
    c.close()


def current():
    import torch
    return torch.cuda.current_stream().cuda_stream


def finish():
    import torch
    torch.cuda.synchronize()


def attend(ctx, c, scale=None, window=0, cap=0.0, bias=0.0, dst="f16"):
    scale = 1 / math.sqrt(c.hd) if scale is None else scale
    d = Device8(c, dst, window)
    ctx.flash_attn_ext_paged_q8(d.q, d.k, d.ks, d.v, d.vs, d.batch, d.dst, scale, bias, cap, stream=current())
    finish()
    want, err = p8.reference(c, scale, window, cap, bias)
    check_out(d.out(), want, err, dst == "f16")
    d.check_guards()


# ---- appends -------------------------------------------------------------------------


def store(ctx, c, k_new, v_new, d=None, rope=None, q=None):
    from gpu_util import guarded, vxfa
    d = d or Device8(c)
    w, T = c.hkv * c.hd, len(k_new)
    new = [guarded(np.ascontiguousarray(x, dtype=np.float32)) for x in (k_new, v_new)]
    nd = [vxfa.desc(t.data_ptr(), vxfa.F32, (w, T, 1, 1), (4, 4 * w, 4 * w * T, 4 * w * T)) for t in new]
    kw = {}
    if rope is not None:
        pos = guarded(np.ascontiguousarray(rope[0], dtype=np.int32))
        kw["rope"] = vxfa.rope(pos.data_ptr(), rope[1], 1e6)
        if q is not None:
            qt, qo = guarded(q), guarded(np.zeros(q.shape, np.float16))
            kw["q"] = vxfa.desc(qt.data_ptr(), vxfa.F32, *d.views.decoder_q(T, c.hq, c.hd))
            kw["q_out"] = vxfa.desc(qo.data_ptr(), vxfa.F16, *d.views.decoder_q(T, c.hq, c.hd, 2))
    ctx.paged_append_q8(*nd, d.batch, d.k, d.ks, d.v, d.vs, stream=current(), **kw)
    finish()
    d.check_guards()
    if q is not None:
        d.q_out = qo.cpu().numpy().view(np.float16).reshape(T, c.hq, c.hd)
    return d


def rows_of(rng, c, T, spread=2.0):
    """New rows whose sizes differ by powers of two from token to token, and some of one value or zeros."""
    x = rng.standard_normal((T, c.hkv, c.hd)) * 2.0 ** rng.uniform(-spread, spread, (T, c.hkv, 1))
    x[rng.random((T, c.hkv)) < 0.1] = 0
    return x.astype(np.float32)


def same_stored(c, d, k_new, v_new):
    for name, new in (("k", k_new), ("v", v_new)):
        ints, scales = p8.append(c, getattr(c, name), getattr(c, name + "s"), new)
        assert np.array_equal(d.ints(name), ints), f"{name}: first at {np.argwhere(d.ints(name) != ints)[0]}"
        assert np.array_equal(d.scale(name), scales, equal_nan=True)


@pytest.mark.parametrize("hq,hkv,hd", [(8, 2, 128), (5, 5, 64), (8, 1, 128), (4, 2, 64)])
@pytest.mark.parametrize("layout,page", [("row", 16), ("head", 64), ("row", 128)])
def test_append(ctx, hq, hkv, hd, layout, page):
    sizes = [(n, 1) for n in EDGES] + [(n + t, t) for n, t in ((0, 1), (0, 16), (3, 20), (16, 16), (15, 2), (40, 100), (5, 3))] + [(9, 0), (0, 0)]
    c = Batch8(sizes, hq, hkv, hd, page, layout=layout, seed=hd + page, behind=3)
    rng = np.random.default_rng(page)
    k_new, v_new = rows_of(rng, c, c.T + 3), rows_of(rng, c, c.T + 3)
    same_stored(c, store(ctx, c, k_new, v_new), k_new, v_new)


def test_append_values_at_the_ends(ctx):
    """Just at and past 127 steps, halves (to even), infinities, NaN, tiny and huge values."""
    c = Batch8([(20, 4), (16, 16), (33, 1), (7, 7)], hd=64, seed=3)
    k_new = np.zeros((c.T, c.hkv, c.hd), np.float32)
    k_new[0, :, :4] = [127.0, 0.5, 1.5, -2.5]
    k_new[1, :, 0] = 127.0 * (1 - 2.0 ** -24)
    k_new[2, :, 0] = np.nextafter(np.float32(127), np.float32(200))
    k_new[4, :, :3] = [1.0, np.nan, -1.0]
    k_new[5, 0, :2] = [np.inf, 1.0]
    k_new[5, 1, :2] = [1e38, -1e38]
    k_new[20, :, :2] = [1e-30, -1e-44]
    k_new[21:, :, 0] = 2.0 ** -70
    v_new = -k_new
    same_stored(c, store(ctx, c, k_new, v_new), k_new, v_new)


def test_append_token_by_token(ctx):
    """A stream grows from nothing, a token at a time and in chunks: scales grow, held rows are rounded again, and
    stay within the documented distance of what was stored."""
    rng = np.random.default_rng(0)
    steps = [1] * 20 + [5, 1, 1, 17, 1, 3]
    total = sum(steps)
    c = Batch8([(total, 0), (total, 0)], hkv=2, hd=64, page=32, seed=4)
    full_k, full_v = (rows_of(rng, c, 2 * total).reshape(2, total, c.hkv, c.hd) for _ in "kv")
    n, grew = 0, np.zeros((2, c.hkv, -(-total // 16), 16))
    for t in steps:
        n += t
        c.sizes = [(n, t), (n, t)]
        c.T, c.q_start, c.n_kv = 2 * t, np.array([0, t, 2 * t], np.int32), np.array([n, n], np.int32)
        c.q = np.zeros((2 * t, c.hq, c.hd), np.float16)
        k_new, v_new = (x[:, n - t:n].reshape(2 * t, c.hkv, c.hd) for x in (full_k, full_v))
        d = store(ctx, c, k_new, v_new)
        same_stored(c, d, k_new, v_new)
        old = c.ks
        c.k, c.v, c.ks, c.vs = d.ints("k"), d.ints("v"), d.scale("k"), d.scale("v")
        for s in range(2):
            for i in range(-(-n // 16)):
                p = c.table[s, i * 16 // c.page], slice(None), i * 16 % c.page // 16
                held = np.arange(16) < (n - t) - 16 * i
                grew[s, :, i] += (c.ks[p] > old[p])[:, None] & held[None]
    for s in range(2):
        for h in range(c.hkv):
            x, _ = c.rows(s, h, c.k)
            r = np.arange(total)
            step = c.ks[c.table[s, r // c.page], h, r % c.page // 16]
            far = 0.5 * step * (1 + grew[s, h].reshape(-1)[:total])
            assert (np.abs(x - full_k[s, :, h]) <= far[:, None]).all()


@pytest.mark.parametrize("hd,dims", [(128, 128), (64, 64), (128, 64), (64, 2)])
def test_append_turned(ctx, hd, dims):
    """Keys and queries turned, at far positions too, against 64 bits: an element is off by the roundings of cos and
    sin (1e-6 each) and of three operations in F32, all of |x0| + |x1| of its pair, then by half a step of its type."""
    sizes = [(1, 1), (40, 40), (100, 3), (8000, 17), (30, 0), (64, 16)]
    c = Batch8(sizes, 6, 3, hd, page=32, seed=dims, absent=[(3, 249)], behind=2)
    rng = np.random.default_rng(dims)
    T = c.T + 2
    k_new, v_new = (rng.standard_normal((T, 3, hd)).astype(np.float32) for _ in "kv")
    q = rng.standard_normal((T, 6, hd)).astype(np.float32)
    pos = np.concatenate([np.arange(n - t, n) for n, t in sizes] + [[5, 6]]).astype(np.int32)
    pos[:c.T] += 100000 * (np.arange(c.T) % 3 == 0)      # (positions need not be the rows' numbers)
    d = store(ctx, c, k_new, v_new, rope=(pos, dims), q=q)

    def turned(x):
        y, err = x.astype(np.float64), np.zeros(x.shape)
        a = pos[:, None, None] * 1e6 ** (-2.0 / dims * np.arange(dims // 2))[None, None]
        x0, x1 = y[..., 0:dims:2].copy(), y[..., 1:dims:2].copy()
        y[..., 0:dims:2], y[..., 1:dims:2] = x0 * np.cos(a) - x1 * np.sin(a), x0 * np.sin(a) + x1 * np.cos(a)
        err[..., 0:dims:2] = err[..., 1:dims:2] = (np.abs(x0) + np.abs(x1)) * (1e-6 + 3 * 2.0 ** -24)
        return y, err

    want, err = turned(q)
    assert (np.abs(d.q_out[:c.T] - want[:c.T]) <= err[:c.T] + HALF * np.abs(want[:c.T]) * 1.001 + 2.0 ** -25).all()
    assert (d.q_out[c.T:] == 0).all()
    k_want, k_err = turned(k_new)
    for name, want, err in (("k", k_want, k_err), ("v", v_new.astype(np.float64), np.zeros(v_new.shape))):
        ints, scales = d.ints(name), d.scale(name)
        for s, (n, t) in enumerate(sizes):
            for r in range(n - t, n):
                p = c.table[s, r // 32]
                if not 0 <= p < c.n_pages:
                    continue
                step = scales[p, :, r % 32 // 16].astype(np.float64)[:, None]
                i = c.q_start[s] + r - (n - t)
                assert (np.abs(ints[p, r % 32] * step - want[i]) <= 0.5 * step + err[i]).all()


# ---- attention over all rows -------------------------------------------------------------


@pytest.mark.parametrize("hq,hkv,hd", HEADS)
def test_single_tokens(ctx, hq, hkv, hd):
    attend(ctx, Batch8([(n, 1) for n in EDGES], hq, hkv, hd, seed=hq))


@pytest.mark.parametrize("hq,hkv,hd", HEADS)
def test_few_tokens(ctx, hq, hkv, hd):
    attend(ctx, Batch8([(n + t, t) for n, t in ((0, 1), (0, 2), (0, 3), (16, 2), (31, 3), (100, 1), (255, 3), (700, 2))], hq, hkv, hd, seed=hq + 1))


OPTIONS = [dict(cap=30.0), dict(bias=8.0), dict(cap=50.0, bias=8.0), dict(cap=100.0), dict(window=1), dict(window=31), dict(window=33, cap=20.0),
           dict(window=200, bias=4.0), dict(scale=0.0), dict(scale=-0.2), dict(scale=1.0), dict(scale=0.0, cap=3.0, bias=1.0)]


@pytest.mark.parametrize("opt", OPTIONS, ids=str)
@pytest.mark.parametrize("hq,hkv,hd", [(8, 2, 128), (6, 2, 64)])
@pytest.mark.parametrize("t", [1, 3, 50])
def test_scores(ctx, opt, hq, hkv, hd, t):
    attend(ctx, Batch8([(t, t), (97, t), (300, t), (1000, t)], hq, hkv, hd, seed=t), **opt)


@pytest.fixture(params=[1, 2, 7])
def pieces(request, monkeypatch):
    """A context whose chunk calls cut the longest walk into this many pieces."""
    from gpu_util import vxfa
    monkeypatch.setenv("VXFA_PAGED_PIECES", str(request.param))
    c = vxfa.Context(0)
    yield c
    c.close()


CHUNKS = [(70, 70), (33, 17), (300, 1), (500, 129), (64, 64), (5, 5), (2, 6)]


@pytest.mark.parametrize("hq,hkv,hd", HEADS)
def test_chunks(ctx, hq, hkv, hd):
    attend(ctx, Batch8(CHUNKS, hq, hkv, hd, seed=hq + 2))


@pytest.mark.parametrize("opt", [dict(), dict(cap=30.0, bias=8.0), dict(bias=8.0), dict(cap=90.0), dict(window=70), dict(window=300, cap=20.0)], ids=str)
@pytest.mark.parametrize("hd", [128, 64])
def test_chunks_in_pieces(pieces, opt, hd):
    """Walks of more than 16 steps, whose granules are read 64 at a time, in pieces."""
    attend(pieces, Batch8([(2600, 200), (1500, 40), (17, 17)], 8, 2, hd, page=32, seed=hd), **opt)


@pytest.mark.parametrize("dst", ["f16", "f32"])
@pytest.mark.parametrize("q", ["f16", "f32"])
def test_chunk_types(ctx, dst, q):
    attend(ctx, Batch8([(50, 50), (200, 50), (431, 50)], q_type=q, seed=5), dst=dst)
    for opt in (dict(), dict(bias=2.0), dict(cap=9.0), dict(cap=70.0)):
        attend(ctx, Batch8([(50, 50), (200, 50)], hd=64, q_type=q, seed=5), dst=dst, **opt)


@pytest.mark.parametrize("sizes", [[(1, 1), (77, 1), (500, 1), (3000, 1)], [(50, 50), (777, 40), (1200, 200)]])
@pytest.mark.parametrize("hd", [64, 128])
def test_scales_as_far_apart_as_they_may_be(ctx, hd, sizes):
    """V's scales from 2^-64 to 2^32. (Exponents of two numbers behind the comma: a weight of F32 reaches 2^-126.)"""
    c = Batch8(sizes, hd=hd, spread=50, seed=17)
    ok = (c.vs > 0) & (c.vs < 2.0 ** 60)
    with np.errstate(invalid="ignore", over="ignore"):
        e = np.where(ok, np.log2(np.where(ok, c.vs, 1)), 0)
        c.vs = np.where(ok, 2.0 ** np.rint(-64 + (e + 55) * 96 / 50), c.vs).astype(np.float32)
    attend(ctx, c, dst="f32")


@pytest.mark.parametrize("hd", [64, 128])
def test_chunk_scales_far_apart(ctx, hd):
    attend(ctx, Batch8([(50, 50), (777, 40), (1200, 200)], hd=hd, spread=50, seed=7), dst="f32")
    attend(ctx, Batch8([(50, 50), (777, 40), (1200, 200)], hd=hd, powers=False, seed=8), dst="f32")


@pytest.mark.parametrize("hd", [64, 128])
def test_chunks_of_absent_pages_and_many_tiles(ctx, hd):
    """Absent pages; chunks with more rows behind them than fit a tile; two groups of wavefronts at hd 64 and one."""
    c = Batch8([(100, 30), (0, 40), (300, 100), (5, 9), (700, 33)], 8, 2, hd, seed=9, behind=4,
               absent=[(0, 0), (0, 6), (2, 3), (2, 18), (4, 0), (4, 1), (4, 20), (4, 43)])
    attend(ctx, c)
    attend(ctx, Batch8([(40, 40)], 8, 2, hd, seed=10, absent=[(0, 0), (0, 1), (0, 2)]))
    attend(ctx, Batch8([(400, 100)] * 12, 16, 8, hd, page=64, seed=11), bias=1.0)


FEW_AMONG_CHUNKS = [(3000, 1), (2500, 300), (700, 4), (0, 0), (900, 5), (64, 3), (2048, 1), (33, 33), (2, 6), (600, 2)]


@pytest.mark.parametrize("opt", [dict(), dict(cap=30.0, bias=8.0), dict(window=500)], ids=str)
@pytest.mark.parametrize("hq,hkv,hd", [(8, 2, 128), (5, 1, 128), (32, 1, 128), (7, 7, 64), (40, 2, 64)])
def test_few_tokens_among_chunks(ctx, opt, hq, hkv, hd):
    """Streams of a few tokens beside chunks: either kernel's streams, and nobody else's rows of dst."""
    attend(ctx, Batch8(FEW_AMONG_CHUNKS, hq, hkv, hd, seed=hq, behind=3, absent=[(0, 0), (0, 100), (1, 5)]), **opt)


def test_few_tokens_among_chunks_in_pieces(pieces):
    attend(pieces, Batch8(FEW_AMONG_CHUNKS, 8, 2, 128, seed=3), bias=2.0)


def test_few_tokens_among_chunks_of_many_streams(ctx):
    """More streams than lanes; no chunks at all under a bound that allows them; chunks alone."""
    rng = np.random.default_rng(5)
    sizes = [(int(n), int(t)) for n, t in zip(rng.integers(1, 700, 150), rng.choice([0, 1, 1, 2, 4, 5, 40], 150))]
    attend(ctx, Batch8(sizes, 8, 2, 64, 64, seed=6))
    from gpu_util import vxfa
    for sizes in ([(900, 1), (30, 1), (700, 2), (600, 4)], [(900, 100), (700, 30), (600, 5), (10, 7)]):
        c = Batch8(sizes, 8, 2, 128, seed=7)
        d = Device8(c)
        d.batch = vxfa.paged(d.table.data_ptr(), d.n_kv.data_ptr(), d.q_start.data_ptr(), 4, c.max_pages, 100)
        ctx.flash_attn_ext_paged_q8(d.q, d.k, d.ks, d.v, d.vs, d.batch, d.dst, 0.1, stream=current())
        finish()
        want, err = p8.reference(c, 0.1)
        check_out(d.out(), want, err, True)
        d.check_guards()


@pytest.mark.parametrize("layout", ["row", "head"])
@pytest.mark.parametrize("page", [16, 128, 1024])
def test_chunk_pages_and_strides(ctx, page, layout):
    attend(ctx, Batch8([(n, 40) for n in (40, 45, 100, 333, 1030)], page=page, layout=layout, seed=page))


@pytest.mark.parametrize("page", [16, 32, 64, 128, 1024])
@pytest.mark.parametrize("layout", ["row", "head"])
def test_pages_and_strides(ctx, page, layout):
    attend(ctx, Batch8([(n, 1) for n in (1, 45, 100, 333, 1030)], page=page, layout=layout, seed=page))


@pytest.mark.parametrize("dst", ["f16", "f32"])
@pytest.mark.parametrize("q", ["f16", "f32"])
def test_types(ctx, dst, q):
    attend(ctx, Batch8([(1, 1), (200, 1), (431, 1)], q_type=q, seed=5), dst=dst)


@pytest.mark.parametrize("hd", [64, 128])
def test_scales_far_apart(ctx, hd):
    """Scales of V from 2^-60 up in one stream, scales that are no powers of two."""
    attend(ctx, Batch8([(1, 1), (77, 1), (500, 1), (3000, 1)], hd=hd, spread=50, seed=7), dst="f32")
    attend(ctx, Batch8([(1, 1), (77, 1), (500, 1), (3000, 1)], hd=hd, powers=False, seed=8), dst="f32")


def test_absent_pages_and_empty_streams(ctx):
    attend(ctx, Batch8([(0, 0), (100, 1), (0, 1), (300, 1), (5, 3), (2, 3)], seed=9, behind=4, absent=[(1, 0), (3, 2), (3, 3), (3, 18)]))
    attend(ctx, Batch8([(40, 1)], seed=10, absent=[(0, 0), (0, 1), (0, 2)]))


def test_long_streams(ctx):
    """Parts and their joins; more streams than a wavefront's lanes."""
    attend(ctx, Batch8([(8192, 1), (5000, 1), (300, 1)], seed=11))
    attend(ctx, Batch8([(9000, 1)], hq=4, hkv=1, hd=64, page=64, seed=12))
    attend(ctx, Batch8([(n % 97 + 1, 1) for n in range(150)], hq=4, hkv=2, hd=64, seed=13))


# ---- bounds and the choice ------------------------------------------------------------------


@pytest.mark.parametrize("kind", [Batch, Batch8])
@pytest.mark.parametrize("hkv,hd", [(2, 128), (5, 64), (4, 128)])
@pytest.mark.parametrize("page,block", [(16, 16), (64, 16), (64, 32), (64, 64), (256, 128)])
@pytest.mark.parametrize("layout", ["row", "head"])
def test_bounds(ctx, kind, hkv, hd, page, block, layout):
    sizes = [(1, 1), (16, 1), (17, 1), (100, 100), (130, 3), (64, 64), (65, 2), (300, 290), (20, 0), (0, 0)]
    c = kind(sizes, hkv, hkv, hd, page, layout=layout, seed=block, absent=[(7, 1)])
    if kind is Batch:
        c.k[c.table[4, 100 // page], 100 % page, 0, :3] = [60000, -60000, 6e-8]
    d = Device8(c, block=block)
    ctx.paged_bounds(d.k, d.ks, d.batch, d.b, d.bs, stream=current())
    finish()
    want, wants = p8.bounds(c, block, d.b_np, d.bs_np)
    got, gots = d.bounds()
    assert np.array_equal(gots, wants), np.argwhere(gots != wants)[0]
    assert np.array_equal(got, want), np.argwhere(got != want)[0]
    d.check_guards()


@pytest.mark.parametrize("max_nq", [1, 30])
def test_bounds_of_chunks_longer_than_max_nq(ctx, max_nq):
    """Tokens past max_nq are left out, and the others stay in the rows that q_start gives them, in however many
    streams; the host knows no count of all tokens."""
    from gpu_util import vxfa
    c = Batch8([(100, 90), (70, 10), (130, 64), (40, 1)], 2, 2, 64, 64, seed=max_nq)
    d = Device8(c, block=16)
    batch = vxfa.paged(d.table.data_ptr(), d.n_kv.data_ptr(), d.q_start.data_ptr(), 4, c.max_pages, max_nq)
    ctx.paged_bounds(d.k, d.ks, batch, d.b, d.bs, stream=current())
    finish()
    want, wants = d.b_np.copy(), d.bs_np.copy()
    full, fulls = p8.bounds(c, 16, d.b_np, d.bs_np)
    for s, (n, t) in enumerate(c.sizes):
        for i in range((n - t) // 16, (n - t + min(t, max_nq) - 1) // 16 + 1):
            page, b = c.table[s, i // 4], i % 4
            want[page, :, b], wants[page, :, b] = full[page, :, b], fulls[page, :, b]
    got, gots = d.bounds()
    assert np.array_equal(got, want) and np.array_equal(gots, wants)
    d.check_guards()


def test_bounds_of_all_rows_again(ctx):
    """Chunks as long as the streams, with bounds of the host's far above them."""
    from gpu_util import vxfa
    c = Batch8([(100, 100), (1, 1), (300, 300)], 2, 2, 128, 64, seed=3)
    d = Device8(c, block=32)
    batch = vxfa.paged(d.table.data_ptr(), d.n_kv.data_ptr(), d.q_start.data_ptr(), 3, c.max_pages, 2 ** 31 - 1)
    ctx.paged_bounds(d.k, d.ks, batch, d.b, d.bs, stream=current())
    finish()
    want, wants = p8.bounds(c, 32, d.b_np, d.bs_np)
    got, gots = d.bounds()
    assert np.array_equal(got, want) and np.array_equal(gots, wants)


def test_bounds_of_nan_and_infinite_keys(ctx):
    c = Batch([(20, 20)], 1, 1, 64, 32, seed=1)
    p = c.table[0, 0]
    c.k[p, 3, 0, 0], c.k[p, 4, 0, 1], c.k[p, 5, 0, 2] = np.nan, np.inf, -np.inf
    d = Device8(c, block=32)
    ctx.paged_bounds(d.k, None, d.batch, d.b, d.bs, stream=current())
    finish()
    got, gots = d.bounds()
    # 127 2^64 stands for the infinities; beside it all else is 0, or 1 where it was rounded up or down
    assert gots[p, 0, 0] == 2.0 ** 64 and got[p, 0, 0, 1] == 127 and got[p, 0, 0, 64 + 2] == -127
    assert set(np.delete(got[p, 0, 0, :64], [1])) <= {0, 1} and set(np.delete(got[p, 0, 0, 64:], [2])) <= {0, -1}


def choose(ctx, c, block, top, n_sink=0, n_recent=0, window=0, b=None, seed=0):
    rng = np.random.default_rng(seed)
    d = Device8(c, window=window, block=block)
    n = c.page // block
    if b is None:
        hi = np.clip(np.rint(77 + 13 * rng.standard_normal((c.n_pages, c.hkv, n, c.hd))), -127, 127)
        lo = np.clip(np.rint(-77 + 13 * rng.standard_normal((c.n_pages, c.hkv, n, c.hd))), -127, 127)
        b = np.concatenate([hi, lo], -1).astype(np.int8), 2.0 ** rng.integers(-6, -4, (c.n_pages, c.hkv, n)).astype(np.float32)
    d.set_bounds(*b, block)
    d.set_list(np.full((c.T + c.behind, c.hkv, top), -7, np.int32), block, n_sink, n_recent)
    ctx.paged_select(d.q, d.b, d.bs, d.batch, d.blocks, stream=current())
    finish()
    want = p8.select(c, block, *b, top, n_sink, n_recent, window)
    got = d.list()
    bad = np.argwhere((got[:c.T] != want).any(-1))
    assert len(bad) == 0, f"{len(bad)} lists, first {bad[0]}: {got[tuple(bad[0])]} for {want[tuple(bad[0])]}"
    assert (got[c.T:] == -7).all()
    d.check_guards()


@pytest.mark.parametrize("hq,hkv,hd", HEADS)
@pytest.mark.parametrize("page,block", [(16, 16), (64, 32)])
def test_choice(ctx, hq, hkv, hd, page, block):
    sizes = [(1, 1), (16, 1), (17, 1), (700, 1), (3000, 1), (100, 20), (333, 5), (600, 3), (0, 0)]
    c = Batch(sizes, hq, hkv, hd, page, seed=hq, behind=2)
    choose(ctx, c, block, 8, 1, 2, seed=hd)


@pytest.mark.parametrize("top,n_sink,n_recent", [(1, 0, 0), (1, 1, 0), (1, 0, 1), (5, 2, 3), (40, 0, 1), (64, 1, 2), (300, 4, 4), (1024, 0, 0)])
@pytest.mark.parametrize("window", [0, 1, 100, 1000])
def test_choice_ends_and_windows(ctx, top, n_sink, n_recent, window):
    c = Batch([(5000, 1), (40, 1), (900, 17), (16, 16)], 8, 2, 64, 16, seed=top, absent=[(0, 5), (0, 300), (2, 0), (2, 56)])
    choose(ctx, c, 16, top, n_sink, n_recent, window, seed=window)


def test_choice_of_equal_scores(ctx):
    """Few distinct bounds: ties go to the first; all alike; F32 queries; queries of zeros."""
    for values in ([3, 4], [5]):
        c = Batch([(2000, 1), (300, 9)], 4, 2, 64, 16, q_type="f32", seed=len(values))
        c.q[3] = 0
        rng = np.random.default_rng(2)
        b = rng.choice(values, (c.n_pages, c.hkv, 1, 1)).astype(np.int8) * np.ones((1, 1, 1, 2 * c.hd), np.int8)
        choose(ctx, c, 16, 20, 1, 1, b=(b, np.full((c.n_pages, c.hkv, 1), 0.5, np.float32)))


@pytest.mark.parametrize("q_type", ["f16", "f32"])
def test_choice_by_queries_of_all_sizes(ctx, q_type):
    """Queries of zeros, of the least f16 numbers, of the largest, one head far above the others; F32 ones are rounded to f16."""
    c = Batch8([(500, 6), (300, 1), (900, 20)], 8, 2, 128, 32, q_type=q_type, seed=3)
    rng = np.random.default_rng(4)
    c.q[0] = 0
    c.q[1] = rng.choice([-1, 0, 1], c.q[1].shape) * 2.0 ** -24
    c.q[2] = rng.choice([-65504, 65504], c.q[2].shape)
    c.q[3, 0] *= 1000
    c.q[4, :, 1:] = 0
    c.q[6] *= 2.0 ** -13
    choose(ctx, c, 16, 5, 1, 1)


def test_choice_of_many_blocks(ctx):
    """Streams of more blocks than a segment, scores of either sign."""
    rng = np.random.default_rng(5)
    for hq, hkv, t in ((4, 1, 1), (2, 2, 3), (1, 1, 20)):
        c = Batch([(80000, t), (300, t), (16 * 4096, 1), (16 * 4096 + 1, 1)], hq, hkv, 64, 16, seed=t)
        b = rng.integers(-127, 128, (c.n_pages, c.hkv, 1, 2 * c.hd)).astype(np.int8)
        choose(ctx, c, 16, 33, 1, 2, b=(b, 2.0 ** rng.integers(-3, 3, (c.n_pages, c.hkv, 1)).astype(np.float32)))


# ---- attention over chosen blocks ----------------------------------------------------------------


def some_blocks(c, block, top, rng, wild=False):
    """Lists of distinct blocks that a token sees, the last among them, in any order; wild: others and doubles, too."""
    out = np.full((c.T, c.hkv, top), -1, np.int32)
    for s, (n, t) in enumerate(c.sizes):
        for i in range(t):
            last = (n - t + i) // block
            for h in range(c.hkv):
                if last < 0:
                    continue
                x = rng.permutation(last + 1)[:top]
                x[rng.integers(len(x))] = last
                x = np.unique(x)
                rng.shuffle(x)
                out[c.q_start[s] + i, h, :len(x)] = x
    if wild:
        m = rng.random(out.shape)
        out = np.where(m < 0.1, rng.choice([-1, -5, 10 ** 6, 2 ** 31 - 1, -2 ** 31], out.shape), out)
        out = np.where((m > 0.9) & (out[..., :1] >= 0), out[..., :1], out).astype(np.int32)
    return out


def attend_blocks(ctx, c, block, top, window=0, cap=0.0, bias=0.0, dst="f16", scale=None, wild=False, seed=0, lists=None):
    scale = 1 / math.sqrt(c.hd) if scale is None else scale
    if lists is None:
        lists = some_blocks(c, block, top, np.random.default_rng(seed), wild)
    d = Device8(c, dst, window, block)
    d.set_list(lists, block)
    ctx.flash_attn_ext_paged_blocks(d.q, d.k, d.ks, d.v, d.vs, d.batch, d.blocks, d.dst, scale, bias, cap, stream=current())
    finish()
    seen = np.where(lists * np.int64(block) < 2 ** 20, lists, -1)
    want, err = p8.reference(c, scale, window, cap, bias, seen, block)
    check_out(d.out(), want, err, dst == "f16")
    d.check_guards()


@pytest.mark.parametrize("kind", [Batch, Batch8])
@pytest.mark.parametrize("hq,hkv,hd", HEADS)
def test_blocks(ctx, kind, hq, hkv, hd):
    c = kind([(n, 1) for n in EDGES] + [(900, 7), (3, 3), (0, 0), (2000, 2)], hq, hkv, hd, 64, seed=hq, behind=3)
    attend_blocks(ctx, c, 32, 6)


@pytest.mark.parametrize("kind", [Batch, Batch8])
@pytest.mark.parametrize("opt", OPTIONS, ids=str)
def test_blocks_scores(ctx, kind, opt):
    c = kind([(1, 1), (300, 1), (1000, 5)], 6, 2, 128, 32, seed=3)
    attend_blocks(ctx, c, 16, 20, **opt)
    attend_blocks(ctx, kind([(1, 1), (300, 1), (1000, 5)], 6, 2, 64, 32, seed=3), 32, 9, **opt)


@pytest.mark.parametrize("kind", [Batch, Batch8])
@pytest.mark.parametrize("page,block,layout", [(16, 16, "row"), (64, 16, "head"), (128, 128, "row"), (1024, 64, "head"), (1024, 1024, "row")])
def test_blocks_pages(ctx, kind, page, block, layout):
    attend_blocks(ctx, kind([(1, 1), (45, 1), (333, 3), (2500, 2)], page=page, layout=layout, seed=page), block, 4)


@pytest.mark.parametrize("kind", [Batch, Batch8])
def test_blocks_wild_lists(ctx, kind):
    """Numbers outside the stream, doubles, absent pages, lists without a block, tokens without rows."""
    c = kind([(300, 4), (1000, 1), (50, 1), (3, 5)], 8, 2, 128, 16, seed=5, absent=[(0, 2), (1, 0), (1, 33)])
    attend_blocks(ctx, c, 16, 25, wild=True, dst="f32")
    attend_blocks(ctx, c, 16, 3, lists=np.full((c.T, 2, 3), -1, np.int32))


@pytest.mark.parametrize("kind", [Batch, Batch8])
def test_blocks_long_lists(ctx, kind):
    """A token's list in parts; more of it than a wavefront's lanes hold; many tokens."""
    attend_blocks(ctx, kind([(16384, 1)], 4, 1, 128, 64, seed=6), 64, 200)
    attend_blocks(ctx, kind([(40000, 1), (40, 1)], 2, 1, 64, 16, seed=6), 16, 1024)
    attend_blocks(ctx, kind([(700, 300), (300, 200)], 8, 4, 64, 32, seed=7), 32, 3)
    attend_blocks(ctx, kind([(n % 50 + 1, 1) for n in range(130)], 2, 1, 64, 16, seed=8), 16, 2)


def test_blocks_are_all_rows(ctx):
    """Lists of all blocks give what the call over all rows does, within its bounds."""
    c = Batch8([(500, 1), (77, 1)], seed=9)
    lists = np.broadcast_to(np.arange(32, dtype=np.int32), (2, c.hkv, 32)).copy()
    attend_blocks(ctx, c, 16, 32, lists=lists)


@pytest.mark.parametrize("kind", [Batch, Batch8])
def test_blocks_lists_longer_than_the_lanes(ctx, kind):
    """Whole lists of more than 32 steps a wavefront, whose pages are read 32 steps at a time."""
    attend_blocks(ctx, kind([(6000, 70)], 8, 8, 64, 16, seed=12), 16, 300)


def test_whole_streams_longer_than_the_lanes(ctx):
    """Streams that the workspace's records leave whole (1024 query heads), of more than 32 steps a wavefront."""
    attend(ctx, Batch8([(5000, 1)] + [(3, 1)] * 59, 1024, 64, 64, 16, seed=13))


def test_many_rows_of_neighbouring_heads(ctx):
    """The bounds' rows where a workgroup takes four heads, with short streams and long ones, absent pages, a window."""
    sizes = [(n, 1) for n in (1, 17, 200, 5000, 9000, 33, 64, 1000, 2, 3000, 700, 40)]
    attend(ctx, Batch8(sizes, 8, 8, 64, 16, seed=14, absent=[(3, 0), (4, 100), (4, 562)]))
    attend(ctx, Batch8(sizes, 32, 8, 128, 32, seed=15), window=2500, cap=20.0, bias=4.0)


# ---- memory and streams ----------------------------------------------------------------------


@pytest.mark.parametrize("kind", [Batch, Batch8])
@pytest.mark.parametrize("hd", [128, 64])
def test_pages_past_4_gib(ctx, kind, hd):
    """Pages 2 GiB and more apart: offsets within the pool pass 32 bits."""
    import torch
    from gpu_util import guarded, vxfa
    c = kind([(60, 1), (100, 40)], 4, 2, hd, 64, seed=hd)
    d = Device8(c, block=16)
    far = (2 ** 31 + 4096)
    e = 1 if kind is Batch8 else 2
    page = 64 * 2 * hd * e
    for name in "kv":
        big = torch.empty(far * (c.n_pages - 1) + page, dtype=torch.uint8, device="cuda")
        small = d.pools[name][0].view(c.n_pages, page)
        for i in range(c.n_pages):
            big[far * i:far * i + page] = small[i]
        d.pools[name] = (big, vxfa.desc(big.data_ptr(), vxfa.I8 if e == 1 else vxfa.F16, (hd, 64, 2, c.n_pages), (e, 2 * hd * e, hd * e, far)))
    d.k, d.v = d.pools["k"][1], d.pools["v"][1]
    if e == 1:
        ctx.flash_attn_ext_paged_q8(d.q, d.k, d.ks, d.v, d.vs, d.batch, d.dst, 0.1, stream=current())
        finish()
        want, err = p8.reference(c, 0.1)
        check_out(d.out(), want, err, True)
        d.dt.fill_(0xA5)
    ctx.paged_bounds(d.k, d.ks, d.batch, d.b, d.bs, stream=current())
    finish()
    b, bs = p8.bounds(c, 16, d.b_np, d.bs_np)
    assert np.array_equal(d.bounds()[0], b) and np.array_equal(d.bounds()[1], bs)
    lists = some_blocks(c, 16, 5, np.random.default_rng(1))
    d.set_list(lists, 16)
    ctx.flash_attn_ext_paged_blocks(d.q, d.k, d.ks, d.v, d.vs, d.batch, d.blocks, d.dst, 0.1, stream=current())
    finish()
    want, err = p8.reference(c, 0.1, lists=lists)
    check_out(d.out(), want, err, True)
    if e == 1:
        rng = np.random.default_rng(2)
        new = [rng.standard_normal((c.T, 2, hd)).astype(np.float32) for _ in "kv"]
        t = [guarded(x) for x in new]
        w = 2 * hd
        nd = [vxfa.desc(x.data_ptr(), vxfa.F32, (w, c.T, 1, 1), (4, 4 * w, 4 * w * c.T, 4 * w * c.T)) for x in t]
        ctx.paged_append_q8(*nd, d.batch, d.k, d.ks, d.v, d.vs, stream=current())
        finish()
        for name, x in zip("kv", new):
            ints, scales = p8.append(c, getattr(c, name), getattr(c, name + "s"), x)
            got = np.stack([d.pools[name][0][far * i:far * i + page].cpu().numpy().view(np.int8) for i in range(c.n_pages)])
            assert np.array_equal(got.reshape(ints.shape), ints) and np.array_equal(d.scale(name), scales, equal_nan=True)


@pytest.mark.parametrize("kind", [Batch, Batch8])
def test_a_pool_without_pages(ctx, kind):
    """Zeros, and no choice; nothing of the pool is read."""
    import torch
    c = kind([(60, 1), (100, 40)], 4, 2, 64, 64, seed=1)
    d = Device8(c, block=32)
    lists = some_blocks(c, 32, 3, np.random.default_rng(1))
    d.set_list(lists, 32)
    for t in (d.k, d.v, d.ks, d.vs, d.b, d.bs):
        if t is not None:
            t.ne[2 if t.type == d.vxfa.F32 else 3] = 0
            t.data = None
    ctx.flash_attn_ext_paged_blocks(d.q, d.k, d.ks, d.v, d.vs, d.batch, d.blocks, d.dst, 0.1, stream=current())
    finish()
    assert (d.out() == 0).all()
    if kind is Batch8:
        ctx.flash_attn_ext_paged_q8(d.q, d.k, d.ks, d.v, d.vs, d.batch, d.dst, 0.1, stream=current())
        finish()
        assert (d.out() == 0).all()
    ctx.paged_bounds(d.k, d.ks, d.batch, d.b, d.bs, stream=current())
    ctx.paged_select(d.q, d.b, d.bs, d.batch, d.blocks, stream=current())
    finish()
    assert (d.list() == -1).all()


def test_two_contexts_at_once(ctx):
    """Two streams, a context each, one in a graph and one eager, several times: each as alone."""
    import torch
    from gpu_util import vxfa
    cs = [Batch8([(3000, 1), (700, 1), (90, 1)], 8, 2, 128, 32, seed=s) for s in (1, 2)]
    ds = [Device8(c, block=32) for c in cs]
    streams, ctxs = [torch.cuda.Stream() for _ in cs], [vxfa.Context(0) for _ in cs]
    for d, c in zip(ds, cs):
        d.set_list(np.zeros((3, 2, 9), np.int32), 32, 1, 2)

    def step(i, st):
        d = ds[i]
        ctxs[i].paged_bounds(d.k, d.ks, d.batch, d.b, d.bs, stream=st)
        ctxs[i].paged_select(d.q, d.b, d.bs, d.batch, d.blocks, stream=st)
        ctxs[i].flash_attn_ext_paged_blocks(d.q, d.k, d.ks, d.v, d.vs, d.batch, d.blocks, d.dst, 0.1, stream=st)

    try:
        graph = torch.cuda.CUDAGraph()
        torch.cuda.synchronize()
        with torch.cuda.graph(graph, stream=streams[0]):
            step(0, streams[0].cuda_stream)
        want = []
        for i in range(2):
            step(i, current())
            finish()
            want.append((ds[i].out(), ds[i].list().copy()))
            full, err = p8.reference(cs[i], 0.1, lists=want[i][1], block=32)
            check_out(want[i][0], full, err, True)
        for _ in range(20):
            for d in ds:
                d.dt.fill_(0xA5)
                d.lt.zero_()
            torch.cuda.synchronize()
            with torch.cuda.stream(streams[0]):
                graph.replay()
            for _ in range(3):
                step(1, streams[1].cuda_stream)
            torch.cuda.synchronize()
            for d, w in zip(ds, want):
                assert np.array_equal(d.out(), w[0]) and np.array_equal(d.list(), w[1])
    finally:
        for x in ctxs:
            x.close()


@pytest.mark.parametrize("max_nq", [1, 3, 20])
def test_chunks_longer_than_max_nq(ctx, max_nq):
    """Tokens past max_nq are left out by each call; the others keep their rows."""
    from gpu_util import vxfa
    rng = np.random.default_rng(max_nq)
    sizes = [(90, 40), (33, 33), (200, 1), (64, 5)]
    kept = [(n - t + min(t, max_nq), min(t, max_nq)) for n, t in sizes]
    c = Batch8(sizes, 8, 2, 128, 32, seed=max_nq)
    live = np.concatenate([np.arange(t) < max_nq for _, t in sizes])
    d = Device8(c, block=16)
    d.batch = vxfa.paged(d.table.data_ptr(), d.n_kv.data_ptr(), d.q_start.data_ptr(), 4, c.max_pages, max_nq)
    # attention, over all rows and over lists
    want, err = p8.reference(c, 0.1)
    before = d.out().copy()
    ctx.flash_attn_ext_paged_q8(d.q, d.k, d.ks, d.v, d.vs, d.batch, d.dst, 0.1, stream=current())
    finish()
    check_out(d.out()[:c.T][live], want[live], err[live], True)
    assert np.array_equal(d.out()[:c.T][~live], before[:c.T][~live], equal_nan=True)
    b, bs = p8.bounds(c, 16, d.b_np, d.bs_np)
    d.set_bounds(b, bs, 16)
    d.set_list(np.full((c.T, 2, 3), -7, np.int32), 16, 1, 1)
    ctx.paged_select(d.q, d.b, d.bs, d.batch, d.blocks, stream=current())
    finish()
    lists = p8.select(c, 16, b, bs, 3, 1, 1)
    assert np.array_equal(d.list()[live], lists[live]) and (d.list()[~live] == -7).all()
    want, err = p8.reference(c, 0.1, lists=lists, block=16)
    ctx.flash_attn_ext_paged_blocks(d.q, d.k, d.ks, d.v, d.vs, d.batch, d.blocks, d.dst, 0.1, stream=current())
    finish()
    check_out(d.out()[:c.T][live], want[live], err[live], True)
    assert np.array_equal(d.out()[:c.T][~live], before[:c.T][~live], equal_nan=True)
    # appends
    k_new, v_new = rows_of(rng, c, c.T), rows_of(rng, c, c.T)
    store(ctx, c, k_new, v_new, d)
    c.sizes = kept
    same_stored(c, d, k_new, v_new)


# ---- together -------------------------------------------------------------------------------


@pytest.mark.parametrize("hd", [128, 64])
def test_served_together(ctx, hd):
    """Streams grow by chunks and single tokens: append, bounds, choice, attention over the choice, each step checked
    against what the pools then hold; captured once and replayed for the single tokens."""
    import torch
    from gpu_util import guarded, vxfa
    rng = np.random.default_rng(hd)
    block, top = 32, 4
    sizes = [(200, 0), (330, 0), (64, 0)]
    c = Batch8(sizes, 8, 2, hd, 64, seed=hd)
    c.table = np.concatenate([c.table, np.full((3, 2), -1, np.int32)], 1)
    # (a page more for each)
    for s in range(3):
        c.table[s, -(-c.n_kv[s] // 64)] = c.free[s]
    c.max_pages += 2
    c.sizes = [(n + 1, 1) for n, _ in sizes]
    c.T, c.q_start, c.n_kv = 3, np.arange(4, dtype=np.int32), np.array([n for n, _ in c.sizes], np.int32)
    c.q = rng.standard_normal((3, 8, hd)).astype(np.float16)
    d = Device8(c, block=block)
    # bounds of all rows that are there
    whole = vxfa.paged(d.table.data_ptr(), d.n_kv.data_ptr(), d.q_start.data_ptr(), 3, c.max_pages, 400)
    d.set_list(np.zeros((3, 2, top), np.int32), block, 1, 1)
    w = c.hkv * hd
    new = [guarded(np.zeros((3, w), np.float32)) for _ in "kv"]
    nd = [vxfa.desc(t.data_ptr(), vxfa.F32, (w, 3, 1, 1), (4, 4 * w, 12 * w, 12 * w)) for t in new]
    own = vxfa.Context(0)

    def step(st):
        own.paged_append_q8(*nd, d.batch, d.k, d.ks, d.v, d.vs, stream=st)
        own.paged_bounds(d.k, d.ks, d.batch, d.b, d.bs, stream=st)
        own.paged_select(d.q, d.b, d.bs, d.batch, d.blocks, stream=st)
        own.flash_attn_ext_paged_blocks(d.q, d.k, d.ks, d.v, d.vs, d.batch, d.blocks, d.dst, 0.1, stream=st)

    # the bounds of the rows before, by chunks as long as the streams
    before = [n - 1 for n, _ in c.sizes]
    qs = np.concatenate([[0], np.cumsum(before)]).astype(np.int32)
    d.n_kv.copy_(torch.from_numpy(np.array(before, np.int32).view(np.uint8)))
    d.q_start.copy_(torch.from_numpy(qs.view(np.uint8)))
    own.paged_bounds(d.k, d.ks, whole, d.b, d.bs, stream=current())
    d.q_start.copy_(torch.from_numpy(c.q_start.view(np.uint8)))
    finish()
    save = c.sizes, c.q_start
    c.sizes, c.q_start = [(n, n) for n in before], qs
    b, bs = p8.bounds(c, block, d.b_np, d.bs_np)
    c.sizes, c.q_start = save
    assert np.array_equal(d.bounds()[0], b) and np.array_equal(d.bounds()[1], bs)
    graph = torch.cuda.CUDAGraph()
    side = torch.cuda.Stream()
    try:
        with torch.cuda.graph(graph, stream=side):
            step(side.cuda_stream)
        for turn in range(5):
            c.sizes = [(n + turn + 1, 1) for n, _ in sizes]
            c.n_kv = np.array([n for n, _ in c.sizes], np.int32)
            d.n_kv.copy_(torch.from_numpy(c.n_kv.view(np.uint8)))
            k_new, v_new = rows_of(rng, c, 3), rows_of(rng, c, 3)
            for t, x in zip(new, (k_new, v_new)):
                t.copy_(torch.from_numpy(x.reshape(-1).view(np.uint8)))
            c.q = rng.standard_normal(c.q.shape).astype(np.float16)
            d.qt.copy_(torch.from_numpy(c.q.reshape(-1).view(np.uint8)))
            if turn == 3:
                step(current())      # (eagerly, among the replays)
            else:
                torch.cuda.synchronize()
                graph.replay()
            finish()
            same_stored(c, d, k_new, v_new)
            c.k, c.v, c.ks, c.vs = d.ints("k").copy(), d.ints("v").copy(), d.scale("k").copy(), d.scale("v").copy()
            b, bs = p8.bounds(c, block, b, bs)
            assert np.array_equal(d.bounds()[0], b) and np.array_equal(d.bounds()[1], bs)
            lists = p8.select(c, block, b, bs, top, 1, 1)
            assert np.array_equal(d.list(), lists)
            want, err = p8.reference(c, 0.1, lists=lists, block=block)
            check_out(d.out(), want, err, True)
            d.check_guards()
    finally:
        own.close()
