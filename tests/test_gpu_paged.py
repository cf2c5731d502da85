"""The paged entry points on the GPU against a plain implementation in 64 bits
(paged_util.py, which derives the bounds): appends byte for byte, attention
of ragged chunks with score caps, distance slopes and windows, accumulated
weights, evictions, and a run of them together."""
import math

import numpy as np
import pytest

import cases
from paged_util import Batch, Device, check_out, check_weights, reference

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def ctx():
    from gpu_util import vxfa
    c = vxfa.Context(0)
    yield c
    c.close()


@pytest.fixture(params=[1, 2, 7])
def pieces(request, monkeypatch):
    """A context whose chunk calls cut the longest walk into this many pieces."""
    from gpu_util import vxfa
    monkeypatch.setenv("VXFA_PAGED_PIECES", str(request.param))
    c = vxfa.Context(0)
    yield c
    c.close()


def attend(ctx, c, scale=None, window=0, cap=0.0, bias=0.0, dst="f16", weights=None):
    """One call, checked; weights: "new", "on top" or "in place". Returns the output."""
    import torch
    scale = 1 / math.sqrt(c.hd) if scale is None else scale
    d = Device(c, dst, window)
    kw, w_out = {}, None
    if weights:
        from gpu_util import guarded, guards_intact
        views = __import__("conftest").load_package().views
        before = np.full(c.w.shape, 7.0, np.float32)
        w_out = d.wt if weights == "in place" else guarded(before)
        if weights == "in place":
            before = c.w
        kw["weights"] = d.vxfa.desc(w_out.data_ptr(), d.vxfa.F32, *views.weight_pages(c.n_pages, c.page, c.hkv))
        if weights != "new":
            kw["weights_in"] = d.w
    ctx.flash_attn_ext_paged(d.q, d.k, d.v, d.batch, d.dst, scale, bias, cap, stream=torch.cuda.current_stream().cuda_stream, **kw)
    torch.cuda.synchronize()
    want, add, err, adderr = reference(c, scale, window, cap, bias)
    got = d.out()
    check_out(got, want, err, dst == "f16")
    if weights:
        assert guards_intact(w_out)
        check_weights(c, d.weights(w_out), None if weights == "new" else c.w, add, adderr, before)
    d.check_guards()
    return got


# lengths around the units that kernels may walk in: 16, 32, 64, 128, 256
EDGES = [1, 2, 15, 16, 17, 31, 32, 33, 63, 64, 65, 127, 128, 129, 255, 257]
HEADS = [(8, 2, 128), (4, 4, 128), (16, 1, 128), (6, 2, 128), (5, 1, 128), (32, 1, 128), (7, 7, 64), (12, 3, 64), (8, 1, 64), (40, 2, 64)]


@pytest.mark.parametrize("hq,hkv,hd", HEADS)
def test_single_tokens(ctx, hq, hkv, hd):
    attend(ctx, Batch([(n, 1) for n in EDGES], hq, hkv, hd, seed=hq))


@pytest.mark.parametrize("hq,hkv,hd", HEADS)
def test_few_tokens(ctx, hq, hkv, hd):
    attend(ctx, Batch([(n + t, t) for n, t in ((0, 1), (0, 2), (0, 3), (16, 2), (31, 3), (100, 1), (255, 3), (700, 2))], hq, hkv, hd, seed=hq + 1))


@pytest.mark.parametrize("hq,hkv,hd", HEADS)
def test_chunks(ctx, hq, hkv, hd):
    attend(ctx, Batch([(70, 70), (33, 17), (300, 1), (500, 129), (64, 64), (5, 5)], hq, hkv, hd, seed=hq + 2))


@pytest.mark.parametrize("page", [16, 32, 64, 128, 1024])
@pytest.mark.parametrize("layout", ["row", "head"])
@pytest.mark.parametrize("t", [1, 40])
def test_pages_and_strides(ctx, page, layout, t):
    attend(ctx, Batch([(n, t) for n in (t, 45, 100, 333, 1030)], page=page, layout=layout, seed=page))


OPTIONS = [dict(cap=30.0), dict(bias=8.0), dict(cap=50.0, bias=8.0), dict(window=1), dict(window=31), dict(window=33, cap=20.0), dict(window=200, bias=4.0),
           dict(scale=0.0), dict(scale=-0.2), dict(scale=-0.1, cap=5.0), dict(scale=1.0), dict(scale=0.0, cap=3.0, bias=1.0)]


@pytest.mark.parametrize("opt", OPTIONS, ids=str)
@pytest.mark.parametrize("hq,hkv,hd", [(8, 2, 128), (6, 2, 64)])
@pytest.mark.parametrize("t", [1, 3, 50])
def test_scores(ctx, opt, hq, hkv, hd, t):
    attend(ctx, Batch([(t, t), (97, t), (300, t), (1000, t)], hq, hkv, hd, seed=t), **opt)


@pytest.mark.parametrize("dst", ["f16", "f32"])
@pytest.mark.parametrize("q", ["f16", "f32"])
@pytest.mark.parametrize("t", [1, 50])
def test_types(ctx, dst, q, t):
    attend(ctx, Batch([(t, t), (200, t), (431, t)], q_type=q, seed=5), dst=dst)
    attend(ctx, Batch([(t, t), (200, t)], hd=64, q_type=q, seed=5), dst=dst, weights="on top")


@pytest.mark.parametrize("weights", ["new", "on top", "in place"])
@pytest.mark.parametrize("hq,hkv,hd", [(8, 2, 128), (3, 3, 64), (16, 1, 128), (40, 2, 64)])
@pytest.mark.parametrize("opt", [dict(), dict(cap=30.0, bias=8.0), dict(window=70)], ids=str)
def test_weights(ctx, weights, hq, hkv, hd, opt):
    attend(ctx, Batch([(300, 1), (1, 1), (77, 1)], hq, hkv, hd, seed=8), weights=weights, **opt)
    attend(ctx, Batch([(300, 90), (20, 20), (1, 1), (700, 3), (129, 129)], hq, hkv, hd, page=32, seed=9), weights=weights, **opt)


@pytest.mark.parametrize("t", [1, 60])
def test_empty_and_short_streams(ctx, t):
    """Streams without tokens, without rows, and with fewer rows than tokens (the first tokens see nothing)."""
    c = Batch([(0, 0), (50, t), (30, 0), (t, t), (0, 0)], seed=3, behind=5)
    attend(ctx, c, weights="on top")
    c = Batch([(90, t), (80, t), (120, t)], seed=4)
    c.n_kv[1] = t // 2
    c.sizes[1] = (t // 2, t)
    got = attend(ctx, c)
    a = c.q_start[1]
    assert (got[a:a + t - t // 2] == 0).all()


@pytest.mark.parametrize("t", [1, 2, 60])
def test_absent_pages(ctx, t):
    c = Batch([(200, t), (100, t), (333, t), (65, t)], absent=[(0, 0), (0, 1), (0, 5), (1, 3), (2, 20), (2, 2), (3, 0), (3, 1), (3, 2), (3, 3), (3, 4)], seed=6)
    attend(ctx, c, weights="on top")
    # the pages that a window has left behind
    c = Batch([(200 + t, t), (150 + t, t)], absent=[(0, i) for i in range(6)] + [(1, 0)], seed=7)
    attend(ctx, c, window=40)


def test_no_tokens_and_no_streams(ctx):
    import torch
    c = Batch([(40, 0), (10, 0)], behind=3, seed=1)
    attend(ctx, c, weights="on top")
    d = Device(c)
    d.batch.n_streams = 0
    ctx.flash_attn_ext_paged(d.q, d.k, d.v, d.batch, d.dst, 0.1)
    torch.cuda.synchronize()
    assert (d.dt == 0xA5).all()


@pytest.mark.parametrize("t", [1, 50])
def test_sizes_out_of_range_do_no_harm(ctx, t):
    """Sizes on the device that break the bounds: clamped, nothing written elsewhere."""
    import torch
    c = Batch([(100, t), (60, t), (90, t)], seed=2)
    for n_kv, q_start in (([2 ** 31 - 1, -5, 90], [0, t, 2 * t, 3 * t]), ([100, 60, 90], [-7, t, 5 * t, 2 ** 31 - 1]),
                          ([100, 60, 90], [2 * t, t, 0, 3 * t]), ([100, 60, 90], [0, 3 * t, 0, 3 * t])):
        for limit in (t, 1):
            d = Device(c)
            d.n_kv.copy_(torch.from_numpy(np.array(n_kv, np.int32).view(np.uint8)))
            d.q_start.copy_(torch.from_numpy(np.array(q_start, np.int64).astype(np.int32).view(np.uint8)))
            d.batch.max_nq = limit
            ctx.flash_attn_ext_paged(d.q, d.k, d.v, d.batch, d.dst, 0.1, weights=d.w)
            torch.cuda.synchronize()
            raw = d.dt.cpu().numpy()
            assert (raw[:1024] == 0xA5).all() and (raw[-1024:] == 0xA5).all()
            d.check_guards()


@pytest.mark.parametrize("sizes", [[(5000, 1)], [(9000, 2)], [(3000 + 37 * i, 1) for i in range(9)], [(1100, 1100)],
                                   [(3333, 150)], [(2000, 1), (2600, 600), (90, 3), (4000, 1)]], ids=str)
@pytest.mark.parametrize("hq,hkv,hd", [(32, 8, 128), (8, 8, 64), (3, 1, 128)])
def test_long(ctx, sizes, hq, hkv, hd):
    """Enough rows for every stream to be cut into parts that are joined."""
    attend(ctx, Batch(sizes, hq, hkv, hd, page=16 if hd == 128 else 64, seed=hq), weights="on top")


@pytest.mark.parametrize("t", [1, 40])
def test_peaked_and_rising_scores(ctx, t):
    """Scores of hundreds, growing along the rows: the running maximum moves at every step."""
    c = Batch([(400, t), (1500, t)], seed=11, kv_scale=1.0, q_scale=1.0)
    g = np.linspace(0.1, 12.0, 1500).astype(np.float16)
    for s, (n, _) in enumerate(c.sizes):
        r = np.arange(n)
        c.k[c.table[s, r // c.page], r % c.page] *= g[:n, None, None]
    attend(ctx, c, scale=0.5, weights="new")
    attend(ctx, c, scale=0.5, cap=25.0)


def test_same_bits_again_and_beside_another_context(ctx):
    import torch
    from gpu_util import vxfa
    c = Batch([(3000, 1), (500, 1), (2222, 1)], 32, 8, seed=12)
    e = Batch([(1500, 200), (700, 1)], 32, 8, seed=13)
    other = vxfa.Context(0)
    try:
        first = [attend(ctx, c), attend(ctx, e)]
        d = [Device(c), Device(e)]
        streams = [torch.cuda.Stream(), torch.cuda.Stream()]
        torch.cuda.synchronize()
        for _ in range(3):
            for x, y, st in zip(d, (ctx, other), streams):
                y.flash_attn_ext_paged(x.q, x.k, x.v, x.batch, x.dst, 1 / math.sqrt(128), stream=st.cuda_stream)
        torch.cuda.synchronize()
        for x, want in zip(d, first):
            assert np.array_equal(x.out().view(np.uint16), want.view(np.uint16))
    finally:
        other.close()


@pytest.mark.parametrize("t", [1, 40])
def test_captured_call_follows_the_sizes(ctx, t):
    """A replay reads the tables and sizes as they are then; eager calls on the same context in between."""
    import torch
    c = Batch([(900, t), (900, t), (900, t)], seed=14)
    d = Device(c)
    st = torch.cuda.Stream()
    call = lambda s: ctx.flash_attn_ext_paged(d.q, d.k, d.v, d.batch, d.dst, 0.1, weights=d.w, stream=s)   # noqa: E731
    call(st.cuda_stream)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=st):
        call(st.cuda_stream)
    for sizes in ([900, 40, 300], [41, 800, 900], [500, 500, 500]):
        n = np.array(sizes, np.int32)
        d.n_kv.copy_(torch.from_numpy(n.view(np.uint8)))
        c.n_kv, c.sizes = n, [(int(x), t) for x in n]
        graph.replay()
        torch.cuda.synchronize()
        want, _, err, _ = reference(c, 0.1)
        got = d.out()
        check_out(got, want, err, True)
        attend(ctx, Batch([(1200, 30), (5, 5)], seed=15))
        d.dt.fill_(0xA5)
        graph.replay()
        torch.cuda.synchronize()
        assert np.array_equal(d.out(), got)


@pytest.mark.parametrize("t", [1, 33])
def test_pool_beyond_32_bits(ctx, t):
    """Pages more than 4 GiB apart."""
    import torch
    from gpu_util import vxfa
    c = Batch([(100, t), (70, t)], hq=4, hkv=1, page=32, seed=16, spare=20)   # (27 pages)
    row = 7 << 20                        # 7 MiB between rows, 224 MiB a page
    pools = [torch.zeros((c.n_pages * c.page * row,), dtype=torch.uint8, device="cuda") for _ in range(2)]
    assert pools[0].numel() > (1 << 32)
    for name, p in zip("kv", pools):
        x = torch.from_numpy(getattr(c, name).view(np.uint8).reshape(c.n_pages * c.page, -1)).cuda()
        p.view(-1, row)[:, :x.shape[1]] = x
    d = Device(c)
    nb = (2, row, 256, c.page * row)
    k, v = (vxfa.desc(p.data_ptr(), vxfa.F16, (128, c.page, 1, c.n_pages), nb) for p in pools)
    ctx.flash_attn_ext_paged(d.q, k, v, d.batch, d.dst, 0.09)
    torch.cuda.synchronize()
    want, _, err, _ = reference(c, 0.09)
    check_out(d.out(), want, err, True)


@pytest.mark.parametrize("opt", [dict(), dict(bias=8.0), dict(cap=30.0, bias=2.0), dict(window=900)], ids=str)
@pytest.mark.parametrize("hq,hkv,hd", [(8, 2, 128), (5, 5, 64)])
def test_walks_of_many_steps_with_absent_pages(pieces, opt, hq, hkv, hd):
    """Pages are looked up 16 steps (1024 rows) at a time; absent ones on both sides of that."""
    absent = [(0, i) for i in (0, 1, 7, 31, 32, 33, 63, 64, 65, 100, 126, 127, 128, 129, 130, 191, 192, 200, 218)] + [(1, i) for i in range(60, 70)]
    attend(pieces, Batch([(3500, 70), (2100, 150), (40, 3)], hq, hkv, hd, absent=absent, seed=21), weights="new", **opt)


@pytest.mark.parametrize("t", [1, 20])
@pytest.mark.parametrize("weights", [None, "on top"])
def test_many_streams(ctx, t, weights):
    """More streams than a wavefront has lanes."""
    rng = np.random.default_rng(22)
    attend(ctx, Batch([(int(n) + t, int(x)) for n, x in zip(rng.integers(0, 300, 150), rng.integers(0, t + 1, 150))], 4, 2, 64, seed=22), weights=weights)


def test_streams_whose_parts_have_no_room(ctx):
    """Records of 16 heads for 300 streams do not fit the workspace: whole streams, more than 64 tiles a wavefront, absent pages among them."""
    sizes = [(9000, 1)] + [(1 + i % 20, 1) for i in range(299)]
    attend(ctx, Batch(sizes, 256, 16, 64, seed=23, absent=[(0, i) for i in (0, 3, 250, 255, 256, 257, 300, 511, 512, 562)]))


@pytest.mark.parametrize("t", [1, 2])
def test_weights_without_room_for_scores(ctx, t):
    """Bounds so wide that single tokens' scores do not fit the workspace: the weights form them again."""
    c = Batch([(500, t), (33, t), (260, t), (1, 1)] * 10, 16, 4, 128, seed=24)
    wide = np.full((c.B, 1 << 12), -1, np.int32)          # 65536 rows a stream
    wide[:, :c.max_pages] = c.table
    c.table, c.max_pages = wide, 1 << 12
    attend(ctx, c, weights="on top")


@pytest.mark.parametrize("t", [1, 40])
@pytest.mark.parametrize("q_type", ["f16", "f32"])
def test_strided_queries(ctx, t, q_type):
    """Queries [head][token] with room between the rows."""
    import torch
    c = Batch([(100, t), (300, t)], 8, 2, 64, q_type=q_type, seed=25)
    d = Device(c)
    e = c.q.itemsize
    x = np.full((c.hq, c.T, c.hd + 16), np.nan, c.q.dtype)
    x[..., :c.hd] = c.q.transpose(1, 0, 2)
    g = torch.from_numpy(x).cuda()
    row = (c.hd + 16) * e
    q = d.vxfa.desc(g.data_ptr(), d.q.type, (c.hd, c.T, c.hq, 1), (e, row, c.T * row, c.hq * c.T * row))
    ctx.flash_attn_ext_paged(q, d.k, d.v, d.batch, d.dst, 0.12, weights=d.w)
    torch.cuda.synchronize()
    want, add, err, adderr = reference(c, 0.12)
    check_out(d.out(), want, err, True)
    check_weights(c, d.weights(), None, add, adderr, c.w)


@pytest.mark.parametrize("t", [1, 40])
def test_no_pages_at_all(ctx, t):
    """An empty pool: every row is absent, outputs are zeros."""
    import torch
    c = Batch([(0, t), (0, t)], seed=26, spare=1)
    c.n_kv[:] = 50
    c.sizes = [(0, t), (0, t)]
    d = Device(c)
    d.n_kv.copy_(torch.from_numpy(c.n_kv.view(np.uint8)))
    for x in (d.k, d.v):
        x.ne[3] = 0
    d.w.ne[2] = 0
    ctx.flash_attn_ext_paged(d.q, d.k, d.v, d.batch, d.dst, 0.12, weights=d.w)
    torch.cuda.synchronize()
    assert (d.out() == 0).all()
    d.batch.max_nq = 0
    d.dt.fill_(0xA5)
    ctx.flash_attn_ext_paged(d.q, d.k, d.v, d.batch, d.dst, 0.12, weights=d.w)
    torch.cuda.synchronize()
    assert (d.dt == 0xA5).all()


def test_rising_scores_with_slopes(ctx):
    """Keys that grow along the rows, the nearest the largest or the smallest, under distance slopes: the walk from the last block, too, has
    to follow a rising maximum."""
    for t in (1, 3, 70):
        for lo, hi in ((0.1, 12.0), (12.0, 0.1)):
            c = Batch([(700, t), (1500, t)], seed=27)
            g = np.linspace(lo, hi, 1500).astype(np.float16)
            for s, (n, _) in enumerate(c.sizes):
                r = np.arange(n)
                c.k[c.table[s, r // c.page], r % c.page] *= g[:n, None, None]
            attend(ctx, c, scale=0.4, bias=8.0, weights="new")
            attend(ctx, c, scale=0.4, bias=1.0, cap=60.0)


# ---- append ----------------------------------------------------------------------


def append(ctx, c, rope_dims=0, with_q=False, base=1e6, seed=0):
    """Appends random rows; pools and rotated queries checked. Returns the device batch."""
    import torch
    from gpu_util import guarded, vxfa
    views = __import__("conftest").load_package().views
    rng = np.random.default_rng(seed)
    T, w = c.T + c.behind, c.hkv * c.hd
    new = [rng.standard_normal((T, c.hkv, c.hd)).astype(np.float32) for _ in range(2)]
    new[0].reshape(-1)[:4] = [1e30, -1e30, 65520.0, 1e-8]
    q = rng.standard_normal((T, c.hq, c.hd)).astype(np.float32)
    pos = rng.integers(0, 9000, T).astype(np.int32)
    d = Device(c)
    before = [d.pool(n).copy() for n in "kv"]
    t = [guarded(x) for x in (*new, q, pos)]
    nd = [vxfa.desc(x.data_ptr(), vxfa.F32, (w, T, 1, 1), (4, 4 * w, 4 * w * T, 4 * w * T)) for x in t[:2]]
    rope = vxfa.rope(t[3].data_ptr(), rope_dims, base) if rope_dims else None
    qo = guarded(np.full((T, c.hq, c.hd), 0x1234, np.uint16))
    kw = dict(q=vxfa.desc(t[2].data_ptr(), vxfa.F32, *views.decoder_q(T, c.hq, c.hd)),
              q_out=vxfa.desc(qo.data_ptr(), vxfa.F16, *views.decoder_q(T, c.hq, c.hd, 2))) if with_q else {}
    ctx.paged_append(*nd, d.batch, d.k, d.v, rope=rope, stream=torch.cuda.current_stream().cuda_stream, **kw)
    torch.cuda.synchronize()
    kr, qr = new[0], q
    if rope_dims:
        kr, qr = cases.rope_ggml(new[0], pos, rope_dims, base), cases.rope_ggml(q, pos, rope_dims, base)
    want = [x.copy() for x in before]
    mask = np.zeros(want[0].shape, bool)
    with np.errstate(over="ignore"):
        for s, (n, tk) in enumerate(c.sizes):
            for i in range(tk):
                r = n - tk + i
                p = c.table[s, r // c.page] if r >= 0 else -1
                if 0 <= p < c.n_pages:
                    want[0][p, r % c.page] = kr[c.q_start[s] + i].astype(np.float16)
                    want[1][p, r % c.page] = new[1][c.q_start[s] + i].astype(np.float16)
                    mask[p, r % c.page] = True
    gk, gv = d.pool("k"), d.pool("v")
    assert np.array_equal(gv.view(np.uint16), want[1].view(np.uint16))
    if not rope_dims:
        assert np.array_equal(gk.view(np.uint16), want[0].view(np.uint16))
    else:
        # cos and sin are off by a few F32 steps: products of up to 2^3 by 2^-20, then the rounding to f16
        assert np.array_equal(gk.view(np.uint16)[~mask], want[0].view(np.uint16)[~mask])
        a, b = gk[mask].astype(np.float64), want[0][mask].astype(np.float64)
        fin = np.isfinite(b)
        assert np.array_equal(fin, np.isfinite(a))
        assert (np.abs(a[fin] - b[fin]) <= 2.0 ** -10 * np.abs(b[fin]) + 2.0 ** -17).all()
    got_q = qo.cpu().numpy().view(np.uint16).reshape(T, c.hq, c.hd)
    assert (got_q[c.T:] == 0x1234).all()
    if with_q:
        assert (np.abs(got_q[:c.T].view(np.float16).astype(np.float64) - qr[:c.T]) <= 2.0 ** -10 * np.abs(qr[:c.T]) + 2.0 ** -17).all()
    else:
        assert (got_q == 0x1234).all()
    d.check_guards()
    return d


@pytest.mark.parametrize("hq,hkv,hd", [(8, 2, 128), (7, 7, 64), (16, 1, 128), (5, 1, 64)])
@pytest.mark.parametrize("form", ["plain", "rope", "rope+q", "part"])
@pytest.mark.parametrize("sizes", [[(1, 1)], [(n, 1) for n in (1, 16, 17, 40, 100)], [(70, 70), (33, 0), (100, 5), (0, 0), (64, 33)]], ids=str)
def test_append(ctx, hq, hkv, hd, form, sizes):
    c = Batch(sizes, hq, hkv, hd, behind=2, layout="head" if form == "part" else "row", seed=hq)
    append(ctx, c, {"plain": 0, "part": hd // 2}.get(form, hd), form in ("rope+q", "part"))


def test_append_to_absent_pages_and_before_the_first_row(ctx):
    c = Batch([(40, 10), (30, 20)], absent=[(0, 2), (1, 0)], seed=2)
    append(ctx, c)
    c = Batch([(40, 10), (30, 20)], seed=2)
    c.n_kv[1], c.sizes[1] = 5, (5, 20)
    append(ctx, c, 128, True)


# ---- eviction --------------------------------------------------------------------


def kept_rows(w, n, budget, sink, recent):
    """Row numbers, ascending: by weight, ties to the first, NaN last."""
    if n <= budget:
        return np.arange(n)
    mid = np.arange(sink, n - recent)
    x = np.where(np.isnan(w[mid]), -np.inf, w[mid].astype(np.float64))
    isnan = np.isnan(w[mid])
    order = np.lexsort((mid, -x, isnan))
    return np.sort(np.concatenate([np.arange(sink), np.arange(n - recent, n), mid[order[:budget - sink - recent]]]))


def evict(ctx, c, budget, sink=0, recent=0, with_kept=True, drop=()):
    import torch
    from gpu_util import guarded, guards_intact, vxfa
    need = -(-min(budget, max(n for n, _ in c.sizes) or 1) // c.page)
    assert len(c.free) >= need * c.B
    to = np.full((c.B, need), -1, np.int32)
    to[:] = c.free[:need * c.B].reshape(c.B, need)
    for s, i in drop:
        to[s, i] = -1
    d = Device(c)
    before = [d.pool(n).copy() for n in "kv"] + [d.weights().copy()]
    tt, kt, nt = guarded(to), guarded(np.full((c.B, c.hkv, budget), -7, np.int32)), guarded(np.full((c.B,), -7, np.int32))
    ev = vxfa.evict(tt.data_ptr(), need, budget, sink, recent, kept=kt.data_ptr() if with_kept else 0, n_kv=nt.data_ptr() if with_kept else 0)
    ctx.paged_evict(d.k, d.v, d.w, d.batch, ev, stream=torch.cuda.current_stream().cuda_stream)
    torch.cuda.synchronize()
    want = [x.copy() for x in before]
    kept = np.full((c.B, c.hkv, budget), -1, np.int32)
    for s, (n, _) in enumerate(c.sizes):
        r = np.arange(n)
        p = c.table[s, r // c.page].astype(np.int64)
        ok = (p >= 0) & (p < c.n_pages)
        for h in range(c.hkv):
            w = np.where(ok, before[2][np.where(ok, p, 0), h, r % c.page], np.nan)
            j = kept_rows(w, n, budget, sink, recent)
            kept[s, h, :len(j)] = j
            for i, x in enumerate(j):
                q = to[s, i // c.page]
                if q < 0:
                    continue
                for m in range(2):
                    want[m][q, i % c.page, h] = before[m][p[x], x % c.page, h] if ok[x] else 0
                want[2][q, h, i % c.page] = w[x]
    got = [d.pool("k"), d.pool("v"), d.weights()]
    for a, b in zip(got, want):
        assert np.array_equal(np.isnan(a), np.isnan(b)) and np.array_equal(a[~np.isnan(a)], b[~np.isnan(b)])
    if with_kept:
        assert np.array_equal(kt.cpu().numpy().view(np.int32).reshape(kept.shape), kept)
        assert np.array_equal(nt.cpu().numpy().view(np.int32), np.minimum(c.n_kv, budget))
    for t in (tt, kt, nt):
        assert guards_intact(t)
    d.check_guards()


@pytest.mark.parametrize("hkv,hd,page,layout", [(2, 128, 16, "row"), (3, 64, 32, "head"), (8, 128, 16, "row")])
@pytest.mark.parametrize("budget,sink,recent", [(1, 0, 0), (1, 1, 0), (1, 0, 1), (40, 0, 0), (64, 4, 16), (100, 50, 50), (333, 7, 99), (1000, 4, 100)])
def test_evict(ctx, hkv, hd, page, layout, budget, sink, recent):
    c = Batch([(n, 0) for n in (0, 1, 39, 40, 41, 101, 333, 1000, 2100)], hkv * 2, hkv, hd, page, layout, seed=budget, spare=9 * (-(-budget // page)) + 2)
    evict(ctx, c, budget, sink, recent)
    evict(ctx, c, budget, sink, recent, with_kept=False)


def test_evict_long_streams(ctx):
    """Streams of several segments of 8192 rows, ties across them."""
    c = Batch([(20000, 0), (8193, 0), (8192, 0)], 2, 2, 64, 64, seed=6, spare=3 * 150)
    c.w = np.round(c.w * 50) / 50
    evict(ctx, c, 9000, 100, 1000)
    evict(ctx, c, 8192, 0, 0)
    evict(ctx, c, 5, 1, 2)


@pytest.mark.parametrize("kind", ["equal", "few", "signs", "nan", "inf", "tiny"])
def test_evict_ties_and_odd_weights(ctx, kind):
    c = Batch([(1500, 0), (600, 0), (5000, 0)], 4, 2, seed=3, spare=3 * 20)
    rng = np.random.default_rng(4)
    live = ~np.isnan(c.w)
    c.w[live] = {"equal": lambda n: np.full(n, 0.5), "few": lambda n: rng.integers(0, 3, n) / 2, "signs": lambda n: rng.integers(-2, 3, n) * rng.choice([0.0, -0.0, 1.0], n),
                 "nan": lambda n: np.where(rng.random(n) < 0.9, np.nan, rng.random(n)), "inf": lambda n: rng.choice([np.inf, -np.inf, 1.0], n),
                 "tiny": lambda n: rng.integers(0, 5, n) * 1e-45}[kind](int(live.sum())).astype(np.float32)
    evict(ctx, c, 300, 3, 20)


def test_evict_absent_pages(ctx):
    c = Batch([(400, 0), (100, 0)], absent=[(0, 0), (0, 3), (1, 6)], seed=5, spare=2 * 20)
    evict(ctx, c, 130, 20, 30)
    evict(ctx, c, 130, 20, 30, drop=[(0, 1), (1, 0)])


def test_captured_step_of_all_three(ctx):
    """Append, attention with weights and eviction in one graph, replayed on other sizes with eager work in between, against the same calls
    made directly."""
    import torch
    from gpu_util import vxfa
    T, hkv, hd, page = 3, 2, 128, 16
    c = Batch([(300, 1), (300, 1), (300, 1)], 8, hkv, hd, page, seed=28, spare=3 * 6)
    new = torch.randn((2, T, hkv * hd), device="cuda")
    pos = torch.tensor([299, 5, 1000], device="cuda", dtype=torch.int32)
    to = torch.from_numpy(c.free[:18].reshape(3, 6).copy()).cuda()
    w = hkv * hd

    def bind(d):
        nd = [vxfa.desc(x.data_ptr(), vxfa.F32, (w, T, 1, 1), (4, 4 * w, 4 * w * T, 4 * w * T)) for x in new]
        kept = torch.full((3, hkv, 90), -7, device="cuda", dtype=torch.int32)
        ev = vxfa.evict(to.data_ptr(), 6, 90, 4, 20, kept=kept.data_ptr())
        rope = vxfa.rope(pos.data_ptr(), hd, 1e6)

        def step(s):
            ctx.paged_append(*nd, d.batch, d.k, d.v, rope=rope, stream=s)
            ctx.flash_attn_ext_paged(d.q, d.k, d.v, d.batch, d.dst, 0.09, 2.0, 20.0, weights_in=d.w, weights=d.w, stream=s)
            ctx.paged_evict(d.k, d.v, d.w, d.batch, ev, stream=s)
        return step, kept

    a, b = Device(c), Device(c)
    (sa, ka), (sb, kb) = bind(a), bind(b)
    st = torch.cuda.Stream()
    graph = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph, stream=st):
        sa(st.cuda_stream)
    for sizes in ([300, 250, 120], [299, 33, 300], [100, 300, 17]):
        n = torch.from_numpy(np.array(sizes, np.int32).view(np.uint8)).cuda()
        for d in (a, b):
            d.n_kv.copy_(n)
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        attend(ctx, Batch([(900, 40), (70, 1)], seed=29), weights="new")
        sb(torch.cuda.current_stream().cuda_stream)
        torch.cuda.synchronize()
        assert torch.equal(ka, kb) and torch.equal(a.dt, b.dt)
        assert torch.equal(a.wt.view(torch.int32), b.wt.view(torch.int32))
        for name in "kv":
            assert torch.equal(a.pools[name][0], b.pools[name][0])


def test_serving_run(ctx):
    """Prompts, then decode steps with accumulated weights, an eviction, and further steps over what it kept: each step against the reference
    on the caches as they are."""
    import torch
    from gpu_util import guarded, vxfa
    scale = 1 / math.sqrt(128)
    c = Batch([(150, 150), (40, 40), (0, 0)], seed=20, spare=60)
    c.max_pages = 16
    table = np.full((3, 16), -1, np.int32)
    table[:, :c.table.shape[1]] = c.table[:, :16]
    c.table, free = table, list(c.free)
    state = {}

    def step(sizes):
        c.sizes = sizes
        c.n_kv = np.array([n for n, _ in sizes], np.int32)
        c.q_start = np.concatenate([[0], np.cumsum([t for _, t in sizes])]).astype(np.int32)
        c.T = int(c.q_start[-1])
        for s, (n, t) in enumerate(sizes):
            for i in range(-(-n // c.page)):
                if c.table[s, i] < 0:
                    c.table[s, i] = free.pop()
            # new rows begin with no weight
            r = np.arange(n - t, n)
            c.w[c.table[s, r // c.page], :, r % c.page] = 0
        c.q = np.random.default_rng(c.T).standard_normal((c.T, c.hq, c.hd)).astype(np.float16)
        d = append(ctx, c, 128, seed=c.T + len(state))
        state[len(state)] = 1
        c.k, c.v = d.pool("k").copy(), d.pool("v").copy()
        c.k[~np.isfinite(c.k) & ~np.isnan(c.k)] = 1.0    # (the append test's infinities)
        d = Device(c)
        ctx.flash_attn_ext_paged(d.q, d.k, d.v, d.batch, d.dst, scale, 0.0, 30.0, weights_in=d.w, weights=d.w, stream=torch.cuda.current_stream().cuda_stream)
        torch.cuda.synchronize()
        want, add, err, adderr = reference(c, scale, 0, 30.0)
        check_out(d.out(), want, err, True)
        check_weights(c, d.weights(), c.w, add, adderr, c.w)
        c.w = d.weights().copy()

    step([(150, 150), (40, 40), (0, 0)])
    step([(151, 1), (41, 1), (60, 60)])
    step([(152, 1), (42, 1), (61, 1)])
    # a budget of 48 rows
    to = np.full((3, 3), -1, np.int32)
    for s in range(3):
        for i in range(3):
            to[s, i] = free.pop()
    d = Device(c)
    tt, nt = guarded(to), guarded(np.zeros(3, np.int32))
    ctx.paged_evict(d.k, d.v, d.w, d.batch, vxfa.evict(tt.data_ptr(), 3, 48, 2, 10, n_kv=nt.data_ptr()), stream=torch.cuda.current_stream().cuda_stream)
    torch.cuda.synchronize()
    left = nt.cpu().numpy().view(np.int32)
    assert list(left) == [48, 42, 48]
    c.k, c.v, c.w = d.pool("k").copy(), d.pool("v").copy(), d.weights().copy()
    c.table[:] = -1
    c.table[:, :3] = to
    step([(49, 1), (43, 1), (49, 1)])
    step([(53, 4), (44, 1), (90, 41)])
