"""Single tokens over pages of 8 bits with four heads a workgroup, lists of all blocks beside the call over all rows,
calls that repeat themselves, strides, the largest pages, on the GPU (against a plain implementation in 64 bits, paged8_util.py)."""
import math

import numpy as np
import pytest

import paged8_util as p8
from paged8_util import Batch8, Device8
from paged_util import Batch, check_out

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def ctx():
    from gpu_util import vxfa
    c = vxfa.Context(0)
    yield c
    c.close()


def finish():
    import torch
    torch.cuda.synchronize()


def current():
    import torch
    return torch.cuda.current_stream().cuda_stream


def attend(ctx, d, scale, bias=0.0, cap=0.0):
    """dst over all rows, of whichever pool."""
    if d.ks is not None:
        ctx.flash_attn_ext_paged_q8(d.q, d.k, d.ks, d.v, d.vs, d.batch, d.dst, scale, bias, cap, stream=current())
    else:
        ctx.flash_attn_ext_paged(d.q, d.k, d.v, d.batch, d.dst, scale, bias, cap, stream=current())
    finish()
    return d.out()


# heads (hq, hkv, hd) and streams that take four heads a workgroup under a bound of 8192 rows, and the rows that they have
WIDE = [((32, 8, 128), 12), ((8, 8, 128), 12), ((8, 4, 64), 24), ((24, 8, 64), 12)]


@pytest.mark.parametrize("opt", [dict(), dict(cap=30.0), dict(bias=8.0), dict(window=300)], ids=str)
@pytest.mark.parametrize("heads,streams", WIDE)
def test_four_heads_a_workgroup(ctx, heads, streams, opt):
    rows = np.random.default_rng(streams).integers(1, 900, streams)
    rows[:3] = 1, 8000, 513
    c = Batch8([(int(n), 1) for n in rows], *heads, 64, seed=heads[0], behind=2, absent=[(1, 3), (1, 124)])
    c.table = np.concatenate([c.table, np.full((streams, 128 - c.max_pages), -1, np.int32)], 1)
    c.max_pages = 128
    d = Device8(c, window=opt.get("window", 0))
    scale = 1 / math.sqrt(c.hd)
    got = attend(ctx, d, scale, opt.get("bias", 0.0), opt.get("cap", 0.0))
    want, err = p8.reference(c, scale, **opt)
    check_out(got, want, err, True)
    d.check_guards()


def test_four_heads_a_workgroup_beyond_the_lanes(ctx):
    """Parts of more than 32 steps of a wavefront, whose pages are read 32 steps at a time: 8 streams that share
    their pages, 64 heads."""
    c = Batch8([(8300, 1)] + [(1, 1)] * 7, 64, 64, 64, 64, seed=21)
    c.sizes = [(8300 - 9 * s, 1) for s in range(8)]
    c.n_kv = np.array([n for n, _ in c.sizes], np.int32)
    c.table[:] = c.table[0]
    d = Device8(c, "f32")
    got = attend(ctx, d, 0.125)
    want, err = p8.reference(c, 0.125)
    check_out(got, want, err, False)
    d.check_guards()


@pytest.mark.parametrize("kind", [Batch, Batch8])
@pytest.mark.parametrize("hq,hkv,hd", [(8, 2, 128), (6, 2, 64), (32, 1, 128)])
def test_lists_of_all_blocks_are_all_rows(ctx, kind, hq, hkv, hd):
    """The call over lists of all blocks against the call over all rows: no further apart than either may be from 64
    bits. Single tokens, and chunks, which the one walks token by token and the other in tiles."""
    for sizes in ([(500, 1), (77, 1), (1000, 1)], [(500, 40), (77, 77), (300, 3)]):
        c = kind(sizes, hq, hkv, hd, 64, seed=9)
        scale = 1 / math.sqrt(hd)
        for opt in (dict(), dict(cap=20.0, bias=4.0), dict(window=90)):
            d = Device8(c, "f32", opt.get("window", 0))
            args = opt.get("bias", 0.0), opt.get("cap", 0.0)
            rows = attend(ctx, d, scale, *args)
            want, err = p8.reference(c, scale, **opt)
            check_out(rows, want, err, False)
            n = -(-max(n for n, _ in sizes) // 32)
            d.set_list(np.broadcast_to(np.arange(n, dtype=np.int32), (c.T, hkv, n)).copy(), 32)
            d.dt.fill_(0xA5)
            ctx.flash_attn_ext_paged_blocks(d.q, d.k, d.ks, d.v, d.vs, d.batch, d.blocks, d.dst, scale, *args, stream=current())
            finish()
            assert (np.abs(d.out() - rows) <= 2 * err + 2.0 ** -23 * np.abs(want)).all()
            check_out(d.out(), want, err, False)


def test_calls_repeat_themselves(ctx):
    """The same calls again give the same bits: all five entry points, in tokens and chunks, with sizes that are cut."""
    from gpu_util import guarded, vxfa
    rng = np.random.default_rng(3)
    for sizes in ([(8192, 1), (700, 1), (5000, 2)], [(3000, 200), (600, 1), (90, 90)]):
        c = Batch8(sizes, 8, 2, 128, 64, seed=4)
        w = c.hkv * c.hd
        new = [guarded(rng.standard_normal((c.T, w)).astype(np.float32)) for _ in "kv"]
        nd = [vxfa.desc(t.data_ptr(), vxfa.F32, (w, c.T, 1, 1), (4, 4 * w, 4 * w * c.T, 4 * w * c.T)) for t in new]
        seen = []
        for _ in range(3):
            d = Device8(c, "f32", block=32)
            d.set_list(np.full((c.T, 2, 20), -7, np.int32), 32, 1, 2)
            ctx.paged_append_q8(*nd, d.batch, d.k, d.ks, d.v, d.vs, stream=current())
            ctx.paged_bounds(d.k, d.ks, d.batch, d.b, d.bs, stream=current())
            ctx.paged_select(d.q, d.b, d.bs, d.batch, d.blocks, stream=current())
            ctx.flash_attn_ext_paged_blocks(d.q, d.k, d.ks, d.v, d.vs, d.batch, d.blocks, d.dst, 0.1, stream=current())
            finish()
            some = d.out().copy()
            d.dt.fill_(0xA5)
            seen.append([some, attend(ctx, d, 0.1), d.list().copy(), d.ints("k").copy(), d.ints("v").copy(), d.scale("k").copy(),
                         d.scale("v").copy(), *(x.copy() for x in d.bounds())])
        for other in seen[1:]:
            for a, b in zip(seen[0], other):
                assert a.tobytes() == b.tobytes()


def spread(x, order, pad):
    """x's bytes with its dims in memory order `order` (slowest first), `pad` bytes behind each innermost row; the buffer
    and bytes between neighbours of each dim."""
    from gpu_util import guarded
    y = np.ascontiguousarray(x.transpose(order))
    rows = y.reshape(-1, y.shape[-1]).view(np.uint8)
    full = np.concatenate([rows, np.full((len(rows), pad), 0x5A, np.uint8)], 1)
    nb, at = [0] * x.ndim, full.shape[1]
    nb[order[-1]] = x.itemsize
    for i in range(x.ndim - 2, -1, -1):
        nb[order[i]] = at
        at *= y.shape[i]
    return guarded(full), nb


def test_strides(ctx):
    """Queries by head, padded rows, scales and bounds by page with room between: the same bits as tensors as they lie
    in the other tests."""
    import torch
    from gpu_util import guarded, vxfa
    rng = np.random.default_rng(6)
    for sizes in ([(500, 1), (77, 2)], [(500, 60), (90, 90)]):
        c = Batch8(sizes, 8, 2, 128, 64, seed=8)
        w, T = c.hkv * c.hd, c.T
        k_new, v_new = (rng.standard_normal((T, w)).astype(np.float32) for _ in "kv")
        q32 = rng.standard_normal((T, c.hq, c.hd)).astype(np.float32)
        pos = guarded(np.arange(T, dtype=np.int32))
        outs = []
        for strided in (False, True):
            d = Device8(c, "f32", block=32)
            lists = np.full((T, c.hkv, 6), -7, np.int32)
            d.set_list(lists, 32, 1, 1)
            order, pad = ((1, 0, 2), 48) if strided else ((0, 1, 2), 0)
            keep = []

            def tensor(x, type_, order, pad, dims):
                """dims: x's dim of each ne."""
                t, nb = spread(x, order, pad)
                keep.append(t)
                ne = [x.shape[i] if i is not None else 1 for i in dims]
                return t, vxfa.desc(t.data_ptr(), type_, tuple(ne), tuple(nb[i] if i is not None else t.numel() for i in dims))

            kn, kd = tensor(k_new, vxfa.F32, (0, 1), pad, (1, 0, None, None))
            vn, vd = tensor(v_new, vxfa.F32, (0, 1), pad, (1, 0, None, None))
            qt, qd = tensor(q32, vxfa.F32, order, pad, (2, 0, 1, None))
            qo, qod = tensor(np.zeros(q32.shape, np.float16), vxfa.F16, order, pad, (2, 0, 1, None))
            ks, ksd = tensor(c.ks, vxfa.F32, order, 4 if strided else 0, (2, 1, 0, None))
            vs, vsd = tensor(c.vs, vxfa.F32, order, 4 if strided else 0, (2, 1, 0, None))
            bt, bd = tensor(d.b_np, vxfa.I8, (1, 0, 2, 3) if strided else (0, 1, 2, 3), pad, (3, 2, 1, 0))
            bst, bsd = tensor(d.bs_np, vxfa.F32, order, 4 if strided else 0, (2, 1, 0, None))
            st = current()
            ctx.paged_append_q8(kd, vd, d.batch, d.k, ksd, d.v, vsd, rope=vxfa.rope(pos.data_ptr(), 128, 1e6), q=qd, q_out=qod, stream=st)
            ctx.paged_bounds(d.k, ksd, d.batch, bd, bsd, stream=st)
            ctx.paged_select(qod, bd, bsd, d.batch, d.blocks, stream=st)
            ctx.flash_attn_ext_paged_blocks(qod, d.k, ksd, d.v, vsd, d.batch, d.blocks, d.dst, 0.1, stream=st)
            finish()
            some = d.out().copy()
            ctx.flash_attn_ext_paged_q8(qod, d.k, ksd, d.v, vsd, d.batch, d.dst, 0.1, stream=st)
            finish()
            d.check_guards()

            def back(t, x, order, pad):
                rows = t.cpu().numpy().reshape(-1, x.shape[order[-1]] * x.itemsize + pad)
                assert (rows[:, rows.shape[1] - pad:] == 0x5A).all() or pad == 0, "write between rows"
                y = np.ascontiguousarray(rows[:, :rows.shape[1] - pad]).view(x.dtype).reshape([x.shape[i] for i in order])
                return y.transpose(np.argsort(order)).tobytes()

            small = 4 if strided else 0
            outs.append([some.tobytes(), d.out().tobytes(), d.list().tobytes(), d.ints("k").tobytes(), d.ints("v").tobytes(),
                         back(qo, np.zeros(q32.shape, np.float16), order, pad), back(ks, c.ks, order, small), back(vs, c.vs, order, small),
                         back(bt, d.b_np, (1, 0, 2, 3) if strided else (0, 1, 2, 3), pad), back(bst, d.bs_np, order, small)])
            torch.cuda.synchronize()
        assert [a == b for a, b in zip(*outs)] == [True] * 10


@pytest.mark.parametrize("sizes", [[(66000, 1), (300, 2)], [(66000, 30), (300, 300)]])
def test_the_largest_pages(ctx, sizes):
    c = Batch8(sizes, 2, 1, 64, 65536, seed=5, spare=1)
    d = Device8(c, "f32", block=65536)
    got = attend(ctx, d, 0.125)
    want, err = p8.reference(c, 0.125)
    check_out(got, want, err, False)
    # a block a page: both of the long stream's, the one of the other
    ctx.paged_bounds(d.k, d.ks, d.batch, d.b, d.bs, stream=current())
    d.set_list(np.full((c.T, 1, 2), -7, np.int32), 65536)
    ctx.paged_select(d.q, d.b, d.bs, d.batch, d.blocks, stream=current())
    d.dt.fill_(0xA5)
    ctx.flash_attn_ext_paged_blocks(d.q, d.k, d.ks, d.v, d.vs, d.batch, d.blocks, d.dst, 0.125, stream=current())
    finish()
    b, bs = p8.bounds(c, 65536, d.b_np, d.bs_np)
    assert np.array_equal(d.bounds()[0], b) and np.array_equal(d.bounds()[1], bs)
    assert (d.list()[:, 0] == np.where(np.arange(c.T)[:, None] < sizes[0][1], [0, 1], [0, -1])).all()
    check_out(d.out(), want, err, False)
    d.check_guards()
