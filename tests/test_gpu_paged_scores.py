"""Score caps of every size, on the GPU against 64 bits: scores far below the cap
are what they are without one, scores about and above it are bent, and neither may
lose digits to the cap's size. Bounds that do not grow with the cap."""
import math

import numpy as np
import pytest

from paged_util import HALF, Batch, Device, check_out, check_weights, slopes

pytestmark = pytest.mark.gpu

MANY = [(700, 250), (650, 131), (300, 200), (250, 250), (900, 129), (129, 129), (400, 160), (500, 240)]


@pytest.fixture(scope="module")
def ctx():
    from gpu_util import vxfa
    c = vxfa.Context(0)
    yield c
    c.close()


def exact(c, scale, cap=0.0, bias=0.0, window=0):
    """Outputs, their bounds, weights added and theirs, as paged_util.reference gives them, with the cap's part of a
    score's error taken relative to the score:
    dx = 2^-24 nz Smax        F32 sums of at most nz products that are not 0
       + 2^-22 X              scaling, distance term, subtraction of the maximum
       + 2^-18 Xfar           a wide cap's form from a fifth of the cap on, where cap - 2 cap / (1 + E) is off by at
                              most 1.9 * 2^-22 cap (E, 1 + E, reciprocal and result rounded, a step of the reciprocal
                              and of the exponential), 1.9 / tanh(0.2) * 2^-22 = 2^-18.6 of |x|; below, the series
                              is off by 2^-23 |x|, a part of X's
       or + 2^-22 cap         a cap of at most 64."""
    G, D = c.hq // c.hkv, c.hd
    out, err = np.zeros((c.T, c.hq, D)), np.zeros((c.T, c.hq, D))
    add, adderr = {}, {}
    nz = np.count_nonzero(c.q[:c.T], axis=-1).max()
    sl = slopes(c.hq, bias)
    for s, (n, t) in enumerate(c.sizes):
        for h in range(c.hkv):
            add[s, h], adderr[s, h] = np.zeros(n), np.zeros(n)
            k, there = c.rows(s, h, c.k)
            v, _ = c.rows(s, h, c.v)
            j, p = np.arange(n)[None], (n - t + np.arange(t))[:, None]
            live = (j <= p) & there[None] & ((j > p - window) | (window == 0))
            for g in range(h * G, (h + 1) * G):
                at = slice(c.q_start[s], c.q_start[s] + t)
                q = c.q[at, g].astype(np.float64)
                S = abs(scale) * (np.abs(q) @ np.abs(k).T)
                xc = scale * (q @ k.T)
                if cap:
                    xc = cap * np.tanh(xc / cap)
                x = np.where(live, xc + sl[g] * (j - p), -np.inf)
                m = np.maximum(x.max(1, initial=-np.inf), -1e300)[:, None]
                e = np.exp(x - m)
                l = e.sum(1, keepdims=True)
                P = e / np.where(l > 0, l, 1)
                out[at, g] = P @ v
                near = live & (x > m - 40)
                X = np.where(near, np.abs(x) + np.abs(x - m) + np.abs(xc), 0).max(1, initial=0)
                dx = 2.0 ** -24 * nz * np.where(live, S, 0).max(1, initial=0) + 2.0 ** -22 * X
                if cap > 64:
                    dx = dx + 2.0 ** -18 * np.where(near & (np.abs(xc) > 0.19 * cap), np.abs(xc), 0).max(1, initial=0)
                else:
                    dx = dx + 2.0 ** -22 * cap
                if c.q_type == "f32":
                    dx = dx + HALF * np.where(live, S, 0).max(1, initial=0)
                N = live.sum(1)
                err[at, g] = 2 * ((HALF + 3 * dx)[:, None] * (P @ np.abs(v))
                                  + (2.0 ** -25 * P.max(1, initial=0) * N * np.abs(v).max(initial=0))[:, None])
                add[s, h] += P.sum(0)
                adderr[s, h] += (P * (3 * dx + 2.0 ** -24 * (N + t * G))[:, None]).sum(0) + t * 2.0 ** -126
    return out, err, add, adderr


def check(ctx, c, scale=None, cap=0.0, bias=0.0, window=0):
    import torch
    scale = 1 / math.sqrt(c.hd) if scale is None else scale
    d = Device(c, "f32", window)
    ctx.flash_attn_ext_paged(d.q, d.k, d.v, d.batch, d.dst, scale, bias, cap, weights_in=d.w, weights=d.w,
                             stream=torch.cuda.current_stream().cuda_stream)
    torch.cuda.synchronize()
    out, err, add, adderr = exact(c, scale, cap, bias, window)
    check_weights(c, d.weights(), c.w, add, adderr, c.w)
    check_out(d.out(), out, err, False)
    d.check_guards()


def without_weights(c):
    """Accumulators at 0, so that what a call adds is seen to its last digits."""
    c.w[~np.isnan(c.w)] = 0
    return c


CAPS = [64.0, 65.0, 1e3, 1e5, 1e7, 1e30, 2e38]


@pytest.mark.parametrize("cap", CAPS)
@pytest.mark.parametrize("opt", [dict(), dict(bias=8.0), dict(window=70, scale=-0.2)], ids=str)
@pytest.mark.parametrize("hq,hkv,hd", [(8, 2, 128), (6, 2, 64)])
@pytest.mark.parametrize("t", [1, 3, 50])
def test_caps_far_above_the_scores(ctx, cap, opt, hq, hkv, hd, t):
    check(ctx, without_weights(Batch([(t, t), (97, t), (300, t), (1000, t)], hq, hkv, hd, seed=t)), cap=cap, **opt)


@pytest.mark.parametrize("cap", [50.0, 64.0, 65.0, 100.0, 300.0, 1500.0])
@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("t", [1, 40])
def test_caps_that_the_scores_pass(ctx, cap, hd, t):
    """Scores from 0 to several times the cap, of two products each, so that their sums leave little rounding of their own."""
    c = without_weights(Batch([(500, t), (1200, t), (60, t)], 4, 2, hd, seed=31))
    c.q[..., 2:] = 0
    for s in range(3):   # rows' sizes fall, so that many rows compete below the cap, too
        n = c.sizes[s][0]
        r = np.arange(n)
        c.k[c.table[s, r // c.page], r % c.page] *= np.float16(0.1) + (4 * (r / n) ** 4).astype(np.float16)[:, None, None]
    check(ctx, c, scale=cap / 3, cap=cap)


@pytest.mark.parametrize("cap", [64.0, 1e4])
@pytest.mark.parametrize("hq,hkv,hd,q", [(20, 20, 64, "f16"), (20, 20, 64, "f32"), (8, 2, 128, "f32"), (6, 2, 64, "f32")])
def test_caps_in_larger_batches_and_of_f32_queries(ctx, cap, hq, hkv, hd, q):
    check(ctx, without_weights(Batch(MANY, hq, hkv, hd, page=32, q_type=q, seed=33)), cap=cap, bias=4.0)


def test_the_bounds_hold_a_planted_error():
    """(the bounds are tight enough to see a cap of 1e5 lose 2^-22 of its size)"""
    c = Batch([(300, 4)], 2, 1, 64, seed=1)
    _, _, add, adderr = exact(c, 0.125, 1e5)
    k, _ = c.rows(0, 0, c.k)
    x = 0.125 * c.q[:4, 0].astype(np.float64) @ k.T + 2.0 ** -22 * 1e5 * (np.arange(300) % 2)
    live = np.arange(300)[None] <= (296 + np.arange(4))[:, None]
    e = np.where(live, np.exp(x), 0)
    one = (e / e.sum(1, keepdims=True)).sum(0)
    x2 = 0.125 * c.q[:4, 1].astype(np.float64) @ k.T
    e2 = np.where(live, np.exp(x2), 0)
    assert (np.abs(one + (e2 / e2.sum(1, keepdims=True)).sum(0) - add[0, 0]) > adderr[0, 0]).any()


@pytest.mark.parametrize("bias", [1e-45, 1e-38, 1e-3])
@pytest.mark.parametrize("hq,hkv,hd", [(8, 2, 128), (6, 2, 64)])
@pytest.mark.parametrize("t", [1, 50])
def test_smallest_exponents_of_the_slopes(ctx, bias, hq, hkv, hd, t):
    """Slopes near 1 for all heads (max_bias over the number of heads may be 0 in F32: no less a slope)."""
    check(ctx, without_weights(Batch([(t, t), (97, t), (300, t)], hq, hkv, hd, seed=t + 1)), bias=bias)


@pytest.mark.parametrize("hq,hkv,hd", [(8, 2, 128), (5, 5, 64)])
def test_wide_caps_on_cut_walks_with_absent_pages(ctx, hq, hkv, hd):
    absent = [(0, i) for i in (0, 31, 32, 63, 64, 65, 127, 128, 200, 218)] + [(1, i) for i in range(60, 70)]
    check(ctx, without_weights(Batch([(3500, 70), (2100, 150), (40, 3)], hq, hkv, hd, absent=absent, seed=34)), cap=2e3, bias=2.0)
    check(ctx, without_weights(Batch([(3500, 1), (2100, 1), (40, 1)], hq, hkv, hd, absent=absent, seed=35)), cap=2e3)
