"""Pages of 8 bits, bounds of blocks and chosen blocks against a plain implementation in
64 bits: batches, references with error bounds, buffers on the GPU.

What no token sees holds what would show if it took part: in pages of 8 bits scales that
are NaN, infinite, negative or 0 wherever no row of a stream lies and any whole numbers behind
a stream's last row, in F16 pages NaN."""
from __future__ import annotations

import math

import numpy as np

import paged_util
from paged_util import HALF, slopes

BAD = np.array([np.nan, np.inf, -np.inf, 0.0, -1.0, 3.0e38, 1.0e-44], np.float32)


def exponent(x):
    """The least e from -64 to 64 with x <= 127 2^e."""
    e = -64
    while e < 64 and x > 127.0 * 2.0 ** e:
        e += 1
    return e


class Batch8(paged_util.Batch):
    """A batch (paged_util.Batch) whose pool holds whole numbers of 8 bits: k, v int8, scales ks, vs
    [page][head][16 rows]. spread: exponents of the scales of V lie that far apart."""

    def __init__(self, sizes, hq=8, hkv=2, hd=128, page=16, spread=3, absent=(), seed=0, powers=True, **kw):
        super().__init__(sizes, hq, hkv, hd, page, absent=absent, seed=seed, **kw)
        rng = np.random.default_rng(seed + 1000)
        shape = self.k.shape
        self.k = rng.integers(-128, 128, shape).astype(np.int8)
        self.v = rng.integers(-128, 128, shape).astype(np.int8)
        n = page // 16
        self.ks = BAD[rng.integers(0, len(BAD), (self.n_pages, hkv, n))]
        self.vs = BAD[rng.integers(0, len(BAD), (self.n_pages, hkv, n))]
        for s, (rows, _) in enumerate(self.sizes):
            r = np.arange(rows)
            p = self.table[s, r // page].astype(np.int64)
            ok = (p >= 0) & (p < self.n_pages)
            p, r = p[ok], r[ok]
            for x in (self.k, self.v):
                x[p, r % page] = np.clip(np.rint(32 * rng.standard_normal((len(r), hkv, hd))), -127, 127)
            for x, e in ((self.ks, rng.integers(-6, -4, (len(r), hkv))), (self.vs, rng.integers(-5 - spread, -4, (len(r), hkv)))):
                f = 2.0 ** e if powers else 2.0 ** (e + rng.random(e.shape))
                x[p, :, r % page // 16] = f

    def rows(self, s, h, pool):
        n = self.sizes[s][0]
        r = np.arange(n)
        p = self.table[s, r // self.page].astype(np.int64)
        there = (p >= 0) & (p < self.n_pages)
        p = np.where(there, p, 0)
        scale = (self.ks if pool is self.k else self.vs)[p, h, r % self.page // 16].astype(np.float64)
        with np.errstate(invalid="ignore"):     # (rows of absent pages; a line below)
            x = pool[p, r % self.page, h] * scale[:, None]
        return np.where(there[:, None], x, 0.0), there


def reference(c, scale, window=0, cap=0.0, bias=0.0, lists=None, block=16):
    """Outputs [T, hq, D] and bounds on their errors; lists [T][hkv][top]: over chosen blocks only.

    The bounds are those of paged_util.reference with, for 8 bits, what differs: the products with
    K's whole numbers are of D steps in F32 as there, the scale's multiplication one rounding more
    (2^-24 of the score) and the logarithm of V's scale, up to 64 and rounded to F32 as the sum with it
    is: 2^-22 (64 + X). Weights P s are rounded to f16: half a step relative, or 2^-25 of the largest P s
    where f16 is subnormal, times whole numbers of up to 127. A reciprocal and a product (2^-22) in
    the sum's terms."""
    G, D, i8 = c.hq // c.hkv, c.hd, isinstance(c, Batch8)
    out = np.zeros((c.T, c.hq, D))
    err = np.zeros_like(out)
    sl = slopes(c.hq, bias)
    for s, (n, t) in enumerate(c.sizes):
        for h in range(c.hkv):
            k, there = c.rows(s, h, c.k)
            v, _ = c.rows(s, h, c.v)
            j = np.arange(n)
            at = slice(c.q_start[s], c.q_start[s] + t)
            times = np.ones((t, n))
            if lists is not None:
                times[:] = 0
                for i in range(t):
                    for b in lists[c.q_start[s] + i, h]:
                        if b >= 0:
                            times[i, b * block:(b + 1) * block] += 1
            for g in range(h * G, (h + 1) * G):
                q = c.q[at, g].astype(np.float64)
                x = scale * (q @ k.T)
                S = abs(scale) * (np.abs(q) @ np.abs(k).T)
                if cap:
                    x = cap * np.tanh(x / cap)
                p = n - t + np.arange(t)
                x = x + sl[g] * (j[None] - p[:, None])
                live = (j[None] <= p[:, None]) & there[None] & (times > 0)
                if window:
                    live &= j[None] > p[:, None] - window
                x = np.where(live, x, -np.inf)
                m = np.maximum(x.max(1, initial=-np.inf), -1e300)[:, None]
                e = np.exp(x - m) * times
                l = e.sum(1, keepdims=True)
                P = e / np.where(l > 0, l, 1)
                out[at, g] = P @ v
                Smax = np.where(live, S, 0).max(1, initial=0)
                X = np.where(live & (x > m - 40), np.abs(x) + np.abs(x - m), 0).max(1, initial=0)
                dx = 2.0 ** -24 * D * Smax + 2.0 ** -22 * (X + cap) + (HALF * Smax if c.q_type == "f32" else 0)
                N = times.sum(1)
                big = P.max(1, initial=0) * np.abs(v).max(initial=0)
                if i8:
                    dx = dx + 2.0 ** -24 * Smax + 2.0 ** -22 * (64 + X) + 2.0 ** -22
                    # (largest P s: of a row's largest whole number at least 1, if it is not all 0)
                    r = np.arange(n)
                    pg = np.clip(c.table[s, r // c.page], 0, c.n_pages - 1)
                    sv = np.where(there, c.vs[pg, h, r % c.page // 16], 0).astype(np.float64)
                    big = (P * sv[None]).max(1, initial=0) * 127
                err[at, g] = 2 * ((HALF + 3 * dx)[:, None] * (P @ np.abs(v)) + (2.0 ** -25 * big * N)[:, None])
    return out, err


# ---- appends, bounds and the choice, exactly ---------------------------------------


def append(c, ints, scales, new):
    """The pools (copies) after new [T, hkv, D] (F32) of the batch's tokens were stored in them."""
    ints, scales = ints.copy(), scales.copy()
    for s, (n, t) in enumerate(c.sizes):
        for b in range(max(n - t, 0) // 16, -(-n // 16)):
            page = c.table[s, b * 16 // c.page]
            if not 0 <= page < c.n_pages:
                continue
            i, r = b * 16 % c.page // 16, b * 16 % c.page
            r0, r1 = max(n - t - 16 * b, 0), min(n - 16 * b, 16)
            x = new[c.q_start[s] + 16 * b + r0 - (n - t):c.q_start[s] + 16 * b + r1 - (n - t)].astype(np.float64)
            for h in range(c.hkv):
                y = x[:, h]
                e = exponent(np.nanmax(np.abs(y), initial=0.0))
                if r0 > 0:
                    was = int(math.log2(scales[page, h, i]))
                    e = max(e, was)
                    ints[page, r:r + r0, h] = np.rint(ints[page, r:r + r0, h] * 2.0 ** (was - e))
                z = np.clip(np.rint(y / 2.0 ** e), -127, 127)
                ints[page, r + r0:r + r1, h] = np.where(np.isnan(y), 0, z)
                scales[page, h, i] = 2.0 ** e
    return ints, scales


def bounds(c, block, b, bs):
    """Bounds [page][head][block][2 D] and their scales (copies) with those of the new tokens' blocks."""
    b, bs = b.copy(), bs.copy()
    for s, (n, t) in enumerate(c.sizes):
        if t == 0:
            continue
        for i in range(max(n - t, 0) // block, -(-n // block)):
            page = c.table[s, i * block // c.page]
            if not 0 <= page < c.n_pages:
                continue
            for h in range(c.hkv):
                k = c.rows(s, h, c.k)[0][i * block:(i + 1) * block]
                e = exponent(np.abs(k).max())
                at = i * block % c.page // block
                b[page, h, at, :c.hd], b[page, h, at, c.hd:] = np.ceil(k.max(0) / 2.0 ** e), np.floor(k.min(0) / 2.0 ** e)
                bs[page, h, at] = 2.0 ** e
    return b, bs


def select(c, block, b, bs, top, n_sink, n_recent, window=0):
    """Lists [T][hkv][top]."""
    out = np.full((c.T, c.hkv, top), -1, np.int32)
    G = c.hq // c.hkv
    for s, (n, t) in enumerate(c.sizes):
        for i in range(t):
            p = n - t + i
            if p < 0:
                continue
            low, last = max(p - window + 1, 0) // block if window else 0, p // block
            j = np.arange(low, last + 1)
            page = c.table[s, j * block // c.page].astype(np.int64)
            there = (page >= 0) & (page < c.n_pages)
            page, at = np.where(there, page, 0), j * block % c.page // block
            ends = (j < low + n_sink) | (j > last - n_recent)
            for h in range(c.hkv):
                score = np.full(len(j), -np.inf)
                hi, lo = b[page, h, at, :c.hd].astype(np.int64), b[page, h, at, c.hd:].astype(np.int64)
                for g in range(h * G, (h + 1) * G):
                    q = c.q[c.q_start[s] + i, g].astype(np.float16).astype(np.float64)
                    f = exponent(np.abs(q).max())
                    r = np.rint(q / 2.0 ** f).astype(np.int64)
                    score = np.maximum(score, np.where(r > 0, r * hi, r * lo).sum(1) * 2.0 ** f * np.where(there, bs[page, h, at], 1))
                order = sorted(range(len(j)), key=lambda y: (not ends[y], -score[y] if not ends[y] else 0, y))
                order = [y for y in order if ends[y] or there[y]][:top]
                got = sorted(j[y] for y in order)
                out[c.q_start[s] + i, h, :len(got)] = got
    return out


# ---- on the GPU ------------------------------------------------------------------


class Device8(paged_util.Device):
    """paged_util.Device, with a pool of 8 bits and its scales where the batch has one, and bounds."""

    def __init__(self, c, dst_type="f16", window=0, block=16):
        from gpu_util import guarded, vxfa
        i8 = isinstance(c, Batch8)
        keep = c.k, c.v
        if i8:      # (the base class takes F16 pools; they are replaced below)
            c.k, c.v = (np.zeros(c.k.shape, np.float16) for _ in "kv")
        super().__init__(c, dst_type, window)
        c.k, c.v = keep
        views = __import__("conftest").load_package().views
        self.views = views
        self.ks = self.vs = None
        if i8:
            self.scales = {}
            for name in "kv":
                x = getattr(c, name)
                nb = views.kv_pages(c.n_pages, c.page, c.hkv, c.hd, 1)[1]
                if c.layout == "head":   # [page][head][row] with 16 bytes between rows
                    x = np.concatenate([x, np.full(x.shape[:3] + (16,), 77, np.int8)], -1).transpose(0, 2, 1, 3)
                    r = c.hd + 16
                    nb = (1, r, c.page * r, c.hkv * c.page * r)
                t = guarded(np.ascontiguousarray(x))
                self.pools[name] = (t, vxfa.desc(t.data_ptr(), vxfa.I8, (c.hd, c.page, c.hkv, c.n_pages), nb))
                z = guarded(getattr(c, name + "s"))
                self.scales[name] = (z, vxfa.desc(z.data_ptr(), vxfa.F32, *views.scale_pages(c.n_pages, c.page, c.hkv)))
            self.k, self.v = self.pools["k"][1], self.pools["v"][1]
            self.ks, self.vs = self.scales["k"][1], self.scales["v"][1]
        n = c.page // block
        self.b_np = np.full((c.n_pages, c.hkv, n, 2 * c.hd), 99, np.int8)
        self.bs_np = np.full((c.n_pages, c.hkv, n), 7.0, np.float32)
        self.set_bounds(self.b_np, self.bs_np, block)

    def set_bounds(self, b, bs, block):
        from gpu_util import guarded
        c, vxfa = self.c, self.vxfa
        self.block = block
        self.bt, self.bst = guarded(b), guarded(bs)
        self.b = vxfa.desc(self.bt.data_ptr(), vxfa.I8, *self.views.bound_pages(c.n_pages, c.page, c.hkv, c.hd, block))
        self.bs = vxfa.desc(self.bst.data_ptr(), vxfa.F32, *self.views.scale_pages(c.n_pages, c.page, c.hkv, block))

    def set_list(self, lists, block, n_sink=0, n_recent=0):
        from gpu_util import guarded
        self.lt = guarded(lists)
        self.list_shape = lists.shape
        self.blocks = self.vxfa.blocks(self.lt.data_ptr(), block, lists.shape[2], n_sink, n_recent)

    def list(self):
        return self.lt.cpu().numpy().view(np.int32).reshape(self.list_shape)

    def ints(self, name):
        c = self.c
        x = self.pools[name][0].cpu().numpy().view(np.int8)
        if c.layout == "head":
            x = x.reshape(c.n_pages, c.hkv, c.page, c.hd + 16)
            assert (x[..., c.hd:] == 77).all(), "write between rows"
            return x[..., :c.hd].transpose(0, 2, 1, 3)
        return x.reshape(c.n_pages, c.page, c.hkv, c.hd)

    def scale(self, name):
        return self.scales[name][0].cpu().numpy().view(np.float32).reshape(self.c.ks.shape)

    def bounds(self):
        return (self.bt.cpu().numpy().view(np.int8).reshape(self.c.n_pages, self.c.hkv, -1, 2 * self.c.hd),
                self.bst.cpu().numpy().view(np.float32).reshape(self.c.n_pages, self.c.hkv, -1))

    def check_guards(self):
        from gpu_util import guards_intact
        super().check_guards()
        more = [self.bt, self.bst] + ([self.lt] if hasattr(self, "lt") else [])
        if self.ks is not None:
            more += [self.scales[n][0] for n in "kv"]
        for t in more:
            assert guards_intact(t), "write outside a buffer"
