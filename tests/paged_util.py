"""The paged entry points against a plain implementation in 64 bits: batches of
streams over a pool of pages, the reference, error bounds, GPU calls.

Everything that a call has no business with holds NaN: pages of no stream,
rows past a stream's end, tokens behind the last stream. Outputs lie
between canaries."""
from __future__ import annotations

import math

import numpy as np

HALF = 2.0 ** -11   # half a step of f16, relative
NAN16 = np.uint16(0x7E00)


class Batch:
    """sizes: (rows, new tokens) per stream. layout: "row" ([page][row][head],
    as the token-major cache) or "head" ([page][head][row], rows padded by 16
    bytes). absent: (stream, page index) pairs whose table entry is -1."""

    def __init__(self, sizes, hq=8, hkv=2, hd=128, page=16, layout="row", absent=(), q_type="f16", behind=0,
                 kv_scale=1.0, q_scale=1.0, seed=0, spare=3, max_nkv=0):
        rng = np.random.default_rng(seed)
        self.sizes, self.hq, self.hkv, self.hd, self.page, self.layout = list(sizes), hq, hkv, hd, page, layout
        self.B, self.T = len(sizes), sum(t for _, t in sizes)
        self.q_type, self.behind = q_type, behind
        self.n_kv = np.array([n for n, _ in sizes], np.int32)
        self.q_start = np.concatenate([[0], np.cumsum([t for _, t in sizes])]).astype(np.int32)
        need = [-(-n // page) for n, _ in sizes]
        self.max_pages = max(need + [1]) + 1
        self.max_nkv = max_nkv
        self.n_pages = sum(need) + spare
        ids = rng.permutation(self.n_pages).astype(np.int32)
        self.table = np.full((self.B, self.max_pages), -1, np.int32)
        at = 0
        for s, m in enumerate(need):
            self.table[s, :m] = ids[at:at + m]
            at += m
        self.free = ids[at:]
        # logical pools [page][row][head][D], NaN but for live rows
        self.k = np.full((self.n_pages, page, hkv, hd), NAN16, np.uint16).view(np.float16)
        self.v = self.k.copy()
        self.w = np.full((self.n_pages, hkv, page), np.nan, np.float32)
        for s, (n, _) in enumerate(sizes):
            r = np.arange(n)
            p = self.table[s, r // page]
            self.k[p, r % page] = (kv_scale * rng.standard_normal((n, hkv, hd))).astype(np.float16)
            self.v[p, r % page] = rng.standard_normal((n, hkv, hd)).astype(np.float16)
            self.w[p, :, r % page] = 4 * rng.random((n, hkv), dtype=np.float32) ** 8
        for s, i in absent:
            p = self.table[s, i]
            self.k[p] = np.float16(np.nan)
            self.v[p] = np.float16(np.nan)
            self.w[p] = np.nan
            self.table[s, i] = (-1, self.n_pages, 2 ** 31 - 1, -2 ** 31)[i % 4]
        q = (q_scale * rng.standard_normal((self.T + behind, hq, hd))).astype(np.float16 if q_type == "f16" else np.float32)
        q[self.T:] = np.nan
        self.q = q

    @property
    def max_nq(self):
        return max([t for _, t in self.sizes] + [0])

    def rows(self, s, h, pool):
        """[n, D] of a stream's head in 64 bits, and which rows are there."""
        n = self.sizes[s][0]
        r = np.arange(n)
        p = self.table[s, r // self.page].astype(np.int64)
        there = (p >= 0) & (p < self.n_pages)
        x = pool[np.where(there, p, 0), r % self.page, h].astype(np.float64)
        return np.where(there[:, None], x, 0.0), there


def slopes(hq, max_bias):
    """ggml's: n the largest power of two in hq."""
    if not max_bias:
        return [0.0] * hq
    n = 2 ** int(math.log2(hq))
    return [2.0 ** (-max_bias * (h + 1) / n) if h < n else 2.0 ** (-max_bias / 2 * (2 * (h - n) + 1) / n) for h in range(hq)]


def reference(c, scale, window=0, cap=0.0, bias=0.0):
    """Outputs [T, hq, D], weights added to each row {(stream, kv head): [n]}, and
    bounds on the errors of both.

    The bounds, of a row with weights P (sum 1) and N of them. dx: how far a
    score may be off: F32 sums of D exact products (each of D steps rounds by
    half a step, 2^-24, of at most S = scale sum |q_d k_d|), the roundings of
    scores up to X (2^-22 X: scaling, distance term and subtraction of the
    maximum, each in F32), the cap's absolute error (2^-22 cap) and, where q
    is F32, its rounding to f16 (2^-11 S). A weight is off by the factor
    exp(2 dx) - 1 < 3 dx (its own score and those of the sum). P is rounded to f16
    before the second product: half a step, 2^-11, or 2^-25 of the row's
    largest weight where f16 is subnormal. So
      |do| <= (2^-11 + 3 dx) sum P |v| + 2^-25 max P N max |v|, twice (the sum
              of the weights is taken of rounded ones or not)
      |dw| <= w (3 dx + 2^-24 (N + rows)) + 2^-126 a token and head (a weight
              below F32's smallest normal number, 2^-126, may be 0)."""
    G, D = c.hq // c.hkv, c.hd
    out = np.zeros((c.T, c.hq, D))
    err = np.zeros_like(out)
    add, adderr = {}, {}
    sl = slopes(c.hq, bias)
    for s, (n, t) in enumerate(c.sizes):
        for h in range(c.hkv):
            add[s, h], adderr[s, h] = np.zeros(n), np.zeros(n)
            k, there = c.rows(s, h, c.k)
            v, _ = c.rows(s, h, c.v)
            j = np.arange(n)
            for g in range(h * G, (h + 1) * G):
                q = c.q[c.q_start[s]:c.q_start[s] + t, g].astype(np.float64)
                x = scale * (q @ k.T)
                S = abs(scale) * (np.abs(q) @ np.abs(k).T)
                if cap:
                    x = cap * np.tanh(x / cap)
                p = n - t + np.arange(t)
                x = x + sl[g] * (j[None] - p[:, None])
                live = (j[None] <= p[:, None]) & there[None]
                if window:
                    live &= j[None] > p[:, None] - window
                x = np.where(live, x, -np.inf)
                m = np.maximum(x.max(1, initial=-np.inf), -1e300)[:, None]
                e = np.exp(x - m)
                l = e.sum(1, keepdims=True)
                P = e / np.where(l > 0, l, 1)
                o = P @ v
                at = slice(c.q_start[s], c.q_start[s] + t)
                out[at, g] = o
                Smax = np.where(live, S, 0).max(1, initial=0)
                # (scores that matter lie within 40 of the maximum)
                X = np.where(live & (x > m - 40), np.abs(x) + np.abs(x - m), 0).max(1, initial=0)
                dx = 2.0 ** -24 * D * Smax + 2.0 ** -22 * (X + cap) + (HALF * Smax if c.q_type == "f32" else 0)
                N = live.sum(1)
                vmax = np.abs(v).max(initial=0)
                err[at, g] = 2 * ((HALF + 3 * dx)[:, None] * (P @ np.abs(v))
                                  + (2.0 ** -25 * P.max(1, initial=0) * N * vmax)[:, None])
                add[s, h] += P.sum(0)
                adderr[s, h] += (P * (3 * dx + 2.0 ** -24 * (N + t * G))[:, None]).sum(0) + t * 2.0 ** -126
    return out, add, err, adderr


# ---- on the GPU ------------------------------------------------------------------

CANARY = 1024


class Device:
    """A batch's buffers on the GPU and its descriptors."""

    def __init__(self, c, dst_type="f16", window=0):
        import torch
        from gpu_util import vxfa, guarded
        self.c, self.vxfa, self.torch = c, vxfa, torch
        views = __import__("conftest").load_package().views
        self.pools = {}
        for name in "kv":
            x = getattr(c, name)
            if c.layout == "head":   # [page][head][row] with 16 bytes between rows
                x = np.concatenate([x, np.full(x.shape[:3] + (8,), NAN16, np.uint16).view(np.float16)], -1).transpose(0, 2, 1, 3)
                r = (c.hd + 8) * 2
                nb = (2, r, c.page * r, c.hkv * c.page * r)
            else:
                nb = views.kv_pages(c.n_pages, c.page, c.hkv, c.hd)[1]
            t = guarded(np.ascontiguousarray(x))
            self.pools[name] = (t, vxfa.desc(t.data_ptr(), vxfa.F16, (c.hd, c.page, c.hkv, c.n_pages), nb))
        self.k, self.v = self.pools["k"][1], self.pools["v"][1]
        self.wt = guarded(c.w)
        self.w = vxfa.desc(self.wt.data_ptr(), vxfa.F32, *views.weight_pages(c.n_pages, c.page, c.hkv))
        self.qt = guarded(c.q)
        n = c.T + c.behind
        self.q = vxfa.desc(self.qt.data_ptr(), vxfa.F16 if c.q_type == "f16" else vxfa.F32,
                           *views.decoder_q(n, c.hq, c.hd, c.q.itemsize))
        self.dst_np = np.float16 if dst_type == "f16" else np.float32
        e = np.dtype(self.dst_np).itemsize
        self.dst_bytes = n * c.hq * c.hd * e
        self.dt = torch.full((self.dst_bytes + 2 * CANARY,), 0xA5, dtype=torch.uint8, device="cuda")
        self.dst = vxfa.desc(self.dt.data_ptr() + CANARY, vxfa.F16 if dst_type == "f16" else vxfa.F32,
                             *views.dst(c.hd, c.hq, n, elt=e))
        self.table, self.n_kv, self.q_start = (guarded(x) for x in (c.table, c.n_kv, c.q_start))
        self.batch = vxfa.paged(self.table.data_ptr(), self.n_kv.data_ptr(), self.q_start.data_ptr(), c.B, c.max_pages,
                                c.max_nq, c.max_nkv, window)

    def out(self):
        """dst [T, hq, D], its canaries and the tokens behind checked."""
        c = self.c
        raw = self.dt.cpu().numpy()
        assert (raw[:CANARY] == 0xA5).all() and (raw[CANARY + self.dst_bytes:] == 0xA5).all(), "write outside dst"
        x = raw[CANARY:CANARY + self.dst_bytes].reshape(c.T + c.behind, -1)
        assert (x[c.T:] == 0xA5).all(), "write behind the last stream"
        return x[:c.T].copy().view(self.dst_np).reshape(c.T, c.hq, c.hd)

    def pool(self, name):
        """The pool as [page][row][head][D]."""
        c = self.c
        x = self.pools[name][0].cpu().numpy().view(np.float16)
        if c.layout == "head":
            return x.reshape(c.n_pages, c.hkv, c.page, c.hd + 8)[..., :c.hd].transpose(0, 2, 1, 3)
        return x.reshape(c.n_pages, c.page, c.hkv, c.hd)

    def weights(self, t=None):
        c = self.c
        return (self.wt if t is None else t).cpu().numpy().view(np.float32).reshape(c.n_pages, c.hkv, c.page)

    def check_guards(self):
        from gpu_util import guards_intact
        for t in (self.pools["k"][0], self.pools["v"][0], self.wt, self.qt, self.table, self.n_kv, self.q_start):
            assert guards_intact(t), "write outside a buffer"


def check_out(got, want, err, half_dst):
    assert np.isfinite(got).all(), "not finite"
    tol = err + (HALF if half_dst else 2.0 ** -24) * np.abs(want) * 1.01 + 1e-30
    if half_dst:
        tol = tol + 2.0 ** -25
    bad = np.abs(got.astype(np.float64) - want) > tol
    assert not bad.any(), (f"{bad.sum()} of {bad.size} outside, worst {np.abs(got - want)[bad].max():.3g} against "
                           f"{tol[bad].min():.3g}, first at {np.argwhere(bad)[0]}")


def check_weights(c, got, base, add, adderr, before):
    """got: the weights tensor afterwards; base: what the sums went on top of; before: what it held."""
    want, tol = before.astype(np.float64).copy(), np.zeros(before.shape)
    for s, (n, _) in enumerate(c.sizes):
        r = np.arange(n)
        p = c.table[s, r // c.page].astype(np.int64)
        ok = (p >= 0) & (p < c.n_pages)
        for h in range(c.hkv):
            old = base[p[ok], h, r[ok] % c.page] if base is not None else 0.0
            want[p[ok], h, r[ok] % c.page] = old + add[s, h][ok]
            tol[p[ok], h, r[ok] % c.page] = adderr[s, h][ok] + 2.0 ** -23 * np.abs(old + add[s, h][ok])
    same = np.isnan(want) & np.isnan(got)
    bad = ~same & ~(np.abs(got - want) <= tol)
    assert not bad.any(), f"{bad.sum()} weights outside, first at {np.argwhere(bad)[0]}: {got[bad][0]} for {want[bad][0]}"
