"""Choices of blocks by bounds alone, without a pool of keys: batches as large as the search's kernels
need, a plain implementation in 64 bits, the call on the GPU."""
from __future__ import annotations

import numpy as np


def exponents(x):
    """Elementwise the least e from -64 to 64 with x <= 127 2^e (NaN: as -64)."""
    m, e = np.frexp(np.where(np.isfinite(x), x, 0.0))
    e = np.where(m > 0, e - 7 + (m > 127.0 / 128.0), -64)
    return np.where(np.isposinf(x), 64, np.clip(e, -64, 64)).astype(np.int64)


# Calls that a team of 16 wavefronts searches (blocks of a tile's tokens beyond 512, 128 workgroups and more, so that
# they are not cut), that are cut beyond 4096 blocks, and whose join has more pairs than a wavefront holds. With what they
# have to launch: threads of the first kernel, blocks and number of its segments, wavefronts of the join (0: none).
def _streams(rows, t=1, n=16):
    return [(rows, t)] * n


LONG = {
    "513_blocks": (dict(sizes=_streams(513 * 16), top=8), (1024, 528, 1, 0)),
    "600_blocks_sinks": (dict(sizes=_streams(600 * 16 - 7), top=64, n_sink=2, n_recent=3, absent=0.1), (1024, 608, 1, 0)),
    "700_blocks_all": (dict(sizes=_streams(700 * 16), top=1024), (1024, 704, 1, 0)),
    "1030_blocks_ties": (dict(sizes=_streams(1030 * 16 + 5), top=100, few=3), (1024, 1040, 1, 0)),
    "1030_blocks_of_128": (dict(sizes=_streams(1030 * 16), hd=128, top=33, n_sink=1), (1024, 1040, 1, 0)),
    "4096_blocks": (dict(sizes=_streams(4096 * 16), top=1024, n_sink=4, n_recent=4), (1024, 4096, 1, 0)),
    "4096_blocks_one_score": (dict(sizes=_streams(4096 * 16), top=7, few=1, n_recent=1), (1024, 4096, 1, 0)),
    "ragged_4096_blocks": (dict(sizes=[(1 + 4096 * s, 1) for s in range(17)], top=48, n_sink=1, n_recent=2, absent=0.05), (1024, 2064, 2, 1)),
    "window_of_many": (dict(sizes=_streams(4000 * 16 + 3), top=65, n_sink=3, window=20000), (1024, 1264, 1, 0)),
    "groups_in_passes": (dict(sizes=_streams(800 * 16), hq=160, top=20, n_sink=1), (1024, 800, 1, 0)),
    "two_tokens": (dict(sizes=_streams(1500 * 16, 2, 16), hq=64, top=40, n_sink=1, n_recent=1), (1024, 1504, 1, 0)),
    "three_tokens_of_four": (dict(sizes=_streams(700 * 16, 3) + [(900 * 16, 4)], hq=32, top=30, n_recent=2, absent=0.1), (1024, 912, 1, 0)),
    "four_tokens_64_kib": (dict(sizes=_streams(4096 * 16, 4), hq=32, top=50, n_sink=1, n_recent=2), (1024, 4096, 1, 0)),
    "sixteen_tokens_64_kib": (dict(sizes=_streams(1024 * 16, 16), top=12, few=40), (1024, 1024, 1, 0)),
    "two_segments": (dict(sizes=_streams(4097 * 16), top=33, n_sink=1, n_recent=2), (1024, 2064, 2, 1)),
    "three_segments_1800_pairs": (dict(sizes=_streams(9000 * 16), top=600, n_sink=1, absent=0.05), (1024, 3008, 3, 16)),
    "three_segments_ties": (dict(sizes=_streams(9000 * 16), top=700, few=5), (1024, 3008, 3, 16)),
    "5120_pairs": (dict(sizes=_streams(20000 * 16, 1, 2), hq=2, hkv=2, top=1024, n_sink=3, n_recent=5), (1024, 4000, 5, 16)),
    "17408_pairs": (dict(sizes=_streams(69000 * 16, 1, 1), hq=2, hkv=1, top=1024, n_sink=3, n_recent=5, absent=0.05), (1024, 4064, 17, 16)),
    "17408_pairs_ties": (dict(sizes=_streams(69000 * 16, 1, 1), hq=1, hkv=1, top=1024, few=4), (1024, 4064, 17, 16)),
}


def long_choice(name, **kw):
    return Choice(**{**dict(hq=8, hkv=8, hd=64, page=4096, block=16, n_sink=0, n_recent=0), **LONG[name][0], **kw})


class Choice:
    """sizes: (rows, new tokens) per stream. Bounds [page][head][block][2 D] with scales, whose pages all streams share
    (any page may be the next). few: so many distinct scores at most."""

    def __init__(self, sizes, hq, hkv, hd, page, block, top, n_sink=0, n_recent=0, window=0, pages=16, few=0, absent=0.0, seed=0, max_nkv=0, max_nq=0):
        rng = np.random.default_rng(seed)
        self.sizes, self.hq, self.hkv, self.hd, self.page, self.block = sizes, hq, hkv, hd, page, block
        self.top, self.n_sink, self.n_recent, self.window, self.n_pages = top, n_sink, n_recent, window, pages
        self.B, self.T, self.max_nkv = len(sizes), sum(t for _, t in sizes), max_nkv
        self.max_nq = max_nq or max(t for _, t in sizes)
        self.n_kv = np.array([n for n, _ in sizes], np.int32)
        self.q_start = np.concatenate([[0], np.cumsum([t for _, t in sizes])]).astype(np.int32)
        self.max_pages = max(-(-max(n, max_nkv) // page) for n, _ in sizes)
        self.table = rng.integers(0, pages, (self.B, self.max_pages)).astype(np.int32)
        self.table[rng.random(self.table.shape) < absent] = -1
        n = page // block
        if few:
            some = rng.integers(-127, 128, (few, 2 * hd)).astype(np.int8)
            self.b = some[rng.integers(0, few, (pages, hkv, n))]
            self.bs = np.full((pages, hkv, n), 0.5, np.float32)
        else:
            self.b = rng.integers(-127, 128, (pages, hkv, n, 2 * hd)).astype(np.int8)
            self.bs = (2.0 ** rng.integers(-3, 3, (pages, hkv, n))).astype(np.float32)
        self.q = rng.standard_normal((self.T, hq, hd)).astype(np.float16)

    def want(self):
        """Lists [T][hkv][top], from the formula."""
        out = np.full((self.T, self.hkv, self.top), -1, np.int32)
        G, bl = self.hq // self.hkv, self.block
        with np.errstate(invalid="ignore"):
            scale = np.clip(np.nan_to_num(self.bs.astype(np.float64), nan=2.0 ** -64, posinf=2.0 ** 64, neginf=2.0 ** -64), 2.0 ** -64, 2.0 ** 64)
        hi, lo = self.b[..., :self.hd].astype(np.float64), self.b[..., self.hd:].astype(np.float64)
        # (whole numbers below 2^22: products and sums are exact in 64 bits, in any order)
        for s, (n, t) in enumerate(self.sizes):
            for i in range(t):
                p = n - t + i
                if p < 0:
                    continue
                low, last = (max(p - self.window + 1, 0) // bl if self.window else 0), p // bl
                j = np.arange(low, last + 1)
                page, at = self.table[s, j * bl // self.page], j * bl % self.page // bl
                there = (page >= 0) & (page < self.n_pages)
                ends = (j < low + self.n_sink) | (j > last - self.n_recent)
                for h in range(self.hkv):
                    score = np.full(hi.shape[0:1] + hi.shape[2:3], -np.inf)
                    for g in range(h * G, (h + 1) * G):
                        q = self.q[self.q_start[s] + i, g].astype(np.float64)
                        f = exponents(np.abs(q).max())
                        with np.errstate(invalid="ignore"):
                            r = np.clip(np.rint(q / 2.0 ** f), -127, 127)
                        score = np.maximum(score, (hi[:, h] @ np.maximum(r, 0) + lo[:, h] @ np.minimum(r, 0)) * 2.0 ** f)
                    mine = np.where(there, score[np.where(there, page, 0), at] * scale[np.where(there, page, 0), h, at], -np.inf)
                    mine = np.where(ends, np.inf, mine)
                    best = np.argsort(-mine, kind="stable")[:self.top]
                    got = j[np.sort(best[mine[best] > -np.inf])]
                    out[self.q_start[s] + i, h, :len(got)] = got
        return out

    def place(self):
        """The call's buffers on the GPU and its arguments."""
        from conftest import load_package
        from gpu_util import guarded, vxfa
        views = load_package().views
        self.host = dict(q=self.q, b=self.b, bs=self.bs, table=self.table, n_kv=self.n_kv, q_start=self.q_start,
                         list=np.full((self.T, self.hkv, self.top), -7, np.int32))
        d = self.dev = {k: guarded(x) for k, x in self.host.items()}
        return (vxfa.desc(d["q"].data_ptr(), vxfa.F16, *views.decoder_q(self.T, self.hq, self.hd, 2)),
                vxfa.desc(d["b"].data_ptr(), vxfa.I8, *views.bound_pages(self.n_pages, self.page, self.hkv, self.hd, self.block)),
                vxfa.desc(d["bs"].data_ptr(), vxfa.F32, *views.scale_pages(self.n_pages, self.page, self.hkv, self.block)),
                vxfa.paged(d["table"].data_ptr(), d["n_kv"].data_ptr(), d["q_start"].data_ptr(), self.B, self.max_pages, self.max_nq,
                           self.max_nkv, self.window),
                vxfa.blocks(d["list"].data_ptr(), self.block, self.top, self.n_sink, self.n_recent))

    def got(self):
        """Lists as the GPU chose them, [T][hkv][top], checked for writes outside the buffers."""
        import torch
        from gpu_util import guards_intact
        torch.cuda.synchronize()
        for k, t in self.dev.items():
            assert guards_intact(t), f"write outside {k}"
            if k != "list":
                assert (t.cpu().numpy() == np.ascontiguousarray(self.host[k]).view(np.uint8).reshape(-1)).all(), f"{k} written"
        return self.dev["list"].cpu().numpy().view(np.int32).reshape(self.T, self.hkv, self.top)

    def check(self, ctx, stream):
        ctx.paged_select(*self.place(), stream=stream)
        self.same()

    def same(self):
        want, got = self.want(), self.got()
        bad = np.argwhere((got != want).any(-1))
        assert len(bad) == 0, f"{len(bad)} lists, first {bad[0]}: {got[tuple(bad[0])]} for {want[tuple(bad[0])]}"
