"""A paged K/V cache of 8 bits, and attention over chosen blocks of a cache: the calls, their inputs, one pass of each, their answers.

A cache is a pool of pages of `page` rows; a stream's rows lie in the pages
that its line of a table names (-1: none), in order. A call takes a batch of
streams, each with its number of rows and a chunk of new tokens, which are its
last rows; the tokens of all streams are packed one after another.

In a pool of 8 bits each 16 rows of a kv head have a scale for K and one for V,
powers of two: a value is the scale times a whole number from -127 to 127. The
scale of rows is the least power of two (2^-64 at least, 2^64 at most) that leaves their
largest value within 127 of it.

  op        "append": the new rows stored in their pages, keys and queries rotated; the scale of
            a block that holds rows already grows where it has to, and those are rounded again.
            "attend": attention of the new tokens over their streams' rows.
            "bounds": of the blocks with new rows the largest and smallest key of each dim, as whole numbers of 8 bits
            (rounded up and down) times a power of two. "select": `top` blocks of the rows that a token sees, for each
            token and kv head: the first `sink`, the last `recent`, and the others by a bound on their keys' products with
            the queries, rounded to 8 bits each. "blocks": attention over such blocks alone
  bits      8 or 16: the pool's ("bounds" and "blocks" take F16 pools, too)
  hq hkv hd query heads, kv heads, head dim
  streams, nq, kv   streams, most new tokens and most rows of one
  ragged    the streams' rows lie between a sixteenth of kv and kv (else all
            have kv), and with nq > 1 about half of them have a single new
            token, the others up to nq (else all have nq)
  window    > 0: a token attends the last `window` rows up to its own
  cap, bias the score cap (0: none) and the largest exponent of the heads' distance slopes (0: none)
  block top sink recent   rows of a block, blocks chosen, the first and last among them
"""
import math
import random

import torch

own = False
ROPE_BASE = 1.0e6
ROWS = 16          # that share a scale


def _case(name, **kw):
    c = {"op": "attend", "bits": 8, "hq": 32, "hkv": 8, "hd": 128, "streams": 1, "nq": 1, "kv": 1, "page": 16, "ragged": False, "window": 0,
         "cap": 0.0, "bias": 0.0, "block": 16, "top": 1, "sink": 0, "recent": 0}
    c.update(kw)
    return {"name": name, **c} if name else c


def listed():
    return [
        # a decode step of 32 young streams stores a row for each
        _case("append_32_tokens", op="append", streams=32, kv=64, ragged=True),
        # a prompt that fills the cache
        _case("append_8192", op="append", nq=8192, kv=8192),
        # a token at the end of a full cache
        _case("decode_8192", kv=8192),
        # 32 streams of ragged lengths served together
        _case("decode_32_streams", streams=32, kv=8192, ragged=True),
        # decode steps and prompt chunks in one call, scores capped and biased by distance
        _case("mixed_16_streams", streams=16, nq=512, kv=4096, ragged=True, page=32, cap=50.0, bias=8.0),
        # a prompt that fills the cache
        _case("chunk_8192", nq=8192, kv=8192, page=64),
        # what a decode step of 32 streams adds to the bounds
        _case("bounds_32_tokens", op="bounds", streams=32, kv=2048, ragged=True, page=64, block=64),
        # the bounds of a prompt's keys, in a pool of 16 bits
        _case("bounds_8192", op="bounds", bits=16, nq=8192, kv=8192, page=64, block=32),
        # a token's blocks in a long cache: latency
        _case("select_32768", op="select", kv=32768, page=64, block=64, top=32, sink=1, recent=2),
        # those of 32 streams, small blocks
        _case("select_32_streams", op="select", streams=32, kv=16384, ragged=True, page=64, block=32, top=64, sink=1, recent=4),
        # a decode step of 32 streams over 2048 rows of each
        _case("blocks_32_streams", op="blocks", streams=32, kv=8192, ragged=True, page=64, block=64, top=32, sink=1, recent=2),
        # 4 tokens a stream, which a cheaper model proposed, over blocks of a cache of 16 bits
        _case("blocks_4_tokens", op="blocks", bits=16, streams=8, nq=4, kv=8192, page=32, block=32, top=32, sink=1, recent=2),
    ]


def _log(rng, lo, hi):
    return min(hi, max(lo, round(math.exp(rng.uniform(math.log(lo), math.log(hi))))))


def draw(rng):
    op = rng.choice(["append", "attend", "attend", "attend", "bounds", "select", "blocks", "blocks"])
    hq, hkv, hd = rng.choice([(32, 8, 128), (32, 8, 128), (16, 4, 128), (8, 2, 128), (8, 1, 128), (12, 4, 128), (20, 20, 64), (32, 32, 64), (16, 4, 64)])
    page = rng.choice([16, 32, 64, 64, 128])
    c = dict(op=op, hq=hq, hkv=hkv, hd=hd, page=page, ragged=rng.random() < 0.6)
    if op == "append":
        streams = rng.choice([1, rng.randrange(2, 33)])
        c.update(streams=streams, nq=rng.choice([1, _log(rng, 2, 8192 // streams)]))
        c["kv"] = min(8192, c["nq"] + _log(rng, 1, 8192 // streams))
    elif op == "attend":
        form = rng.choice(["decode", "decode", "steps", "chunk", "mixed"])
        streams = 1 if form == "chunk" and rng.random() < 0.5 else rng.choice([1, rng.randrange(2, 33)]) if form != "mixed" else rng.randrange(2, 17)
        nq = {"decode": 1, "steps": rng.randrange(2, 5), "chunk": _log(rng, 8, 2048), "mixed": _log(rng, 16, 512)}[form]
        past = _log(rng, 8, 8191)
        if nq > 4:
            past = min(past, 4096)
            nq = min(nq, max(8, 4096 // streams))
        c.update(streams=streams, nq=nq, kv=past + nq, window=rng.choice([0, 0, _log(rng, 64, 4096)]),
                 cap=rng.choice([0.0, 0.0, 30.0, 50.0]), bias=rng.choice([0.0, 0.0, 8.0]))
    else:
        streams = rng.choice([1, rng.randrange(2, 33)])
        nq = rng.choice([1, 1, rng.randrange(2, 5), _log(rng, 8, 8192 if op == "bounds" else 256)])
        nq = min(nq, max(1, (8192 if op == "bounds" else 512 if op == "select" else 256) // streams))
        kv = nq + _log(rng, 16, 8192 // (streams if op == "bounds" else 1))
        block = rng.choice([b for b in (16, 32, 64, 128) if b <= page])
        top = min(_log(rng, 2, 64), max(2, 2048 // block))
        sink = rng.randrange(0, min(top, 4))
        c.update(bits=rng.choice([8, 16]) if op != "select" else 8, streams=streams, nq=nq, kv=kv, block=block, top=top, sink=sink,
                 recent=rng.randrange(0, min(top - sink, 4) + 1), window=0 if op == "bounds" else rng.choice([0, 0, _log(rng, 64, 4096)]))
        if op == "blocks":
            c.update(cap=rng.choice([0.0, 0.0, 30.0, 50.0]), bias=rng.choice([0.0, 0.0, 8.0]))
    return _case(None, **c)


def _sizes(c, seed):
    """Rows and new tokens of each stream. (The chunks are the case's: a call's shapes go by their sum.)"""
    r, chunks = random.Random(seed * 7919 + 13), random.Random(c["streams"] * 8209 + c["nq"])
    kv = [c["kv"]] * c["streams"]
    nq = [c["nq"]] * c["streams"]
    if c["ragged"]:
        if c["nq"] > 1:
            nq = [1 if chunks.random() < 0.5 else chunks.randint(1, c["nq"]) for _ in nq]
        kv = [r.randint(max(t, 1, c["kv"] // 16), c["kv"]) for t in nq]
    return kv, nq


def _two(e):
    """2^e in 32 bits, exactly (a power function need not be): e from -126 to 127."""
    return ((e.int() + 127) << 23).view(torch.float32)


def _inputs(c, seed):
    """Pool [page][row][kv head][hd] of whole numbers of 8 bits with scales [page][kv head][16 rows], or F16; bounds
    [page][kv head][block][upper hd, lower hd] with scales [page][kv head][block]; queries [token][head][hd]: F16, or as
    projected, F32 [token][head * hd], for the append. Each stream's pages are drawn from anywhere in the pool."""
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    kv, nq = _sizes(c, seed)
    B, ps, hq, hkv, D = c["streams"], c["page"], c["hq"], c["hkv"], c["hd"]
    T, most = sum(nq), -(-c["kv"] // ps)
    need = [-(-n // ps) for n in kv]
    total = B * most + 7
    ids = torch.randperm(total, generator=g, device="cuda").to(torch.int32)
    first = torch.tensor([sum(need[:s]) for s in range(B)], device="cuda")[:, None]
    col = torch.arange(most, device="cuda")[None, :]
    table = torch.where(col < torch.tensor(need, device="cuda")[:, None], ids[(first + col).clamp(max=total - 1)], -1)

    def normal(shape, dtype=torch.float32):
        return torch.randn(shape, generator=g, device="cuda", dtype=dtype)

    def whole(shape, middle=0.0, spread=32.0):
        return normal(shape, torch.float16).mul_(spread).add_(middle).round_().clamp_(-127, 127).to(torch.int8)

    def powers(shape, lo, hi):
        return _two(torch.randint(lo, hi + 1, shape, generator=g, device="cuda"))

    x = {"table": table.to(torch.int32).contiguous(), "n_kv": torch.tensor(kv, device="cuda", dtype=torch.int32),
         "q_start": torch.tensor([sum(nq[:s]) for s in range(B + 1)], device="cuda", dtype=torch.int32)}
    if c["op"] != "select":
        if c["bits"] == 8:
            # values of about 1; those of V differ more from block to block
            x.update(k=whole((total, ps, hkv, D)), v=whole((total, ps, hkv, D)),
                     ks=powers((total, hkv, ps // ROWS), -6, -5), vs=powers((total, hkv, ps // ROWS), -7, -4))
        else:
            x.update(k=normal((total, ps, hkv, D), torch.float16), v=normal((total, ps, hkv, D), torch.float16))
    if c["op"] in ("bounds", "select"):
        n = ps // c["block"]
        # (the largest of a block's keys lies about 2.4 above their mean)
        x["b"] = torch.cat([whole((total, hkv, n, D), 77.0, 13.0), whole((total, hkv, n, D), -77.0, 13.0)], -1)
        x["bs"] = powers((total, hkv, n), -6, -5)
    if c["op"] == "append":
        x.update(q=normal((T, hq, D)), k_new=normal((T, hkv * D)), v_new=normal((T, hkv * D)),
                 q_out=torch.zeros((T, hq, D), device="cuda", dtype=torch.float16))
        x["positions"] = torch.cat([torch.arange(n - t, n) for n, t in zip(kv, nq)]).to("cuda", torch.int32)
    elif c["op"] != "bounds":
        x["q"] = normal((T, hq, D), torch.float16)
    if c["op"] in ("attend", "blocks"):
        x["dst"] = torch.zeros((T, hq, D), device="cuda", dtype=torch.float16)
    if c["op"] == "select":
        x["list"] = torch.full((T, hkv, c["top"]), -1, device="cuda", dtype=torch.int32)
    if c["op"] == "blocks":
        # the first, the last and any others of the blocks that a token sees
        p = torch.cat([torch.arange(n - t, n) for n, t in zip(kv, nq)]).to("cuda")
        last, nb = p // c["block"], -(-c["kv"] // c["block"])
        low = torch.clamp(p - c["window"] + 1, min=0) // c["block"] if c["window"] else torch.zeros_like(p)
        j = torch.arange(nb, device="cuda")[None, None, :]
        key = torch.rand((T, hkv, nb), generator=g, device="cuda")
        key = torch.where((j < low[:, None, None] + c["sink"]) | (j > last[:, None, None] - c["recent"]), 2.0, key)
        key = torch.where((j < low[:, None, None]) | (j > last[:, None, None]), -1.0, key)
        best = torch.topk(key, min(c["top"], nb), -1)
        at = torch.where(best.values >= 0, best.indices, nb).sort(-1).values
        x["list"] = torch.full((T, hkv, c["top"]), -1, device="cuda", dtype=torch.int32)
        x["list"][..., :at.shape[-1]] = torch.where(at < nb, at, -1).int()
    return x


def prepare(case, seed):
    return {"case": dict(case), "x": _inputs(case, seed)}


# ---- the plain form --------------------------------------------------------------------------------------------------


def _tokens(c, x):
    """Padded [stream, token]: index of the packed token, whether there is one, its row of the stream."""
    i = torch.arange(c["nq"], device="cuda")[None, :]
    start, end = x["q_start"][:-1, None].long(), x["q_start"][1:, None].long()
    return start + i, start + i < end, x["n_kv"][:, None].long() - (end - start) + i


def _of_tokens(c, x):
    """Stream and row of each packed token."""
    tok, there, row = _tokens(c, x)
    T = (x["q"] if "q" in x else x["k_new"]).shape[0]
    stream = torch.arange(c["streams"], device="cuda")[:, None].expand_as(tok)
    of = torch.empty((T + 1, 2), device="cuda", dtype=torch.int64)
    of[torch.where(there, tok, T).flatten()] = torch.stack([stream.flatten(), row.flatten()], -1)
    return of[:T, 0], of[:T, 1]


def _turn(x, positions):
    """x [token, head, D] turned: pair j of a token at position p by p * base^(-2 j / D)."""
    D = x.shape[-1]
    # (the angle of a far position is a large number: in 64 bits)
    e = torch.arange(D // 2, device="cuda", dtype=torch.float64) * (-2.0 / D)
    a = positions.double()[:, None] * torch.pow(torch.tensor(ROPE_BASE, device="cuda", dtype=torch.float64), e)
    cos, sin = a.cos().float()[:, None, :], a.sin().float()[:, None, :]
    x0, x1 = x[..., 0::2], x[..., 1::2]
    return torch.stack([x0 * cos - x1 * sin, x0 * sin + x1 * cos], -1).flatten(-2)


def _power(largest):
    """Exponents: the least e with largest <= 127 * 2^e, from -64 to 64."""
    m, e = torch.frexp(largest)                       # largest = m 2^e, m from 1/2 to 1
    e = e - 7 + (m > 127.0 / 128.0)
    return torch.where(largest > 0, e, -64).clamp(-64, 64)


def _new_blocks(c, x, size):
    """Padded [stream, block]: the blocks of `size` rows with new ones, whether there is such a block, its page and its
    place in the page; rows of the stream [stream, block, row], and which of them are new."""
    n = x["n_kv"][:, None].long()
    past = n - (x["q_start"][1:, None] - x["q_start"][:-1, None]).long()
    b = past // size + torch.arange((c["nq"] + size - 2) // size + 1, device="cuda")[None, :]
    there = b * size < n
    row = b[..., None] * size + torch.arange(size, device="cuda")
    page = x["table"][torch.arange(c["streams"], device="cuda")[:, None], (b * size // c["page"]).clamp(max=x["table"].shape[1] - 1)].long()
    return there, page, b * size % c["page"] // size, row, (row >= past[..., None]) & (row < n[..., None])


def _append(c, x):
    D, hkv, ps = c["hd"], c["hkv"], c["page"]
    there, page, at, row, new = _new_blocks(c, x, ROWS)
    start = x["q_start"][:-1].long()[:, None, None]
    past = x["n_kv"].long()[:, None, None] - (x["q_start"][1:] - x["q_start"][:-1]).long()[:, None, None]
    tok = (start + row - past).clamp(0, x["q"].shape[0] - 1)
    f = there.nonzero()
    page, at, new, row, tok = (t[f[:, 0], f[:, 1]] for t in (page, at, new, row, tok))
    rows = at[:, None] * ROWS + torch.arange(ROWS, device="cuda")
    past = past[f[:, 0], 0]
    held = row[:, :1] < past                                # there are rows ahead of the new ones
    h = torch.arange(hkv, device="cuda")
    for name, t in (("k", _turn(x["k_new"].view(-1, hkv, D), x["positions"])), ("v", x["v_new"].view(-1, hkv, D))):
        fresh = t[tok]                                       # [block, row, head, D]
        old = x[name][page[:, None], rows]
        olds = x[name + "s"][page[:, None], h, at[:, None]]
        e = _power((fresh.abs() * new[..., None, None]).amax((1, 3)))
        eo = torch.frexp(olds)[1] - 1
        e = torch.where(held, torch.maximum(e, eo), e)
        keep = torch.where((row < past)[..., None], (eo - e)[:, None, :], 0)
        old = (old.float() * _two(keep.clamp(min=-126))[..., None]).round()
        got = (fresh * _two(-e)[:, None, :, None]).round().clamp(-127, 127)
        x[name][page[:, None], rows] = torch.where(new[..., None, None], got, old).to(torch.int8)
        x[name + "s"][page[:, None], h, at[:, None]] = _two(e)
    x["q_out"].copy_(_turn(x["q"], x["positions"]))


def _values(x, scale, rows=ROWS):
    """Pool [page, row, head, D] of whole numbers times the scales [page, head, rows' block]."""
    y = x.float().unflatten(1, (-1, rows)) * scale.permute(0, 2, 1)[:, :, None, :, None]
    return y.flatten(1, 2)


def _gather(c, x, name, rows):
    """[stream, row, head, D] of the streams' pages, in 32 bits."""
    page = x["table"].clamp(min=0).long()
    y = x[name][page].flatten(0, 1)
    y = _values(y, x[name + "s"][page].flatten(0, 1)) if c["bits"] == 8 else y.float()
    return y.unflatten(0, page.shape).flatten(1, 2)[:, :rows]


def _slopes(c):
    if not c["bias"]:
        return torch.zeros(c["hq"], device="cuda")
    n = 1 << (c["hq"].bit_length() - 1)
    h = torch.arange(c["hq"], device="cuda", dtype=torch.float64)
    return torch.where(h < n, torch.exp2(-c["bias"] / n * (h + 1)), torch.exp2(-c["bias"] / n * (h - n + 0.5))).float()


def _softmax(s):
    """In place; a row without a score gets zeros."""
    m = s.amax(-1, keepdim=True).clamp_(min=-3.0e38)
    p = s.sub_(m).exp_()
    l = p.sum(-1, keepdim=True)
    return p.mul_(torch.where(l > 0, 1.0 / l, 0.0))


def _attend(c, x):
    B, NQ, N, hkv, D = c["streams"], c["nq"], c["kv"], c["hkv"], c["hd"]
    G, T = c["hq"] // hkv, x["q"].shape[0]
    tok, there, row = _tokens(c, x)
    q = x["q"][tok.clamp(max=T - 1)].float().view(B, NQ, hkv, G, D).permute(0, 2, 3, 1, 4).reshape(B * hkv, G * NQ, D)
    k = _gather(c, x, "k", N).permute(0, 2, 3, 1).reshape(B * hkv, D, N).contiguous()
    s = torch.bmm(q, k).view(B, hkv, G, NQ, N).mul_(1.0 / math.sqrt(D))
    del k
    if c["cap"]:
        s.div_(c["cap"]).tanh_().mul_(c["cap"])
    j = torch.arange(N, device="cuda")[None, None, :]
    if c["bias"]:
        s += _slopes(c).view(1, hkv, G, 1, 1) * (j - row[:, :, None]).float()[:, None, None]
    dead = (j > row[:, :, None]) | ~there[:, :, None]
    if c["window"]:
        dead |= j <= row[:, :, None] - c["window"]
    p = _softmax(s.masked_fill_(dead[:, None, None], float("-inf")))
    v = _gather(c, x, "v", N).permute(0, 2, 1, 3).reshape(B * hkv, N, D)
    o = torch.bmm(p.view(B * hkv, G * NQ, N), v).view(B, hkv, G, NQ, D).permute(0, 3, 1, 2, 4).reshape(B * NQ, c["hq"], D)
    out = torch.empty((T + 1, c["hq"], D), device="cuda", dtype=torch.float16)
    out[torch.where(there, tok, T).flatten()] = o.half()
    x["dst"].copy_(out[:T])


def _bounds(c, x):
    there, page, at, row, _ = _new_blocks(c, x, c["block"])
    f = there.nonzero()
    page, at, row = (t[f[:, 0], f[:, 1]] for t in (page, at, row))
    live = (row < x["n_kv"].long()[f[:, 0], None])[..., None, None]
    rows = at[:, None] * c["block"] + torch.arange(c["block"], device="cuda")
    k = x["k"][page[:, None], rows].float()                 # [block, row, head, D]
    h = torch.arange(c["hkv"], device="cuda")
    if c["bits"] == 8:
        k *= x["ks"][page[:, None, None], h, (rows // ROWS)[..., None]][..., None]
    hi, lo = k.masked_fill(~live, float("-inf")).amax(1), k.masked_fill(~live, float("inf")).amin(1)
    e = _power(torch.maximum(hi.abs(), lo.abs()).amax(-1))
    x["b"][page[:, None], h, at[:, None]] = torch.cat([(hi * _two(-e)[..., None]).ceil(), (lo * _two(-e)[..., None]).floor()], -1).to(torch.int8)
    x["bs"][page[:, None], h, at[:, None]] = _two(e)


def _select(c, x):
    hkv, D, G, top = c["hkv"], c["hd"], c["hq"] // c["hkv"], c["top"]
    stream, row = _of_tokens(c, x)
    per, nb = c["page"] // c["block"], -(-c["kv"] // c["block"])
    page = x["table"].clamp(min=0).long()
    b = x["b"][page].permute(0, 2, 1, 3, 4).flatten(2, 3)[:, :, :nb].float()          # [stream, head, block, 2 D]
    bs = x["bs"][page].permute(0, 2, 1, 3).flatten(2)[:, :, :nb]
    q = x["q"].float().view(-1, hkv, G, D)
    e = _power(q.abs().amax(-1))
    q = (q * _two(-e)[..., None]).round()
    q = torch.cat([q.clamp(min=0), q.clamp(max=0)], -1)
    score = torch.empty((q.shape[0], hkv, nb), device="cuda")
    for s in range(c["streams"]):
        at = stream == s
        y = torch.matmul(q[at], b[s].transpose(-1, -2).contiguous())                   # [token, head, group, block]
        score[at] = (y * _two(e[at])[..., None]).amax(2) * bs[s]
    j = torch.arange(nb, device="cuda")[None, None, :]
    last = (row // c["block"])[:, None, None]
    low = (torch.clamp(row - c["window"] + 1, min=0) // c["block"])[:, None, None] if c["window"] else torch.zeros_like(last)
    score = torch.where((j < low + c["sink"]) | (j > last - c["recent"]), float("inf"), score)
    score = torch.where((j < low) | (j > last), float("-inf"), score)
    best = torch.sort(score, dim=-1, descending=True, stable=True)
    at = torch.where(best.values[..., :top] > float("-inf"), best.indices[..., :top], nb).sort(-1).values
    x["list"].fill_(-1)
    x["list"][..., :at.shape[-1]] = torch.where(at < nb, at, -1).int()


def _blocks(c, x):
    hkv, D, G, size = c["hkv"], c["hd"], c["hq"] // c["hkv"], c["block"]
    stream, row = _of_tokens(c, x)
    h = torch.arange(hkv, device="cuda")[None, :, None, None]
    slopes = _slopes(c).view(1, hkv, G, 1)
    step = max(1, (1 << 27) // (hkv * c["top"] * size * D))
    for t0 in range(0, stream.shape[0], step):
        t = slice(t0, t0 + step)
        b = x["list"][t].long()
        j = b.clamp(min=0)[..., None] * size + torch.arange(size, device="cuda")       # [token, head, block, row]
        p = row[t, None, None, None]
        dead = (b < 0)[..., None] | (j > p)
        if c["window"]:
            dead |= j <= p - c["window"]
        page = x["table"][stream[t, None, None, None], (j // c["page"]).clamp(max=x["table"].shape[1] - 1)].clamp(min=0).long()
        r = j % c["page"]
        k, v = x["k"][page, r, h].float(), x["v"][page, r, h].float()
        if c["bits"] == 8:
            k *= x["ks"][page, h, r // ROWS][..., None]
            v *= x["vs"][page, h, r // ROWS][..., None]
        n = k.shape[0]
        k, v = (y.view(n * hkv, -1, D) for y in (k, v))
        q = x["q"][t].float().view(n * hkv, G, D)
        s = torch.bmm(q, k.transpose(1, 2).contiguous()).view(n, hkv, G, -1).mul_(1.0 / math.sqrt(D))
        if c["cap"]:
            s.div_(c["cap"]).tanh_().mul_(c["cap"])
        if c["bias"]:
            s += slopes * (j - p).flatten(2)[:, :, None].float()
        a = _softmax(s.masked_fill_(dead.flatten(2)[:, :, None], float("-inf")))
        x["dst"][t] = torch.bmm(a.view(n * hkv, G, -1), v).view(n, c["hq"], D).half()


# ---- the framework's calls -------------------------------------------------------------------------------------------

_kept = {}


def _package():
    """The package's folder name is not a Python identifier."""
    import importlib.util
    import os
    import sys
    if "voxtral_cpp_amd" not in sys.modules:
        folder = os.path.abspath("voxtral.cpp_amd")
        spec = importlib.util.spec_from_file_location("voxtral_cpp_amd", os.path.join(folder, "__init__.py"), submodule_search_locations=[folder])
        sys.modules["voxtral_cpp_amd"] = importlib.util.module_from_spec(spec)
        spec.loader.exec_module(sys.modules["voxtral_cpp_amd"])
    return sys.modules["voxtral_cpp_amd"]


def _call(c, x):
    """The call on these buffers: a function of the stream. A program holds the context and the descriptors of its
    buffers from step to step."""
    pkg = _package()
    vxfa, views = pkg.vxfa, pkg.views
    if "ctx" not in _kept:
        _kept["ctx"] = vxfa.Context(torch.cuda.current_device())
    ctx = _kept["ctx"]
    D, hq, hkv, ps, op = c["hd"], c["hq"], c["hkv"], c["page"], c["op"]
    total = (x["k"] if "k" in x else x["b"]).shape[0]
    k = v = ks = vs = None
    if "k" in x:
        i8 = c["bits"] == 8
        k, v = (vxfa.desc(x[t].data_ptr(), vxfa.I8 if i8 else vxfa.F16, *views.kv_pages(total, ps, hkv, D, 1 if i8 else 2)) for t in "kv")
        if i8:
            ks, vs = (vxfa.desc(x[t].data_ptr(), vxfa.F32, *views.scale_pages(total, ps, hkv)) for t in ("ks", "vs"))
    if "b" in x:
        b = vxfa.desc(x["b"].data_ptr(), vxfa.I8, *views.bound_pages(total, ps, hkv, D, c["block"]))
        bs = vxfa.desc(x["bs"].data_ptr(), vxfa.F32, *views.scale_pages(total, ps, hkv, c["block"]))
    batch = vxfa.paged(x["table"].data_ptr(), x["n_kv"].data_ptr(), x["q_start"].data_ptr(), c["streams"], x["table"].shape[1],
                       max_nq=c["nq"], max_nkv=c["kv"], window=c["window"])
    if op == "bounds":
        return lambda s: ctx.paged_bounds(k, ks, batch, b, bs, stream=s)
    T = x["q"].shape[0]
    if op == "append":
        q = vxfa.desc(x["q"].data_ptr(), vxfa.F32, *views.decoder_q(T, hq, D))
        q_out = vxfa.desc(x["q_out"].data_ptr(), vxfa.F16, *views.decoder_q(T, hq, D, 2))
        w = hkv * D
        new = [vxfa.desc(x[t].data_ptr(), vxfa.F32, (w, T, 1, 1), (4, 4 * w, 4 * w * T, 4 * w * T)) for t in ("k_new", "v_new")]
        rope = vxfa.rope(x["positions"].data_ptr(), D, ROPE_BASE)
        return lambda s: ctx.paged_append_q8(*new, batch, k, ks, v, vs, rope=rope, q=q, q_out=q_out, stream=s)
    q = vxfa.desc(x["q"].data_ptr(), vxfa.F16, *views.decoder_q(T, hq, D, 2))
    if op != "attend":
        chosen = vxfa.blocks(x["list"].data_ptr(), c["block"], c["top"], c["sink"], c["recent"])
    if op == "select":
        return lambda s: ctx.paged_select(q, b, bs, batch, chosen, stream=s)
    dst = vxfa.desc(x["dst"].data_ptr(), vxfa.F16, *views.dst(D, hq, T, elt=2))
    scale = 1.0 / math.sqrt(D)
    if op == "blocks":
        return lambda s: ctx.flash_attn_ext_paged_blocks(q, k, ks, v, vs, batch, chosen, dst, scale, c["bias"], c["cap"], stream=s)
    return lambda s: ctx.flash_attn_ext_paged_q8(q, k, ks, v, vs, batch, dst, scale, c["bias"], c["cap"], stream=s)


def run(state):
    c, x = state["case"], state["x"]
    if not own:
        {"append": _append, "attend": _attend, "bounds": _bounds, "select": _select, "blocks": _blocks}[c["op"]](c, x)
    else:
        if "call" not in state:
            state["call"] = _call(c, x)
        state["call"](torch.cuda.current_stream().cuda_stream)
    if c["op"] == "append":
        # the values that the pools stand for (which bfloat16 holds exactly)
        n = (-1, c["page"] // ROWS, ROWS, c["hkv"], c["hd"])
        kv = [x[t].view(n) * x[t + "s"].bfloat16().transpose(1, 2)[:, :, None, :, None] for t in "kv"]
        return {"k": kv[0], "v": kv[1], "q": x["q_out"]}
    if c["op"] == "bounds":
        return {"bounds": x["b"] * x["bs"][..., None]}
    return {"list": x["list"]} if c["op"] == "select" else {"dst": x["dst"]}


# ---- work and exact answers ------------------------------------------------------------------------------------------


def work(case):
    """Every live row of K and V and every scale, query and bound read once, outputs written once; two products of hd
    multiply-adds for every live pair and query head. (A ragged case's sizes are drawn with its inputs: the mean of 16
    draws. Of chosen blocks that several tokens of a stream share each is counted for each.)"""
    c = case
    D, hq, hkv, size = c["hd"], c["hq"], c["hkv"], c["block"]
    row = hkv * (D + 4.0 / ROWS) if c["bits"] == 8 else hkv * 2 * D     # bytes of K or V
    by = fl = 0
    draws = 16 if c["ragged"] else 1
    for seed in range(draws):
        for n, t in zip(*_sizes(c, seed)):
            if c["op"] == "append":
                by += t * (8 * hkv * D + 2 * row + 6 * hq * D)
            elif c["op"] == "bounds":
                first = (n - t) // size
                by += (n - first * size) * row + (-(-n // size) - first) * hkv * (2 * D + 4)
            elif c["op"] == "attend":
                w = c["window"] or n
                by += 2 * min(n, w + t - 1) * row + 4 * t * hq * D
                fl += 4 * D * hq * sum(min(n - t + i + 1, w) for i in range(t))
            else:
                w = c["window"] or n
                seen = [(p // size + 1 - max(p - w + 1, 0) // size, min(p + 1, w)) for p in range(n - t, n)]
                if c["op"] == "select":
                    by += max(b for b, _ in seen) * hkv * (2 * D + 4) + t * (2 * hq * D + 4 * hkv * c["top"])
                    fl += 4 * D * hq * sum(b for b, _ in seen)
                else:
                    rows = sum(min(c["top"] * size, r) for _, r in seen)
                    by += 2 * rows * row + t * (4 * hq * D + 4 * hkv * c["top"])
                    fl += 4 * D * hq * rows
    return {"bytes": by / draws, "flops": fl / draws}


def exact(case, seed):
    c, x = case, _inputs(case, seed)
    kv, nq = _sizes(c, seed)
    D, hkv, ps, group, size = c["hd"], c["hkv"], c["page"], c["hq"] // c["hkv"], c["block"]
    T = sum(nq)

    def unit(largest):
        """[...] -> the least 2^e with largest <= 127 2^e, e between -64 and 64."""
        u = torch.full_like(largest, 2.0 ** -64)
        for i in range(-63, 65):
            u = torch.where(largest > 127.0 * 2.0 ** (i - 1), 2.0 ** i, u)
        return u

    def held(name, s, n, h):
        """Rows of a stream's head."""
        r = torch.arange(n, device="cuda")
        p = x["table"][s][r // ps].long()
        y = x[name][p, r % ps, h].double()
        return y * x[name + "s"][p, h, r % ps // ROWS].double()[:, None] if c["bits"] == 8 else y

    if c["op"] == "append":
        def turned(t, positions):
            # each pair's angle is the previous one's times a factor
            out, th = t.double().clone(), positions.double()
            for i in range(D // 2):
                co, si = th.cos()[:, None], th.sin()[:, None]
                a, b = t[..., 2 * i].double(), t[..., 2 * i + 1].double()
                out[..., 2 * i], out[..., 2 * i + 1] = a * co - b * si, a * si + b * co
                th = th * ROPE_BASE ** (-2.0 / D)
            return out

        if sum(t // ROWS + 2 for t in nq) > 1200:
            return None
        out = {"q": turned(x["q"], x["positions"])}
        for name in "kv":
            y = x[name].double().unflatten(1, (-1, ROWS)) * x[name + "s"].double().transpose(1, 2)[:, :, None, :, None]
            new = x[name + "_new"].view(T, hkv, D).double()
            if name == "k":
                new = turned(new, x["positions"])
            t0 = 0
            for s, (n, t) in enumerate(zip(kv, nq)):
                for b in range((n - t) // ROWS, (n - 1) // ROWS + 1):
                    p, i = int(x["table"][s, b * ROWS // ps]), b * ROWS % ps // ROWS
                    r0, r1 = max(n - t - b * ROWS, 0), min(n - b * ROWS, ROWS)
                    a = new[t0 + b * ROWS + r0 - (n - t):t0 + b * ROWS + r1 - (n - t)]
                    u = unit(a.abs().amax((0, 2)))[:, None]
                    was = x[name + "s"][p, :, i].double()[:, None]
                    if r0 > 0:
                        u = torch.maximum(u, was)
                    y[p, i, :r0] = (y[p, i, :r0] / u).round() * u
                    y[p, i, r0:r1] = (a / u).round() * u
                    # (rows behind the last keep their whole numbers)
                    y[p, i, r1:] *= u / was
                t0 += t
            out[name] = y
        return out
    if c["op"] == "bounds":
        b = x["b"].double() * x["bs"].double()[..., None]
        for s, (n, t) in enumerate(zip(kv, nq)):
            first, last = (n - t) // size, (n - 1) // size
            if (last - first) * hkv > 4096:
                return None
            for h in range(hkv):
                k = held("k", s, n, h)
                for i in range(first, last + 1):
                    y = k[i * size:(i + 1) * size]
                    u = unit(y.abs().max())
                    p = int(x["table"][s, i * size // ps])
                    b[p, h, i * size % ps // size] = torch.cat([(y.max(0).values / u).ceil() * u, (y.min(0).values / u).floor() * u])
        return {"bounds": b}
    if c["op"] == "select":
        if T * hkv > 3000:
            return None
        out = x["list"].clone()
        t0 = 0
        for s, (n, t) in enumerate(zip(kv, nq)):
            i = torch.arange(-(-n // size), device="cuda")
            p = x["table"][s][i * size // ps].long()
            for h in range(hkv):
                b = x["b"][p, h, i * size % ps // size].double() * x["bs"][p, h, i * size % ps // size].double()[:, None]
                q = x["q"][t0:t0 + t, h * group:(h + 1) * group].double()
                u = unit(q.abs().amax(-1, keepdim=True))
                q = (q / u).round() * u
                score = torch.stack([torch.maximum(q[:, g, None] * b[None, :, :D], q[:, g, None] * b[None, :, D:]).sum(-1) for g in range(group)]).amax(0).tolist()
                for a in range(t):
                    row = n - t + a
                    low, high = max(row - c["window"] + 1, 0) // size if c["window"] else 0, row // size
                    seen = list(range(low, high + 1))
                    ends = sorted(set(seen[:c["sink"]] + seen[len(seen) - min(c["recent"], len(seen)):]))
                    rest = sorted((y for y in seen if y not in set(ends)), key=lambda y: (-score[a][y], y))
                    best = sorted(ends + rest[:c["top"] - len(ends)])
                    out[t0 + a, h] = torch.tensor(best + [-1] * (c["top"] - len(best)), dtype=torch.int32)
            t0 += t
        return {"list": out}
    if c["op"] == "blocks" and T * hkv > 4096:
        return None
    dst = torch.zeros((T, c["hq"], D), device="cuda", dtype=torch.float64)
    n2 = 2 ** int(math.log2(c["hq"]))
    t0 = 0
    for s, (n, t) in enumerate(zip(kv, nq)):
        rows = torch.arange(n, device="cuda")
        for h in range(hkv):
            k, v = held("k", s, n, h), held("v", s, n, h)
            for i0 in range(0, t, 2048):
                i = torch.arange(i0, min(t, i0 + 2048), device="cuda")
                p = (n - t + i)[:, None]
                off = rows[None] > p
                if c["window"]:
                    off = off | (rows[None] <= p - c["window"])
                if c["op"] == "blocks":
                    chosen = torch.zeros((len(i), -(-n // size) + 1), dtype=torch.bool, device="cuda")
                    chosen.scatter_(1, x["list"][t0 + i, h].long() + 1, True)
                    off = off | ~chosen[:, rows // size + 1]
                for g in range(h * group, (h + 1) * group):
                    slope = 0.0
                    if c["bias"]:
                        slope = 2.0 ** (-c["bias"] * (g + 1) / n2) if g < n2 else 2.0 ** (-c["bias"] / 2 / n2 * (2 * (g - n2) + 1))
                    a = x["q"][t0 + i, g].double() @ k.t().contiguous() / math.sqrt(D)
                    if c["cap"]:
                        a = c["cap"] * torch.tanh(a / c["cap"])
                    a = (a + slope * (rows[None] - p)).masked_fill(off, float("-inf"))
                    dst[t0 + i, g] = torch.softmax(a, -1) @ v
        t0 += t
    return {"dst": dst}
