"""Serving from a paged K/V cache: what its calls are, their inputs, one pass of each, their answers.

A cache is a pool of pages of `page` rows; a stream's rows lie in the pages
that its line of a table names (-1: none), in order. A call takes a batch of
streams, each with its number of rows and a chunk of new tokens, which are its
last rows; the tokens of all streams are packed one after another.

  op        "append": the new rows stored in their pages, keys and queries
            rotated. "attend": attention of the new tokens over their streams'
            rows. "evict": of every stream and kv head `budget` rows kept, by
            accumulated attention weight, and moved to other pages
  hq hkv hd query heads, kv heads, head dim
  streams, nq, kv   streams, most new tokens and most rows of one
  ragged    the streams' rows lie between a sixteenth of kv and kv (else all
            have kv), and with nq > 1 about half of them have a single new
            token, the others up to nq (else all have nq)
  window    > 0: a token attends the last `window` rows up to its own
  cap, bias the score cap (0: none) and the largest exponent of the heads'
            distance slopes (0: none)
  weights   the call also adds each row's attention weight to its accumulator
  budget sink recent   rows kept of a stream, among them its first and last
"""
import math
import random

import torch

own = False
ROPE_BASE = 1.0e6


def _case(name, **kw):
    c = {"op": "attend", "hq": 32, "hkv": 8, "hd": 128, "streams": 1, "nq": 1, "kv": 1, "page": 16, "ragged": False, "window": 0, "cap": 0.0,
         "bias": 0.0, "weights": False, "budget": 0, "sink": 0, "recent": 0}
    c.update(kw)
    return {"name": name, **c} if name else c


def listed():
    return [
        # a decode step of 32 streams stores a row for each
        _case("append_32_tokens", op="append", streams=32, kv=8192, ragged=True),
        # a prompt that fills the cache
        _case("append_8192", op="append", nq=8192, kv=8192),
        # the first generated token after a 39-token prompt: latency
        _case("decode_first", kv=40),
        # a token at the end of a full cache
        _case("decode_8192", kv=8192),
        # 32 streams of ragged lengths served together
        _case("decode_32_streams", streams=32, kv=8192, ragged=True),
        # the same step where rows are to be dropped by their weight later
        _case("decode_32_weights", streams=32, kv=8192, ragged=True, weights=True),
        # a further 600 tokens for a session that holds 3000 rows
        _case("chunk_600", nq=600, kv=3600, page=64),
        # a prompt that fills the cache
        _case("chunk_8192", nq=8192, kv=8192, page=64),
        # decode steps and prompt chunks in one call, scores capped and
        # biased by distance
        _case("mixed_16_streams", streams=16, nq=512, kv=4096, ragged=True, page=32, cap=50.0, bias=8.0),
        # chunks of a streaming encoder: 20 heads of 64, window of 750
        _case("chunk_hd64_window", hq=20, hkv=20, hd=64, streams=8, nq=250, kv=1500, page=32, window=750, weights=True),
        # a full cache halved by the weights of its rows
        _case("evict_4096", op="evict", kv=8192, budget=4096, sink=4, recent=512),
        # all streams cut to a thousand rows
        _case("evict_32_streams", op="evict", streams=32, kv=8192, ragged=True, budget=1000, sink=4, recent=128),
    ]


def _log(rng, lo, hi):
    return min(hi, max(lo, round(math.exp(rng.uniform(math.log(lo), math.log(hi))))))


def draw(rng):
    op = rng.choice(["append", "attend", "attend", "attend", "attend", "evict"])
    hq, hkv, hd = rng.choice([(32, 8, 128), (32, 8, 128), (16, 4, 128), (8, 2, 128), (8, 1, 128), (12, 4, 128), (20, 20, 64), (32, 32, 64), (16, 4, 64)])
    page = rng.choice([16, 16, 32, 64, 128])
    c = dict(op=op, hq=hq, hkv=hkv, hd=hd, page=page, ragged=rng.random() < 0.6)
    if op == "append":
        streams = rng.choice([1, rng.randrange(2, 33)])
        c.update(streams=streams, nq=rng.choice([1, _log(rng, 2, 8192 // streams)]))
        c["kv"] = min(8192, c["nq"] + _log(rng, 1, 8192))
    elif op == "evict":
        kv = _log(rng, 64, 8192)
        budget = rng.randrange(kv // 8 + 2, kv)
        sink = rng.randrange(0, min(budget // 2, 64))
        c.update(streams=rng.choice([1, rng.randrange(2, 33)]), kv=kv, budget=budget, sink=sink, recent=rng.randrange(0, budget - sink))
    else:
        form = rng.choice(["decode", "decode", "steps", "chunk", "mixed"])
        streams = 1 if form == "chunk" and rng.random() < 0.5 else rng.choice([1, rng.randrange(2, 33)]) if form != "mixed" else rng.randrange(2, 17)
        nq = {"decode": 1, "steps": rng.randrange(2, 5), "chunk": _log(rng, 8, 2048), "mixed": _log(rng, 16, 512)}[form]
        past = _log(rng, 8, 8191)
        if nq > 4:
            past = min(past, 4096)
            nq = min(nq, max(8, 4096 // streams))
        c.update(streams=streams, nq=nq, kv=past + nq, window=rng.choice([0, 0, _log(rng, 64, 4096)]),
                 cap=rng.choice([0.0, 0.0, 30.0, 50.0]), bias=rng.choice([0.0, 0.0, 8.0]), weights=rng.random() < 0.3)
    return _case(None, **c)


def _sizes(c, seed):
    """Rows and new tokens of each stream. (The chunks are the case's: a call's shapes go by their sum.)"""
    r, chunks = random.Random(seed * 7919 + 13), random.Random(c["streams"] * 8209 + c["nq"])
    kv = [c["kv"]] * c["streams"]
    nq = [0 if c["op"] == "evict" else c["nq"]] * c["streams"]
    if c["ragged"]:
        if c["nq"] > 1:
            nq = [1 if chunks.random() < 0.5 else chunks.randint(1, c["nq"]) for _ in nq]
        kv = [r.randint(max(t, 1, c["kv"] // 16), c["kv"]) for t in nq]
    return kv, nq


def _inputs(c, seed):
    """Pool [page][row][kv head][hd] of F16, accumulators [page][kv head][row] of F32, queries [token][head][hd]: F16
    for attention, and as projected, F32 [token][head * hd], for the append. Each stream's pages are drawn from
    anywhere in the pool."""
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    kv, nq = _sizes(c, seed)
    B, ps, hq, hkv, D = c["streams"], c["page"], c["hq"], c["hkv"], c["hd"]
    T, most = sum(nq), -(-c["kv"] // ps)
    need = [-(-n // ps) for n in kv]
    keep = -(-c["budget"] // ps)
    total = B * most + (B * keep if c["op"] == "evict" else 0) + 7
    ids = torch.randperm(total, generator=g, device="cuda").to(torch.int32)
    first = torch.tensor([sum(need[:s]) for s in range(B)], device="cuda")[:, None]
    col = torch.arange(most, device="cuda")[None, :]
    table = torch.where(col < torch.tensor(need, device="cuda")[:, None], ids[(first + col).clamp(max=total - 1)], -1)

    def normal(shape, dtype=torch.float32):
        return torch.randn(shape, generator=g, device="cuda", dtype=dtype)

    x = {"table": table.to(torch.int32).contiguous(), "n_kv": torch.tensor(kv, device="cuda", dtype=torch.int32),
         "q_start": torch.tensor([sum(nq[:s]) for s in range(B + 1)], device="cuda", dtype=torch.int32),
         "k": normal((total, ps, hkv, D), torch.float16), "v": normal((total, ps, hkv, D), torch.float16)}
    if c["op"] == "append":
        x.update(q=normal((T, hq, D)), k_new=normal((T, hkv * D)), v_new=normal((T, hkv * D)),
                 q_out=torch.zeros((T, hq, D), device="cuda", dtype=torch.float16))
        x["positions"] = torch.cat([torch.arange(n - t, n) for n, t in zip(kv, nq)]).to("cuda", torch.int32)
    elif c["op"] == "attend":
        x.update(q=normal((T, hq, D), torch.float16), dst=torch.zeros((T, hq, D), device="cuda", dtype=torch.float16))
    if c["weights"] or c["op"] == "evict":
        # mostly small and a few large, as accumulated weights are
        x["w"] = torch.rand((total, hkv, ps), generator=g, device="cuda").pow(8).mul_(4.0)
        if c["op"] == "attend":
            x["w_out"] = torch.zeros_like(x["w"])
    if c["op"] == "evict":
        x["to"] = ids[sum(need):sum(need) + B * keep].view(B, keep).contiguous()
        x["kept"] = torch.full((B, hkv, c["budget"]), -1, device="cuda", dtype=torch.int32)
    return x


def prepare(case, seed):
    return {"case": dict(case), "x": _inputs(case, seed)}


# ---- the plain form --------------------------------------------------------------------------------------------------


def _tokens(c, x):
    """Padded [stream, token]: index of the packed token, whether there is one, its row of the stream."""
    i = torch.arange(c["nq"], device="cuda")[None, :]
    start, end = x["q_start"][:-1, None].long(), x["q_start"][1:, None].long()
    return start + i, start + i < end, x["n_kv"][:, None].long() - (end - start) + i


def _turn(x, positions):
    """x [token, head, D] turned: pair j of a token at position p by p * base^(-2 j / D)."""
    D = x.shape[-1]
    # (the angle of a far position is a large number: in 64 bits)
    e = torch.arange(D // 2, device="cuda", dtype=torch.float64) * (-2.0 / D)
    a = positions.double()[:, None] * torch.pow(torch.tensor(ROPE_BASE, device="cuda", dtype=torch.float64), e)
    cos, sin = a.cos().float()[:, None, :], a.sin().float()[:, None, :]
    x0, x1 = x[..., 0::2], x[..., 1::2]
    return torch.stack([x0 * cos - x1 * sin, x0 * sin + x1 * cos], -1).flatten(-2)


def _append(c, x):
    tok, there, row = _tokens(c, x)
    # stream and row of each packed token
    T, ps = x["q"].shape[0], c["page"]
    stream = torch.arange(c["streams"], device="cuda")[:, None].expand_as(tok)
    at = torch.where(there, tok, T).flatten()
    of = torch.empty((T + 1, 2), device="cuda", dtype=torch.int64)
    of[at] = torch.stack([stream.flatten(), row.flatten()], -1)
    stream, row = of[:T, 0], of[:T, 1]
    page = x["table"][stream, row // ps].long()
    x["k"][page, row % ps] = _turn(x["k_new"].view(T, c["hkv"], c["hd"]), x["positions"]).half()
    x["v"][page, row % ps] = x["v_new"].view(T, c["hkv"], c["hd"]).half()
    x["q_out"].copy_(_turn(x["q"], x["positions"]))
    return {"k": x["k"], "v": x["v"], "q": x["q_out"]}


def _slopes(c):
    if not c["bias"]:
        return torch.zeros(c["hq"], device="cuda")
    n = 1 << (c["hq"].bit_length() - 1)
    h = torch.arange(c["hq"], device="cuda", dtype=torch.float64)
    return torch.where(h < n, torch.exp2(-c["bias"] / n * (h + 1)), torch.exp2(-c["bias"] / n * (h - n + 0.5))).float()


def _gather(pool, table, rows):
    """[stream, row, ...] of the streams' pages."""
    x = pool[table.clamp(min=0).long()]
    return x.flatten(1, 2)[:, :rows]


def _attend(c, x):
    B, NQ, N, hkv, D = c["streams"], c["nq"], c["kv"], c["hkv"], c["hd"]
    G, T = c["hq"] // hkv, x["q"].shape[0]
    tok, there, row = _tokens(c, x)
    q = x["q"][tok.clamp(max=T - 1)].float().view(B, NQ, hkv, G, D).permute(0, 2, 3, 1, 4).reshape(B * hkv, G * NQ, D)
    k = _gather(x["k"], x["table"], N).float().permute(0, 2, 3, 1).reshape(B * hkv, D, N).contiguous()
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
    s.masked_fill_(dead[:, None, None], float("-inf"))
    m = s.amax(-1, keepdim=True).clamp_(min=-3.0e38)
    p = s.sub_(m).exp_()
    l = p.sum(-1, keepdim=True)
    p.mul_(torch.where(l > 0, 1.0 / l, 0.0))
    v = _gather(x["v"], x["table"], N).float().permute(0, 2, 1, 3).reshape(B * hkv, N, D)
    o = torch.bmm(p.view(B * hkv, G * NQ, N), v).view(B, hkv, G, NQ, D).permute(0, 3, 1, 2, 4).reshape(B * NQ, c["hq"], D)
    out = torch.empty((T + 1, c["hq"], D), device="cuda", dtype=torch.float16)
    out[torch.where(there, tok, T).flatten()] = o.half()
    x["dst"].copy_(out[:T])
    if not c["weights"]:
        return {"dst": x["dst"]}
    add = p.view(B, hkv, G * NQ, N).sum(2)
    # (past a stream's end its first row once more)
    n, ps, b = torch.arange(N, device="cuda")[None, :], c["page"], torch.arange(B, device="cuda")[:, None]
    n = torch.where(n < x["n_kv"][:, None], n, 0)
    page = x["table"][b, n // ps].long()
    x["w_out"][page, :, n % ps] = x["w"][page, :, n % ps] + add[b, :, n]
    return {"dst": x["dst"], "weights": x["w_out"]}


def _evict(c, x):
    B, N, ps, R = c["streams"], c["kv"], c["page"], c["budget"]
    w = x["w"][x["table"].clamp(min=0).long()].permute(0, 2, 1, 3).flatten(2)[..., :N]
    n = x["n_kv"][:, None, None].long()
    j = torch.arange(N, device="cuda")[None, None, :]
    always = (j < c["sink"]) | (j >= n - c["recent"])
    key = torch.where(j >= n, float("-inf"), torch.where(always, float("inf"), w))
    at = torch.sort(key, dim=-1, descending=True, stable=True).indices[..., :R]
    at = torch.where(at < n, at, N).sort(-1).values
    kept = torch.where(at < N, at, -1)
    x["kept"][..., :kept.shape[-1]] = kept
    r = torch.arange(kept.shape[-1], device="cuda")
    b, h = torch.arange(B, device="cuda")[:, None, None], torch.arange(c["hkv"], device="cuda")[None, :, None]
    # (past the end of the kept rows the first one once more)
    r = torch.where(kept >= 0, r, 0)
    src = torch.where(kept >= 0, kept, kept[..., :1])
    old, new = x["table"][b, src // ps].long(), x["to"][b, r // ps].long()
    for name in ("k", "v"):
        x[name][new, r % ps, h] = x[name][old, src % ps, h]
    x["w"][new, h, r % ps] = x["w"][old, h, src % ps]
    return {"k": x["k"], "v": x["v"], "weights": x["w"], "kept": x["kept"]}


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
    D, hq, hkv, ps, total = c["hd"], c["hq"], c["hkv"], c["page"], x["k"].shape[0]
    k, v = (vxfa.desc(x[t].data_ptr(), vxfa.F16, *views.kv_pages(total, ps, hkv, D)) for t in "kv")
    batch = vxfa.paged(x["table"].data_ptr(), x["n_kv"].data_ptr(), x["q_start"].data_ptr(), c["streams"], x["table"].shape[1],
                       max_nq=c["nq"], max_nkv=c["kv"], window=c["window"])
    if "w" in x:
        wd = [vxfa.desc(x[t].data_ptr(), vxfa.F32, *views.weight_pages(total, ps, hkv)) if t in x else None for t in ("w", "w_out")]
    if c["op"] == "evict":
        ev = vxfa.evict(x["to"].data_ptr(), x["to"].shape[1], c["budget"], c["sink"], c["recent"], kept=x["kept"].data_ptr())
        return lambda s: ctx.paged_evict(k, v, wd[0], batch, ev, stream=s)
    T = x["q"].shape[0]
    if c["op"] == "append":
        q = vxfa.desc(x["q"].data_ptr(), vxfa.F32, *views.decoder_q(T, hq, D))
        q_out = vxfa.desc(x["q_out"].data_ptr(), vxfa.F16, *views.decoder_q(T, hq, D, 2))
        w = hkv * D
        new = [vxfa.desc(x[t].data_ptr(), vxfa.F32, (w, T, 1, 1), (4, 4 * w, 4 * w * T, 4 * w * T)) for t in ("k_new", "v_new")]
        rope = vxfa.rope(x["positions"].data_ptr(), D, ROPE_BASE)
        return lambda s: ctx.paged_append(*new, batch, k, v, rope=rope, q=q, q_out=q_out, stream=s)
    q = vxfa.desc(x["q"].data_ptr(), vxfa.F16, *views.decoder_q(T, hq, D, 2))
    dst = vxfa.desc(x["dst"].data_ptr(), vxfa.F16, *views.dst(D, hq, T, elt=2))
    scale = 1.0 / math.sqrt(D)
    if c["weights"]:
        return lambda s: ctx.flash_attn_ext_paged(q, k, v, batch, dst, scale, c["bias"], c["cap"], weights_in=wd[0], weights=wd[1], stream=s)
    return lambda s: ctx.flash_attn_ext_paged(q, k, v, batch, dst, scale, c["bias"], c["cap"], stream=s)


def run(state):
    c, x = state["case"], state["x"]
    if not own:
        return {"append": _append, "attend": _attend, "evict": _evict}[c["op"]](c, x)
    if "call" not in state:
        state["call"] = _call(c, x)
    state["call"](torch.cuda.current_stream().cuda_stream)
    if c["op"] == "append":
        return {"k": x["k"], "v": x["v"], "q": x["q_out"]}
    if c["op"] == "evict":
        return {"k": x["k"], "v": x["v"], "weights": x["w"], "kept": x["kept"]}
    return {"dst": x["dst"], "weights": x["w_out"]} if c["weights"] else {"dst": x["dst"]}


# ---- work and exact answers ------------------------------------------------------------------------------------------


def work(case):
    """Every live row of K and V, queries and accumulators read once; outputs written once; two products of hd
    multiply-adds for every live pair and query head. (A ragged case's sizes are drawn with its inputs: the mean of 16
    draws.)"""
    c = case
    D, hq, hkv = c["hd"], c["hq"], c["hkv"]
    by = fl = 0
    draws = 16 if c["ragged"] else 1
    for seed in range(draws):
        for n, t in zip(*_sizes(c, seed)):
            if c["op"] == "append":
                by += t * (2 * hkv + hq) * D * (4 + 2)
                continue
            if c["op"] == "evict":
                r = min(n, c["budget"])
                by += 4 * n * hkv + r * hkv * (2 * (4 * D + 4) + 4)
                continue
            w = c["window"] or n
            rows = min(n, w + t - 1)
            by += 4 * rows * hkv * D + 4 * t * hq * D + (8 * n * hkv if c["weights"] else 0)
            fl += 4 * D * hq * sum(min(n - t + i + 1, w) for i in range(t))
    return {"bytes": by / draws, "flops": fl / draws}


def exact(case, seed):
    c, x = case, _inputs(case, seed)
    kv, nq = _sizes(c, seed)
    D, hkv, ps, group = c["hd"], c["hkv"], c["page"], c["hq"] // c["hkv"]

    def turned(t, positions):
        # each pair's angle is the previous one's times a factor
        out, th = t.double().clone(), positions.double()
        for i in range(D // 2):
            co, si = th.cos()[:, None], th.sin()[:, None]
            a, b = t[..., 2 * i].double(), t[..., 2 * i + 1].double()
            out[..., 2 * i], out[..., 2 * i + 1] = a * co - b * si, a * si + b * co
            th = th * ROPE_BASE ** (-2.0 / D)
        return out

    if c["op"] == "append":
        k, v = x["k"].double(), x["v"].double()
        kn, vn = turned(x["k_new"].view(-1, hkv, D), x["positions"]), x["v_new"].view(-1, hkv, D).double()
        t0 = 0
        for s, (n, t) in enumerate(zip(kv, nq)):
            rows = torch.arange(n - t, n, device="cuda")
            pages = x["table"][s][rows // ps].long()
            k[pages, rows % ps], v[pages, rows % ps] = kn[t0:t0 + t], vn[t0:t0 + t]
            t0 += t
        return {"k": k, "v": v, "q": turned(x["q"], x["positions"])}
    if c["op"] == "evict":
        k, v, w, kept = x["k"].double(), x["v"].double(), x["w"].double(), x["kept"]
        for s, n in enumerate(kv):
            rows = torch.arange(n, device="cuda")
            pages = x["table"][s][rows // ps].long()
            score = x["w"][pages, :, rows % ps].cpu()          # [row, head]
            for h in range(hkv):
                ends = {j for j in range(n) if j < c["sink"] or j >= n - c["recent"]}
                one = score[:, h].tolist()
                mid = sorted((-one[j], j) for j in range(n) if j not in ends)
                at = torch.tensor(sorted(ends | {j for _, j in mid[:max(0, c["budget"] - len(ends))]}), device="cuda")
                r = torch.arange(len(at), device="cuda")
                to, src = x["to"][s][r // ps].long(), pages[at]
                kept[s, h, :len(at)] = at.int()
                k[to, r % ps, h], v[to, r % ps, h] = x["k"][src, at % ps, h].double(), x["v"][src, at % ps, h].double()
                w[to, h, r % ps] = x["w"][src, h, at % ps].double()
        return {"k": k, "v": v, "weights": w, "kept": kept}
    dst = torch.zeros((sum(nq), c["hq"], D), device="cuda", dtype=torch.float64)
    w = x["w_out"].double() if c["weights"] else None
    n2 = 2 ** int(math.log2(c["hq"]))
    t0 = 0
    for s, (n, t) in enumerate(zip(kv, nq)):
        rows = torch.arange(n, device="cuda")
        pages = x["table"][s][rows // ps].long()
        for h in range(hkv):
            k, v = x["k"][pages, rows % ps, h].double(), x["v"][pages, rows % ps, h].double()
            total = torch.zeros(n, device="cuda", dtype=torch.float64)
            for g in range(h * group, (h + 1) * group):
                slope = 0.0
                if c["bias"]:
                    slope = 2.0 ** (-c["bias"] * (g + 1) / n2) if g < n2 else 2.0 ** (-c["bias"] / 2 / n2 * (2 * (g - n2) + 1))
                for i0 in range(0, t, 2048):
                    i = torch.arange(i0, min(t, i0 + 2048), device="cuda")
                    p = (n - t + i)[:, None]
                    a = x["q"][t0 + i, g].double() @ k.t().contiguous() / math.sqrt(D)
                    if c["cap"]:
                        a = c["cap"] * torch.tanh(a / c["cap"])
                    a = a + slope * (rows[None] - p)
                    off = (rows[None] > p) | ((rows[None] <= p - c["window"]) if c["window"] else torch.zeros((), dtype=torch.bool, device="cuda"))
                    a = torch.softmax(a.masked_fill(off, float("-inf")), -1)
                    dst[t0 + i, g] = a @ v
                    total += a.sum(0)
            if w is not None:
                w[pages, h, rows % ps] = x["w"][pages, h, rows % ps].double() + total
        t0 += t
    return {"dst": dst, "weights": w} if c["weights"] else {"dst": dst}
