"""The operators of prompts and of pages in use this framework's speed is measured on.

Each case is one pass as a serving program makes it: attention of chunks of new
tokens over a paged key-value cache; beams that fork requests, copy the pages
they cannot share and give the losers' pages back; pages that finished and cut
requests release; a pool whose pages move below a limit; and the log
probabilities, entropy and top alternatives of rows of logits.

listed() holds the named cases and draw() gives more of the same ranges.  run()
does one pass on what prepare() laid out: in elementary torch operations in 32
bits, or, where `own` is set, by the calls a user makes.  exact() is the same
result in 64 bits, by loops over requests, heads and rows.

The cache of a layer is [pages, kv heads, page size, head dim], for keys and for
values; a page's entry in `shares` counts the requests that hold it beyond the
first; the free list holds pages from its head on.
"""
import math

import torch

own = False

TORCH = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
SIZE = {"f32": 4, "f16": 2, "bf16": 2}

# what the largest listed cases cost; drawn ones stay below
MOST_FLOPS = 2 * 32 * 128 * 16384 * 16385
MOST_CACHE = 5 << 29
MOST_LOGITS = 4096 * 131072


def chunk(name, requests, chunks, tokens, history, heads, kv_heads, dim, page, dtype, ragged=True, window=0, softcap=0.0, fused=False):
    return {"name": name, "op": "chunk", "requests": requests, "chunks": chunks, "tokens": tokens, "history": history, "heads": heads,
            "kv_heads": kv_heads, "dim": dim, "page": page, "dtype": dtype, "ragged": ragged, "window": window, "softcap": softcap,
            "fused": fused}


def beam(name, sources, forks, length, page, layers, kv_heads, dim, dtype):
    return {"name": name, "op": "beam", "sources": sources, "forks": forks, "length": length, "page": page, "layers": layers,
            "kv_heads": kv_heads, "dim": dim, "dtype": dtype}


def release(name, requests, length, page):
    return {"name": name, "op": "release", "requests": requests, "length": length, "page": page}


def compact(name, requests, length, page, layers, kv_heads, dim, dtype):
    return {"name": name, "op": "compact", "requests": requests, "length": length, "page": page, "layers": layers,
            "kv_heads": kv_heads, "dim": dim, "dtype": dtype}


def logprobs(name, rows, vocab, top, dtype, scale=1.0, pad=0):
    return {"name": name, "op": "logprobs", "rows": rows, "vocab": vocab, "top": top, "dtype": dtype, "scale": scale, "pad": pad}


def listed():
    return [
        # a short follow-up question on a context of 4096: latency, and too few rows to fill the card unsplit
        chunk("chunk_follow_up", 1, 1, 64, 4096, 32, 8, 128, 16, "f16", ragged=False),
        # a serving step: four chunks of prompts beside 60 requests that decode, out of the fused projection
        chunk("chunk_mixed", 64, 4, 512, 8192, 32, 8, 128, 16, "bf16", fused=True),
        # the first prompt of a long document: the largest
        chunk("chunk_document", 1, 1, 16384, 0, 32, 8, 128, 64, "bf16", ragged=False),
        # the reference core's own tensor type, odd head dim, group, pages, window and cap
        chunk("chunk_f32_window", 5, 5, 700, 2000, 20, 4, 80, 24, "f32", window=1024, softcap=30.0),
        # beams of one small step, a single layer's cache: latency
        beam("beam_small", 8, 24, 4096, 16, 1, 8, 128, "f16"),
        # many beams over the caches of 32 layers
        beam("beam_layers", 32, 224, 512, 16, 32, 8, 128, "bf16"),
        # a step in which some of 64 requests end
        release("release_step", 64, 4096, 16),
        # a large pool, many requests that end or are cut
        release("release_pool", 2048, 4096, 32),
        # a small pool shrinks: latency
        compact("compact_small", 37, 1000, 24, 1, 4, 64, "f32"),
        # the caches of 16 layers shrink
        compact("compact_layers", 16, 4096, 16, 16, 8, 128, "bf16"),
        # the choice among a few beams' next tokens: latency, and too few rows to fill the card unsplit
        logprobs("logprobs_step", 8, 131072, 20, "f32", scale=0.7),
        # the score of a prompt
        logprobs("logprobs_prompt", 4096, 131072, 8, "bf16"),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choices(["chunk", "beam", "release", "compact", "logprobs"], [6, 2, 2, 2, 4])[0]
    dtype = rng.choice(["f32", "f16", "f16", "bf16", "bf16"])
    page = rng.choice([8, 16, 16, 32, 64, 128, 24])
    kv_heads, dim = rng.choice([1, 2, 3, 4, 8, 8, 16]), rng.choice([64, 80, 96, 128, 128, 128, 192, 256])
    if op == "chunk":
        heads = kv_heads * rng.choice([1, 2, 3, 4, 4, 5, 7, 8, 16])
        requests = _log(rng, 1, 64)
        c = chunk("", requests, rng.randint(1, requests), _log(rng, 1, 16384), rng.choice([0, _log(rng, 1, 32768)]), heads, kv_heads, dim,
                  page, dtype, rng.random() < 0.7, rng.choice([0, 0, 0, 0, _log(rng, 16, 4096)]), rng.choice([0.0, 0.0, 0.0, 30.0]),
                  rng.random() < 0.5)
        # f32 products run at a fraction of the others' rate
        while work(c)["flops"] * (8 if dtype == "f32" else 1) > MOST_FLOPS or _cache_bytes(c) > MOST_CACHE:
            c["tokens"], c["history"] = max(1, c["tokens"] * 2 // 3), c["history"] * 2 // 3
    elif op == "beam":
        sources = _log(rng, 1, 64)
        c = beam("", sources, sources * _log(rng, 1, 8), _log(rng, 1, 16384), page, _log(rng, 1, 32), kv_heads, dim, dtype)
        while _cache_bytes(c) > MOST_CACHE:
            c["layers"], c["length"] = max(1, c["layers"] * 2 // 3), max(1, c["length"] * 2 // 3)
    elif op == "release":
        c = release("", _log(rng, 1, 2048), _log(rng, 1, 4096), page)
    elif op == "compact":
        c = compact("", _log(rng, 1, 64), _log(rng, 1, 16384), page, _log(rng, 1, 16), kv_heads, dim, dtype)
        while _cache_bytes(c) > MOST_CACHE:
            c["layers"], c["length"] = max(1, c["layers"] * 2 // 3), max(1, c["length"] * 2 // 3)
    else:
        c = logprobs("", _log(rng, 1, 4096), _log(rng, 64, 262144), rng.choice([0, 1, 5, 8, 20, 64]), dtype, rng.choice([1.0, 1.0, 0.7, 2.5]),
                     rng.choice([0, 0, 8, 13]))
        c["rows"] = max(1, min(c["rows"], MOST_LOGITS // c["vocab"] * 2 // SIZE[dtype]))
    return {k: v for k, v in c.items() if k != "name"}


# --- sizes -----------------------------------------------------------------------------------


def _part(i, most, whole):
    """The i-th of numbers spread over 0 .. most - 1, or most."""
    return most if whole else int(math.modf((i + 0.5) * 0.6180339887498949)[0] * most)


def _lengths(c):
    """New tokens and tokens held before, by request: the chunks' requests first."""
    new = [max(1, _part(2 * r + 1, c["tokens"] + 1, False) if c["ragged"] else c["tokens"]) if r < c["chunks"] else 1
           for r in range(c["requests"])]
    return new, [_part(r, c["history"], not c["ragged"]) for r in range(c["requests"])]


def _held(c):
    """Tokens held, by request, of the cases that move pages."""
    return [1 + _part(r, c["length"], False) for r in range(c["sources"] if c["op"] == "beam" else c["requests"])]


def _pages(n, page):
    return -(-n // page)


def _pool(c):
    """Pages of the pool."""
    if c["op"] == "chunk":
        new, history = _lengths(c)
        return sum(_pages(n + h, c["page"]) for n, h in zip(new, history)) + 3
    live = sum(_pages(n, c["page"]) for n in _held(c))
    if c["op"] == "beam":
        return live + c["forks"] + 5
    return live * 5 // 2 + 3 if c["op"] == "compact" else live + live // 4 + 3


def _cache_bytes(c):
    """Of keys and values, all layers."""
    return 2 * c.get("layers", 1) * _pool(c) * c["kv_heads"] * c["page"] * c["dim"] * SIZE[c["dtype"]]


def _limit(c):
    return _pool(c) * 3 // 5


def _most_moves(c):
    """Live pages that can lie above the limit."""
    return _pool(c) - _limit(c)


# --- inputs --------------------------------------------------------------------------------


def _generator(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _normal(gen, dtype, *shape):
    return torch.empty(*shape, dtype=TORCH[dtype], device="cuda").normal_(generator=gen)


def _order(gen, n):
    """Pages 0 .. n - 1 in any order, as a pool that has been in use hands them out."""
    return torch.randperm(n, generator=gen, device="cuda").to(torch.int32)


def _int(values):
    return torch.tensor(values, dtype=torch.int32, device="cuda")


def _table(order, lens, page, rows, columns):
    """A block table whose requests hold the first pages of `order`, one request after the other; -1 behind them."""
    held = _int([_pages(n, page) for n in lens] + [0] * (rows - len(lens)))
    col = torch.arange(columns, device="cuda")
    at = (torch.cumsum(held, 0) - held)[:, None] + col
    return torch.where(col < held[:, None], order[at.clamp(max=order.shape[0] - 1)], -1).to(torch.int32)


def _inputs(c, seed):
    gen = _generator(seed)
    if c["op"] == "chunk":
        new, history = _lengths(c)
        turn = seed % c["requests"]  # which request is which: another order with another seed, the same work
        new, history = new[turn:] + new[:turn], history[turn:] + history[:turn]
        lens = [n + h for n, h in zip(new, history)]
        H, Hk, D, page, pool = c["heads"], c["kv_heads"], c["dim"], c["page"], _pool(c)
        T = sum(new) + (-sum(new) % 16 if c["fused"] else 0)  # a padded batch: rows behind the last request's
        q = _normal(gen, c["dtype"], T, (H + 2 * Hk) * D)[:, :H * D] if c["fused"] else _normal(gen, c["dtype"], T, H * D)
        starts = [0]
        for n in new:
            starts.append(starts[-1] + n)
        return {"new": new, "history": history, "q": q, "starts": _int(starts), "seq": _int(history), "lens": _int(lens),
                "table": _table(_order(gen, pool), lens, page, c["requests"], _pages(max(lens), page)),
                "kc": _normal(gen, c["dtype"], pool, Hk, page, D), "vc": _normal(gen, c["dtype"], pool, Hk, page, D)}
    if c["op"] == "logprobs":
        T, V = c["rows"], c["vocab"]
        logits = _normal(gen, c["dtype"], T, V + c["pad"])[:, :V].mul_(3.0)
        return {"logits": logits, "tokens": torch.randint(0, V, (T,), generator=gen, device="cuda", dtype=torch.int32)}
    lens, page, pool = _held(c), c["page"], _pool(c)
    turn = seed % len(lens)
    lens = lens[turn:] + lens[:turn]
    columns, live, order = _pages(c["length"], page) + 1, sum(_pages(n, page) for n in lens), _order(gen, pool)
    s = {"shares": torch.zeros(pool, dtype=torch.int32, device="cuda"), "head": _int([live])}
    if c["op"] == "beam":
        S, F = c["sources"], c["forks"]
        s.update(lens=_int(lens + [0] * F), table=_table(order, lens, page, S + F, columns),
                 src=(torch.arange(F, device="cuda") % S).to(torch.int32), dst=torch.arange(S, S + F, dtype=torch.int32, device="cuda"),
                 keep=_int([2 ** 31 - 1] * S + [0] * F),
                 # a list in order, as a compaction leaves it
                 free=torch.cat([order[:live], order[live:].sort()[0]]))
    elif c["op"] == "release":
        R = c["requests"]
        # a third of the requests end, a third are cut, the others stay
        part = torch.rand(R, generator=gen, device="cuda")
        n = _int(lens)
        keep = torch.where(part < 1 / 3, 0, torch.where(part < 2 / 3, (n * part).to(torch.int32), n)).to(torch.int32)
        s.update(lens=n, table=_table(order, lens, page, R, columns), keep=keep, free=order)
        return s
    else:
        s.update(lens=_int(lens), table=_table(order, lens, page, c["requests"], columns), free=order.clone())
    shape = (c["layers"], pool, c["kv_heads"], page, c["dim"])
    s.update(kc=_normal(gen, c["dtype"], *shape), vc=_normal(gen, c["dtype"], *shape))
    return s


def prepare(case, seed):
    state = {"case": case, **_inputs(case, seed)}
    if own:
        # what a program keeps from step to step: the output arrays, the
        # buffer handles and the argument records; the data is the same
        _bind(state)
    return state


# --- the framework's calls --------------------------------------------------------------------

_context = None


def _ctx():
    global _context
    if _context is None:
        from mlx_amd.runtime import Context
        _context = Context(0)
    return _context


def _bind(s):
    from mlx_amd import abi
    c, ctx = s["case"], _ctx()
    DT = {"f32": abi.FLOAT32, "f16": abi.FLOAT16, "bf16": abi.BFLOAT16}

    def buf(t):
        s.setdefault("buffers", []).append(ctx.wrap(t.data_ptr(), (1 + sum((n - 1) * st for n, st in zip(t.shape, t.stride()))) * t.element_size()))
        return s["buffers"][-1].handle

    ints = lambda *shape: torch.empty(*shape, dtype=torch.int32, device="cuda")  # noqa: E731
    floats = lambda *shape: torch.empty(*shape, dtype=torch.float32, device="cuda")  # noqa: E731
    if c["op"] == "chunk":
        T, H, D = s["q"].shape[0], c["heads"], c["dim"]
        s["out"] = {"out": torch.zeros(T, H * D, dtype=TORCH[c["dtype"]], device="cuda"),
                    "lse": torch.zeros(T, H, dtype=torch.float32, device="cuda")}
        s["calls"] = [(ctx.paged_chunk_attention, abi.PagedChunkArgs(
            requests=c["requests"], tokens=T, heads=H, kv_heads=c["kv_heads"], head_dim=D, page_size=c["page"], num_pages=s["kc"].shape[0],
            max_pages=s["table"].shape[1], window=c["window"], dtype=DT[c["dtype"]], scale=D ** -0.5, softcap=c["softcap"],
            q_row_stride=s["q"].stride(0), out_row_stride=H * D, q=buf(s["q"]), k_cache=buf(s["kc"]), v_cache=buf(s["vc"]),
            block_table=buf(s["table"]), token_starts=buf(s["starts"]), seq_lens=buf(s["seq"]), kv_lens=buf(s["lens"]),
            out=buf(s["out"]["out"]), lse=buf(s["out"]["lse"])))]
    elif c["op"] == "logprobs":
        T, k = c["rows"], c["top"]
        o = s["out"] = {"logprobs": floats(T), "entropy": floats(T), "lse": floats(T), "top_ids": ints(T, k), "top_logprobs": floats(T, k)}
        s["calls"] = [(ctx.token_logprobs, abi.TokenLogprobsArgs(
            rows=T, vocab=c["vocab"], top=k, dtype=DT[c["dtype"]], scale=c["scale"], row_stride=s["logits"].stride(0), logits=buf(s["logits"]),
            tokens=buf(s["tokens"]), logprobs=buf(o["logprobs"]), entropy=buf(o["entropy"]), lse=buf(o["lse"]),
            top_ids=buf(o["top_ids"]) if k else None, top_logprobs=buf(o["top_logprobs"]) if k else None))]
    else:
        page, pool, F = c["page"], _pool(c), s["free"].shape[0]
        R, columns = s["table"].shape
        h = {name: buf(s[name]) for name in ("lens", "table", "shares", "free", "head")}
        sizes = dict(requests=R, max_pages=columns, page_size=page, num_pages=pool, free_count=F)
        if c["op"] == "release":
            o = s["out"] = {"lens": ints(R), "free": s["free"], "shares": s["shares"], "counts": ints(4)}
            s["calls"] = [(ctx.paged_release, abi.PagedReleaseArgs(
                **sizes, lens=h["lens"], keep_lens=buf(s["keep"]), block_table=h["table"], shares=h["shares"], free_pages=h["free"],
                free_head=h["head"], kv_lens=buf(o["lens"]), counts=buf(o["counts"])))]
        else:
            n = c["forks"] if c["op"] == "beam" else _most_moves(c)
            o = s["out"] = {"from": ints(n), "to": ints(n), "counts": ints(4), "kc": s["kc"], "vc": s["vc"], "free": s["free"]}
            copied, to, counts = buf(o["from"]), buf(o["to"]), buf(o["counts"])
            copy = (ctx.paged_copy, abi.PagedCopyArgs(
                pages=n, layers=c["layers"], kv_heads=c["kv_heads"], head_dim=c["dim"], page_size=page, num_pages=pool, dtype=DT[c["dtype"]],
                copy_src=copied, copy_dst=to, k_cache=buf(s["kc"]), v_cache=buf(s["vc"])))
            if c["op"] == "beam":
                o.update(lens=s["lens"], table=s["table"], shares=s["shares"], after=ints(4))
                s["calls"] = [
                    (ctx.paged_fork, abi.PagedForkArgs(
                        forks=n, **sizes, src=buf(s["src"]), dst=buf(s["dst"]), lens=h["lens"], block_table=h["table"], shares=h["shares"],
                        free_pages=h["free"], free_head=h["head"], copy_src=copied, copy_dst=to, counts=counts)),
                    copy,
                    (ctx.paged_release, abi.PagedReleaseArgs(
                        **sizes, lens=h["lens"], keep_lens=buf(s["keep"]), block_table=h["table"], shares=h["shares"], free_pages=h["free"],
                        free_head=counts, kv_lens=h["lens"], counts=buf(o["after"])))]
            else:
                o.update(table=torch.empty_like(s["table"]), shares=torch.empty_like(s["shares"]))
                s["calls"] = [
                    (ctx.paged_compact, abi.PagedCompactArgs(
                        **sizes, limit=_limit(c), max_moves=n, lens=h["lens"], block_table=h["table"], shares=h["shares"],
                        table_out=buf(o["table"]), shares_out=buf(o["shares"]), free_pages=h["free"], copy_src=copied, copy_dst=to,
                        counts=counts)),
                    copy]
    torch.cuda.synchronize()  # the plugin has a stream of its own


# --- the plain forms ----------------------------------------------------------------------------


def _seen(c, pos, lens):
    """Which of `lens` tokens the tokens at positions `pos` see."""
    at = torch.arange(lens, device="cuda")
    seen = at <= pos[:, None]
    return seen & (at > pos[:, None] - c["window"]) if c["window"] else seen


def _plain_chunk(s):
    c = s["case"]
    H, Hk, D = c["heads"], c["kv_heads"], c["dim"]
    G, T = H // Hk, s["q"].shape[0]
    out, lse = torch.zeros(T, H * D, dtype=s["q"].dtype, device="cuda"), torch.zeros(T, H, dtype=torch.float32, device="cuda")
    first = 0
    for r, (n, held) in enumerate(zip(s["new"], s["history"])):
        pages = s["table"][r, :_pages(n + held, c["page"])]
        k, v = (cache[pages].transpose(0, 1).reshape(Hk, -1, D)[:, :n + held].float() for cache in (s["kc"], s["vc"]))
        k = k.transpose(1, 2).contiguous()
        step = max(1, (1 << 28) // (H * (n + held)))
        for i in range(0, n, step):
            m = min(step, n - i)
            rows = slice(first + i, first + i + m)
            q = s["q"][rows].float().reshape(m, Hk, G, D).transpose(0, 1).reshape(Hk, m * G, D)
            score = torch.matmul(q, k) * D ** -0.5
            if c["softcap"]:
                score = torch.tanh(score / c["softcap"]) * c["softcap"]
            seen = _seen(c, torch.arange(held + i, held + i + m, device="cuda"), n + held)
            score = torch.where(seen[:, None], score.view(Hk, m, G, -1), -math.inf).view(Hk, m * G, -1)
            most = score.amax(-1, keepdim=True)
            p = torch.exp(score - most)
            total = p.sum(-1, keepdim=True)
            o = torch.matmul(p, v) / total
            out[rows] = o.view(Hk, m, G * D).transpose(0, 1).reshape(m, H * D).to(out.dtype)
            lse[rows] = (most + torch.log(total)).view(Hk, m, G).transpose(0, 1).reshape(m, H)
        first += n
    return {"out": out, "lse": lse}


def _plain_copy(s, src, dst):
    there = src >= 0
    src, dst = src[there].long(), dst[there].long()
    for cache in (s["kc"], s["vc"]):
        cache[:, dst] = cache[:, src]


def _plain_release(s, lens, head, keep):
    """Pages of the columns behind keep lose a holder; those without one return to the list, in order, before its head."""
    page, shares, free = s["case"]["page"], s["shares"], s["free"]
    kept = torch.minimum(lens, keep.clamp(min=0))
    col = torch.arange(s["table"].shape[1], device="cuda")
    gone = (col >= -(-kept // page)[:, None]) & (col < -(-lens // page)[:, None])
    ids = torch.where(gone, s["table"], shares.shape[0]).long().view(-1)  # the others fall behind the pool
    drops = torch.zeros(shares.shape[0] + 1, dtype=torch.int32, device="cuda").index_add_(0, ids, torch.ones_like(ids, dtype=torch.int32))[:-1]
    back = drops > shares
    rank = torch.cumsum(back, 0)
    n = rank[-1]
    at = torch.where(back, head + rank - 1 - n, free.shape[0])
    ids = torch.arange(shares.shape[0], dtype=torch.int32, device="cuda")
    s["free"].copy_(torch.cat([free, free[:1]]).scatter(0, at, ids)[:-1])
    shares.copy_(torch.where(back, 0, shares - drops))
    counts = torch.stack([head[0] - n, n, drops.sum() - n, 0 * n]).to(torch.int32)
    return kept.to(torch.int32), counts


def _plain_beam(s):
    c, page, lens, table = s["case"], s["case"]["page"], s["lens"], s["table"]
    src, dst = s["src"].long(), s["dst"].long()
    n = lens[src]
    col = torch.arange(table.shape[1], device="cuda")
    rows = table[src]
    full, partial = n // page, n % page > 0
    rank = torch.cumsum(partial, 0) - 1
    fresh = s["free"][(s["head"] + rank).clamp(max=s["free"].shape[0] - 1)]
    last = rows.gather(1, full[:, None].long())[:, 0]
    shared = col < full[:, None]
    s["shares"].index_add_(0, rows[shared].long(), torch.ones(1, dtype=torch.int32, device="cuda").expand(rows[shared].shape[0]))
    table[dst] = torch.where(shared, rows, torch.where((col == full[:, None]) & partial[:, None], fresh[:, None], table[dst]))
    lens[dst] = n
    copied, to = torch.where(partial, last, -1), torch.where(partial, fresh, -1)
    counts = torch.stack([s["head"][0] + partial.sum(), shared.sum(), 0 * n[0], 0 * n[0]]).to(torch.int32)
    _plain_copy(s, copied, to)
    kept, after = _plain_release(s, lens, counts[:1], s["keep"])
    lens.copy_(kept)
    return {"from": copied, "to": to, "counts": counts, "kc": s["kc"], "vc": s["vc"], "free": s["free"], "lens": lens, "table": table,
            "shares": s["shares"], "after": after}


def _plain_compact(s):
    c, page, pool, limit, F = s["case"], s["case"]["page"], s["shares"].shape[0], _limit(s["case"]), s["free"].shape[0]
    col = torch.arange(s["table"].shape[1], device="cuda")
    held = (col < -(-s["lens"] // page)[:, None]) & (s["table"] >= 0)
    ids = torch.arange(pool, dtype=torch.int32, device="cuda")
    live = torch.zeros(pool, dtype=torch.bool, device="cuda").index_fill_(0, s["table"][held].long(), True)
    high, low = ids[limit:][live[limit:]], ids[:limit][~live[:limit]]
    n = min(high.shape[0], low.shape[0])
    name = ids.clone()
    name[high[:n].long()] = low[:n]
    shares = s["shares"].clone()
    shares[low[:n].long()] = s["shares"][high[:n].long()]
    shares[high[:n].long()] = 0
    pad = lambda v: torch.cat([v[:n], v.new_full((_most_moves(c) - n,), -1)])  # noqa: E731
    copied, to, left = pad(high), pad(low), low[n:]
    s["free"][F - left.shape[0]:] = left
    _plain_copy(s, copied, to)
    return {"from": copied, "to": to, "counts": _int([F - left.shape[0], n, high.shape[0] - n, 0]) + live.sum() * _int([0, 0, 0, 1]), "kc": s["kc"],
            "vc": s["vc"], "free": s["free"], "table": torch.where(held, name[s["table"].long()], s["table"]).to(torch.int32), "shares": shares}


def _plain_logprobs(s):
    c, V = s["case"], s["case"]["vocab"]
    step = max(1, (1 << 28) // V)
    parts = []
    for i in range(0, c["rows"], step):
        raw = s["logits"][i:i + step].float()
        x = raw * c["scale"]
        most = x.amax(-1, keepdim=True)
        e = torch.exp(x - most)
        total = e.sum(-1, keepdim=True)
        log_total = torch.log(total)
        entropy = log_total - (e * (x - most)).sum(-1, keepdim=True) / total
        token = s["tokens"][i:i + step].long()[:, None]
        at = torch.arange(V, dtype=torch.int32, device="cuda")
        ids = []
        rest = raw.clone()
        for _ in range(c["top"]):
            best = rest.amax(-1, keepdim=True)
            ids.append(torch.where(rest == best, at, V).amin(-1, keepdim=True))
            rest.scatter_(1, ids[-1].long(), -math.inf)
        ids = torch.cat(ids, -1) if ids else at[:0].expand(raw.shape[0], 0)
        parts.append({"logprobs": (x.gather(1, token) - most - log_total)[:, 0], "entropy": entropy[:, 0], "lse": (most + log_total)[:, 0],
                      "top_ids": ids, "top_logprobs": x.gather(1, ids.long()) - most - log_total})
    return {k: torch.cat([p[k] for p in parts]) for k in parts[0]}


def _plain_release_pass(s):
    lens, counts = _plain_release(s, s["lens"], s["head"], s["keep"])
    return {"lens": lens, "free": s["free"], "shares": s["shares"], "counts": counts}


_PLAIN = {"chunk": _plain_chunk, "beam": _plain_beam, "release": _plain_release_pass, "compact": _plain_compact, "logprobs": _plain_logprobs}


def run(state):
    if own:
        for call, args in state["calls"]:
            call(args)
        return state["out"]
    return _PLAIN[state["case"]["op"]](state)


# --- what a pass needs, and what it gives -----------------------------------------------------------


def work(case):
    c = case
    if c["op"] == "chunk":
        H, Hk, D, x = c["heads"], c["kv_heads"], c["dim"], SIZE[c["dtype"]]
        W = c["window"] or 1 << 40
        seen = cached = 0
        new, history = _lengths(c)
        for n, h in zip(new, history):
            # positions h .. h + n - 1 see min(position + 1, W) tokens each
            ramp = max(0, min(n, W - h))
            seen += ramp * h + ramp * (ramp + 1) // 2 + (n - ramp) * min(W, h + n)
            cached += min(h + n, W + n - 1)
        T = sum(new)
        return {"bytes": 2 * cached * Hk * D * x + T * H * (2 * D * x + 4) + 4 * cached // c["page"], "flops": 4 * seen * H * D}
    if c["op"] == "logprobs":
        n = c["rows"] * c["vocab"]
        return {"bytes": n * SIZE[c["dtype"]] + c["rows"] * (16 + 8 * c["top"]), "flops": 6 * n}
    held = [_pages(n, c["page"]) for n in _held(c)]
    if c["op"] == "release":
        # lengths in and out; about half of the pages' entries, counters and places in the list
        return {"bytes": 4 * (3 * c["requests"] + 2 * sum(held)), "flops": 0}
    page = 2 * c["layers"] * c["kv_heads"] * c["page"] * c["dim"] * SIZE[c["dtype"]]
    if c["op"] == "beam":
        # an entry in and out for each page of a fork, its counter in and out twice; the last page in and out
        forked = sum(held[f % c["sources"]] for f in range(c["forks"]))
        return {"bytes": 24 * forked + 2 * c["forks"] * page, "flops": 0}
    moved = sum(held) * 2 // 5
    return {"bytes": 8 * sum(held) + 8 * _pool(c) + 2 * moved * page, "flops": 0}


# --- the same in 64 bits, from the definitions -----------------------------------------------------


def _exact_chunk(c, s):
    H, Hk, D = c["heads"], c["kv_heads"], c["dim"]
    T = s["q"].shape[0]
    out, lse = torch.zeros(T, H, D, dtype=torch.float64, device="cuda"), torch.zeros(T, H, dtype=torch.float64, device="cuda")
    starts = s["starts"].tolist()
    for r, n in enumerate(s["lens"].tolist()):
        first, last = starts[r], starts[r + 1]
        pos = torch.arange(n - (last - first), n, device="cuda")
        ids = s["table"][r, :_pages(n, c["page"])].long()
        for h in range(H):
            k = s["kc"][ids, h // (H // Hk)].reshape(-1, D)[:n].double()
            v = s["vc"][ids, h // (H // Hk)].reshape(-1, D)[:n].double()
            for i in range(first, last, 4096):
                rows = slice(i, min(i + 4096, last))
                x = s["q"][rows, h * D:(h + 1) * D].double() @ k.t() / math.sqrt(D)
                if c["softcap"]:
                    x = c["softcap"] * torch.tanh(x / c["softcap"])
                x = x.masked_fill(~_seen(c, pos[i - first:i - first + x.shape[0]], n), -math.inf)
                lse[rows, h] = torch.logsumexp(x, -1)
                out[rows, h] = torch.exp(x - lse[rows, h][:, None]) @ v
    return {"out": out.view(T, H * D), "lse": lse}


def _exact_logprobs(c, s):
    T = c["rows"]
    log_p, entropy, lse = (torch.zeros(T, dtype=torch.float64, device="cuda") for _ in range(3))
    top = torch.zeros(T, c["top"], dtype=torch.float64, device="cuda")
    for i in range(0, T, 64):
        rows = slice(i, min(i + 64, T))
        x = s["logits"][rows].double() * c["scale"]
        lse[rows] = torch.logsumexp(x, -1)
        every = x - lse[rows][:, None]
        log_p[rows] = every.gather(1, s["tokens"][rows].long()[:, None])[:, 0]
        entropy[rows] = -(torch.exp(every) * every).sum(-1)
        if c["top"]:
            top[rows] = every.sort(-1, descending=True)[0][:, :c["top"]]
    return {"logprobs": log_p, "entropy": entropy, "lse": lse, "top_ids": None, "top_logprobs": top}


def exact(case, seed):
    if case["op"] == "chunk":
        return _exact_chunk(case, _inputs(case, seed))
    if case["op"] == "logprobs":
        return _exact_logprobs(case, _inputs(case, seed))
    return None  # whole numbers, and values that are copied
