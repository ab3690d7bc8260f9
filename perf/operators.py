"""The paged decode operators this framework's speed is measured on.

Each case is one pass through one operator of a decoding step over a paged
key-value cache: the plan that gives new tokens their pages and slots, the
append that writes their keys and values there, the attention of one new token
per request over the cache, and the norms around a block fused with its gate
and residual.

listed() holds the named cases and draw() gives more of the same ranges.  run()
does one pass on what prepare() laid out: in elementary torch operations in 32
bits, or, where `own` is set, by the calls a user makes.  exact() is the same
result in 64 bits, by loops over requests and rows.

The cache of a layer is [pages, kv heads, page size, head dim], for keys and for
values; a token's slot is its page times the page size plus its place there.
"""
import math

import torch

own = False

TORCH = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
SIZE = {"f32": 4, "f16": 2, "bf16": 2}

# the largest listed case reads this much cache; drawn cases stay below it
MOST_BYTES = 8 * 131072 * 8 * 128 * 2 * 2


def plan(name, requests, tokens, length, page):
    return {"name": name, "op": "plan", "requests": requests, "tokens": tokens, "length": length, "page": page}


def append(name, tokens, heads, kv_heads, dim, page, dtype, cache, fused):
    return {"name": name, "op": "append", "tokens": tokens, "heads": heads, "kv_heads": kv_heads, "dim": dim,
            "page": page, "dtype": dtype, "cache": cache, "fused": fused}


def attention(name, requests, length, heads, kv_heads, dim, page, dtype, ragged=True, window=0, softcap=0.0, fused=False):
    return {"name": name, "op": "attention", "requests": requests, "length": length, "heads": heads, "kv_heads": kv_heads,
            "dim": dim, "page": page, "dtype": dtype, "ragged": ragged, "window": window, "softcap": softcap, "fused": fused}


def norm(name, rows, dim, dtype, residual, kind="rms", post=True, gate="none", scale=1.0):
    return {"name": name, "op": "norm", "rows": rows, "dim": dim, "dtype": dtype, "residual": residual, "kind": kind,
            "post": post, "gate": gate, "scale": scale}


def listed():
    return [
        # a decoding step of a small batch: one new token per request; all latency
        plan("plan_decode", 64, 64, 4096, 16),
        # a step that mixes decoding requests with chunks of prompts
        plan("plan_mixed", 1000, 16384, 8192, 32),
        # the same small batch's keys and values, out of one fused projection
        append("append_decode", 64, 32, 8, 128, 16, "bf16", "bf16", True),
        # a chunk of prompts, computed in f32, kept in f16
        append("append_prompt", 8192, 32, 8, 128, 16, "f32", "f16", False),
        # one user, one token, a context of 4096: latency, and too few heads to fill the card unsplit
        attention("attention_one_request", 1, 4096, 32, 8, 128, 16, "f16", ragged=False),
        # a serving batch of ragged contexts, queries out of the fused projection
        attention("attention_batch", 64, 8192, 32, 8, 128, 16, "bf16", fused=True),
        # few requests with long contexts: the largest
        attention("attention_long", 8, 131072, 32, 8, 128, 64, "bf16", ragged=False),
        # the reference core's own tensor type, one head of keys per query head, a sliding window
        attention("attention_f32_window", 23, 2000, 16, 16, 64, 24, "f32", window=1024),
        # one head of keys for all queries, wide heads, capped scores
        attention("attention_shared_head", 37, 5000, 16, 1, 256, 32, "f16", softcap=30.0),
        # one token between two blocks: latency
        norm("norm_one_token", 1, 4096, "f16", "f16"),
        # a chunk of prompts: norm after the block, gate per channel, residual, norm before the next
        norm("norm_prompt", 8192, 4096, "bf16", "bf16", gate="channel"),
        # f32 residual, odd row length, layer norm, a gate for each value, scaled residual
        norm("norm_odd", 1023, 5003, "f16", "f32", kind="layer", gate="full", scale=0.5),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choices(["plan", "append", "attention", "norm"], [2, 2, 6, 3])[0]
    dtype = rng.choice(["f32", "f16", "f16", "bf16", "bf16"])
    page = rng.choice([8, 16, 16, 32, 64, 128, 24])
    if op == "plan":
        requests = _log(rng, 1, 2048)
        return {k: v for k, v in plan("", requests, _log(rng, requests, 32768), _log(rng, 16, 32768), page).items() if k != "name"}
    kv_heads, dim = rng.choice([1, 2, 3, 4, 8, 8, 16]), rng.choice([64, 80, 96, 128, 128, 128, 192, 256])
    heads = kv_heads * rng.choice([1, 2, 3, 4, 4, 5, 7, 8, 16])
    if op == "append":
        c = append("", _log(rng, 1, 8192), heads, kv_heads, dim, page, dtype, rng.choice([dtype, dtype, "f16", "bf16"]), rng.random() < 0.5)
    elif op == "attention":
        requests, length = _log(rng, 1, 256), _log(rng, 1, 131072)
        length = max(1, min(length, MOST_BYTES // (requests * kv_heads * dim * 2 * SIZE[dtype])))
        c = attention("", requests, length, heads, kv_heads, dim, page, dtype, rng.random() < 0.7,
                      rng.choice([0, 0, 0, 0, _log(rng, 16, 4096)]), rng.choice([0.0, 0.0, 0.0, 30.0]), rng.random() < 0.5)
    else:
        c = norm("", _log(rng, 1, 8192), rng.choice([_log(rng, 64, 16384), 64 * _log(rng, 1, 256), 1024 * rng.randint(1, 8)]),
                 dtype, rng.choice([dtype, dtype, "f32"]), rng.choice(["rms", "rms", "layer"]), rng.random() < 0.7,
                 rng.choice(["none", "channel", "row", "full"]), rng.choice([1.0, 1.0, 0.5]))
        c["rows"] = max(1, min(c["rows"], 8192 * 4096 // c["dim"]))
    return {k: v for k, v in c.items() if k != "name"}


# --- inputs --------------------------------------------------------------------------------


def _generator(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _ints(gen, lo, hi, n):
    """n whole numbers of [lo, hi], as the card holds lengths."""
    return torch.randint(lo, hi + 1, (n,), generator=gen, device="cuda", dtype=torch.int32)


def _normal(gen, dtype, *shape):
    return torch.empty(*shape, dtype=TORCH[dtype], device="cuda").normal_(generator=gen)


def _order(gen, n):
    """Pages 0 .. n - 1 in any order, as a pool that has been in use hands them out."""
    return torch.randperm(n, generator=gen, device="cuda").to(torch.int32)


def _pages(c):
    return -(-c["length"] // c["page"])


def _plan_sizes(c):
    """(columns of the block table, pages of the pool)"""
    columns = -(-(c["length"] + c["tokens"]) // c["page"])
    return columns, c["requests"] * _pages(c) + c["requests"] + -(-c["tokens"] // c["page"])


def _inputs(c, seed):
    gen = _generator(seed)
    if c["op"] == "plan":
        R, extra = c["requests"], c["tokens"] - c["requests"]
        columns, pool = _plan_sizes(c)
        seq = _ints(gen, 0, c["length"], R)
        # every request has one token, and a few share the prompts' chunks
        new = torch.ones(R, dtype=torch.int32, device="cuda")
        chunk = max(1, min(R, extra // 512))
        new[:chunk] += extra // chunk
        order = _order(gen, pool)
        held = -(-seq // c["page"])
        ends = torch.cumsum(held, 0)
        col = torch.arange(columns, device="cuda")
        at = (ends - held)[:, None] + col
        table = torch.where(col < held[:, None], order[at.clamp(max=pool - 1)], -1).to(torch.int32)
        # the free list: the pages behind those the requests hold
        return {"seq": seq, "new": new, "free": order, "head": ends[-1:].to(torch.int32), "table": table}
    if c["op"] == "norm":
        T, D = c["rows"], c["dim"]
        given = {"y": _normal(gen, c["dtype"], T, D), "r": _normal(gen, c["residual"], T, D),
                 "pre": _normal(gen, c["dtype"], D).mul_(0.1).add_(1), "post": None, "gate": None, "bias": None}
        if c["post"]:
            given["post"] = _normal(gen, c["dtype"], D).mul_(0.1).add_(1)
        if c["kind"] == "layer":
            given["bias"] = _normal(gen, c["dtype"], D).mul_(0.1)
        if c["gate"] != "none":
            given["gate"] = _normal(gen, c["dtype"], *{"channel": (D,), "row": (T,), "full": (T, D)}[c["gate"]])
        return given
    H, Hk, D, page = c["heads"], c["kv_heads"], c["dim"], c["page"]
    if c["op"] == "append":
        T = c["tokens"]
        pages = -(-T // page) + 64
        slots = (_order(gen, pages)[:, None] * page + torch.arange(page, device="cuda", dtype=torch.int32)).view(-1)[:T].contiguous()
        if c["fused"]:  # queries, keys and values of a token side by side
            qkv = _normal(gen, c["dtype"], T, (H + 2 * Hk) * D)
            k, v = qkv[:, H * D:(H + Hk) * D], qkv[:, (H + Hk) * D:]
        else:
            k, v = _normal(gen, c["dtype"], T, Hk * D), _normal(gen, c["dtype"], T, Hk * D)
        return {"k": k, "v": v, "slots": slots, "kc": _normal(gen, c["cache"], pages, Hk, page, D),
                "vc": _normal(gen, c["cache"], pages, Hk, page, D)}
    R, columns = c["requests"], _pages(c)
    lens = _ints(gen, 1, c["length"], R) if c["ragged"] else torch.full((R,), c["length"], dtype=torch.int32, device="cuda")
    q = _normal(gen, c["dtype"], R, (H + 2 * Hk) * D)[:, :H * D] if c["fused"] else _normal(gen, c["dtype"], R, H * D)
    pool = R * columns
    return {"q": q, "lens": lens, "table": _order(gen, pool).view(R, columns),
            "kc": _normal(gen, c["dtype"], pool, Hk, page, D), "vc": _normal(gen, c["dtype"], pool, Hk, page, D)}


def prepare(case, seed):
    state = {"case": case, **_inputs(case, seed)}
    if own:
        # what a program keeps from step to step: the output arrays, the
        # buffer handles and the argument record; the data is the same
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
        if t is None:
            return None
        s.setdefault("buffers", []).append(ctx.wrap(t.data_ptr(), (1 + sum((n - 1) * st for n, st in zip(t.shape, t.stride()))) * t.element_size()))
        return s["buffers"][-1].handle

    ints = lambda *shape: torch.empty(*shape, dtype=torch.int32, device="cuda")  # noqa: E731
    if c["op"] == "plan":
        R, T = c["requests"], c["tokens"]
        s["out"] = {"table": s["table"], "slots": ints(T), "positions": ints(T), "request": ints(T), "starts": ints(R + 1),
                    "lens": ints(R), "counts": ints(4)}
        o = s["out"]
        columns, pool = _plan_sizes(c)
        s["args"] = abi.PagedPlanArgs(
            requests=R, max_tokens=T, max_pages=columns, page_size=c["page"], num_pages=pool, free_count=pool,
            seq_lens=buf(s["seq"]), new_lens=buf(s["new"]), free_pages=buf(s["free"]), free_head=buf(s["head"]),
            block_table=buf(o["table"]), slots=buf(o["slots"]), positions=buf(o["positions"]), token_request=buf(o["request"]),
            token_starts=buf(o["starts"]), kv_lens=buf(o["lens"]), counts=buf(o["counts"]))
        s["call"] = ctx.paged_plan
    elif c["op"] == "append":
        s["out"] = {"kc": s["kc"], "vc": s["vc"]}
        s["args"] = abi.PagedAppendArgs(
            tokens=c["tokens"], kv_heads=c["kv_heads"], head_dim=c["dim"], page_size=c["page"], num_pages=s["kc"].shape[0],
            k_row_stride=s["k"].stride(0), v_row_stride=s["v"].stride(0), in_dtype=DT[c["dtype"]], cache_dtype=DT[c["cache"]],
            k=buf(s["k"]), v=buf(s["v"]), slots=buf(s["slots"]), k_cache=buf(s["kc"]), v_cache=buf(s["vc"]))
        s["call"] = ctx.paged_append
    elif c["op"] == "attention":
        R, H, D = c["requests"], c["heads"], c["dim"]
        s["out"] = {"out": torch.empty(R, H * D, dtype=TORCH[c["dtype"]], device="cuda"),
                    "lse": torch.empty(R, H, dtype=torch.float32, device="cuda")}
        s["args"] = abi.PagedAttentionArgs(
            requests=R, heads=H, kv_heads=c["kv_heads"], head_dim=D, page_size=c["page"], num_pages=s["kc"].shape[0],
            max_pages=s["table"].shape[1], window=c["window"], scale=D ** -0.5, softcap=c["softcap"], dtype=DT[c["dtype"]],
            q_row_stride=s["q"].stride(0), out_row_stride=H * D, q=buf(s["q"]), k_cache=buf(s["kc"]), v_cache=buf(s["vc"]),
            block_table=buf(s["table"]), kv_lens=buf(s["lens"]), out=buf(s["out"]["out"]), lse=buf(s["out"]["lse"]))
        s["call"] = ctx.paged_attention
    else:
        kind = {"rms": abi.NORM_RMS, "layer": abi.NORM_LAYER}[c["kind"]]
        s["out"] = {"h": torch.empty_like(s["r"]), "n": torch.empty_like(s["y"])}
        s["args"] = abi.BlockNormArgs(
            rows=c["rows"], dim=c["dim"], post_norm=kind if c["post"] else abi.NORM_NONE, pre_norm=kind,
            gate_mode={"none": abi.GATE_NONE, "channel": abi.GATE_CHANNEL, "row": abi.GATE_ROW, "full": abi.GATE_FULL}[c["gate"]],
            residual_scale=c["scale"], eps=1e-5, x_dtype=DT[c["dtype"]], residual_dtype=DT[c["residual"]], weight_dtype=DT[c["dtype"]],
            x=buf(s["y"]), residual=buf(s["r"]), post_weight=buf(s["post"]), post_bias=buf(s["bias"] if c["post"] else None),
            gate=buf(s["gate"]), pre_weight=buf(s["pre"]), pre_bias=buf(s["bias"]), residual_out=buf(s["out"]["h"]), out=buf(s["out"]["n"]))
        s["call"] = ctx.block_norm
    torch.cuda.synchronize()  # the plugin has a stream of its own


# --- the plain forms ----------------------------------------------------------------------------


def _plain_plan(s):
    c, page = s["case"], s["case"]["page"]
    columns, F = s["table"].shape[1], s["free"].shape[0]
    seq, new = s["seq"].clamp(0, columns * page), s["new"].clamp(min=0)
    ends = torch.cumsum(new, 0, dtype=torch.int32)
    starts = torch.cat([ends.new_zeros(1), ends])
    have = (seq + page - 1) // page
    need = ((seq + new + page - 1) // page).clamp(max=columns) - have
    through = torch.cumsum(need, 0, dtype=torch.int32)
    first = through - need + s["head"]
    got = torch.minimum((F - first).clamp(min=0), need)
    lens = torch.minimum(seq + new, (have + got) * page)
    col = torch.arange(columns, dtype=torch.int32, device="cuda")
    at = first[:, None] + col - have[:, None]
    page_at = torch.where(at < F, s["free"][at.clamp(0, F - 1)], -1)
    table = torch.where((col >= have[:, None]) & (col < (have + need)[:, None]), page_at, s["table"])
    t = torch.arange(c["tokens"], dtype=torch.int32, device="cuda")
    live = t < ends[-1]
    r = torch.searchsorted(ends, t, right=True).clamp(max=c["requests"] - 1)
    pos = torch.where(live, seq[r] + t - starts[r], 0)
    there = table[r, (pos // page).clamp(max=columns - 1)]
    slots = torch.where(live & (pos < lens[r]) & (there >= 0), there * page + pos % page, -1)
    counts = torch.stack([s["head"][0] + got.sum(), ends[-1], (need - got).sum(), (seq + new - lens).sum()])
    return {"table": table, "slots": slots, "positions": pos, "request": torch.where(live, r, -1).to(torch.int32), "starts": starts,
            "lens": lens, "counts": counts.to(torch.int32)}


def _plain_append(s):
    c, page = s["case"], s["case"]["page"]
    to, at = s["slots"] // page, s["slots"] % page
    heads = torch.arange(c["kv_heads"], device="cuda")
    for new, cache in ((s["k"], s["kc"]), (s["v"], s["vc"])):
        cache[to[:, None], heads, at[:, None]] = new.float().view(-1, c["kv_heads"], c["dim"]).to(cache.dtype)
    return {"kc": s["kc"], "vc": s["vc"]}


def _plain_attention(s):
    c = s["case"]
    R, H, Hk, D = c["requests"], c["heads"], c["kv_heads"], c["dim"]
    q = s["q"].float().reshape(R, Hk, H // Hk, D)
    k, v = (cache[s["table"]].transpose(1, 2).float().reshape(R, Hk, -1, D) for cache in (s["kc"], s["vc"]))
    score = torch.matmul(q, k.transpose(2, 3).contiguous()) * D ** -0.5
    if c["softcap"]:
        score = torch.tanh(score / c["softcap"]) * c["softcap"]
    at, lens = torch.arange(k.shape[2], device="cuda"), s["lens"][:, None]
    seen = at < lens
    if c["window"]:
        seen = seen & (at >= lens - c["window"])
    score = torch.where(seen[:, None, None], score, -math.inf)
    most = score.amax(-1, keepdim=True).clamp(min=-1e30)
    p = torch.exp(score - most)
    total = p.sum(-1, keepdim=True)
    out = torch.matmul(p, v) / total.clamp(min=1e-37)
    return {"out": out.reshape(R, H * D).to(s["q"].dtype), "lse": (most + torch.log(total)).view(R, H)}


def _plain_norm_of(x, kind, weight, bias):
    if kind == "layer":
        x = x - x.mean(-1, keepdim=True)
    x = x * torch.rsqrt((x * x).mean(-1, keepdim=True) + 1e-5) * weight.float()
    return x if bias is None else x + bias.float()


def _plain_norm(s):
    c = s["case"]
    a = s["y"].float()
    if c["post"]:
        a = _plain_norm_of(a, c["kind"], s["post"], s["bias"])
    if c["gate"] != "none":
        g = s["gate"].float()
        a = a * (g[:, None] if c["gate"] == "row" else g)
    h = s["r"].float() * c["scale"] + a
    n = _plain_norm_of(h, c["kind"], s["pre"], s["bias"])
    return {"h": h.to(s["r"].dtype), "n": n.to(s["y"].dtype)}


_PLAIN = {"plan": _plain_plan, "append": _plain_append, "attention": _plain_attention, "norm": _plain_norm}


def run(state):
    if own:
        state["call"](state["args"])
        return state["out"]
    return _PLAIN[state["case"]["op"]](state)


# --- what a pass needs, and what it gives -----------------------------------------------------------


def work(case):
    c = case
    if c["op"] == "plan":
        R, T = c["requests"], c["tokens"]
        # lengths in and out, starts, three words a token, a word per new page in the list and in the table
        return {"bytes": 4 * (4 * R + 3 * T + 2 * (R // c["page"] + T // c["page"]) + 6), "flops": 0}
    if c["op"] == "append":
        n = 2 * c["tokens"] * c["kv_heads"] * c["dim"]
        return {"bytes": n * (SIZE[c["dtype"]] + SIZE[c["cache"]]) + 4 * c["tokens"], "flops": 0}
    if c["op"] == "attention":
        # the mean of lengths spread evenly over 1 .. length, each cut to the window
        L, W = c["length"], c["window"] or c["length"]
        if c["ragged"]:
            seen = (L + 1) / 2 if W >= L else (W * (W + 1) / 2 + (L - W) * W) / L
        else:
            seen = min(L, W)
        n = c["requests"] * seen
        return {"bytes": 2 * n * c["kv_heads"] * c["dim"] * SIZE[c["dtype"]] + 4 * n / c["page"]
                + c["requests"] * c["heads"] * (2 * c["dim"] * SIZE[c["dtype"]] + 4), "flops": 4 * n * c["heads"] * c["dim"]}
    T, D, x = c["rows"], c["dim"], SIZE[c["dtype"]]
    gate = {"none": 0, "channel": D, "row": T, "full": T * D}[c["gate"]]
    weights = D * (1 + c["post"] + (c["kind"] == "layer"))
    return {"bytes": T * D * 2 * (x + SIZE[c["residual"]]) + (gate + weights) * x, "flops": 12 * T * D}


# --- the same in 64 bits, from the definitions -----------------------------------------------------


def _exact_attention(c, s):
    R, H, Hk, D, page = c["requests"], c["heads"], c["kv_heads"], c["dim"], c["page"]
    out, lse = torch.zeros(R, H, D, dtype=torch.float64, device="cuda"), torch.zeros(R, H, dtype=torch.float64, device="cuda")
    for r, n in enumerate(s["lens"].tolist()):
        first = max(0, n - c["window"]) if c["window"] else 0
        pages = s["table"][r, first // page:-(-n // page)].long()
        cut = slice(first - first // page * page, n - first // page * page)
        for h in range(Hk):
            k = s["kc"][pages, h].reshape(-1, D)[cut].double()
            v = s["vc"][pages, h].reshape(-1, D)[cut].double()
            mine = slice(h * (H // Hk), (h + 1) * (H // Hk))
            x = s["q"][r].double().view(H, D)[mine] @ k.t() / math.sqrt(D)
            if c["softcap"]:
                x = c["softcap"] * torch.tanh(x / c["softcap"])
            lse[r, mine] = torch.logsumexp(x, -1)
            out[r, mine] = torch.exp(x - lse[r, mine][:, None]) @ v
    return {"out": out.view(R, H * D), "lse": lse}


def _exact_norm(c, s):
    def normed(x, weight, bias):
        mean = x.mean(-1, keepdim=True) if c["kind"] == "layer" else 0.0
        x = (x - mean) / torch.sqrt(((x - mean) ** 2).mean(-1, keepdim=True) + 1e-5) * weight.double()
        return x + bias.double() if bias is not None else x

    a = s["y"].double()
    if c["post"]:
        a = normed(a, s["post"], s["bias"])
    if c["gate"] == "row":
        a = s["gate"].double()[:, None] * a
    elif c["gate"] != "none":
        a = s["gate"].double() * a
    h = c["scale"] * s["r"].double() + a
    return {"h": h, "n": normed(h, s["pre"], s["bias"])}


def exact(case, seed):
    c = case
    if c["op"] == "plan":
        return None  # whole numbers
    s = _inputs(c, seed)
    if c["op"] == "norm":
        return _exact_norm(c, s)
    if c["op"] == "attention":
        return _exact_attention(c, s)
    want = {}
    for new, name in ((s["k"], "kc"), (s["v"], "vc")):
        cache = s[name].double().transpose(1, 2).reshape(-1, c["kv_heads"] * c["dim"])
        cache[s["slots"].long()] = new.double()
        want[name] = cache.view(-1, c["page"], c["kv_heads"], c["dim"]).transpose(1, 2)
    return want
