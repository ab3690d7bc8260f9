"""Definitions in 64 bits of the operators of prompts and of pages in use, one
request, fork or row at a time, and their calls on small arrays.

Tolerances of the chunk attention.  u is the rounding of one value of the type
(serving_util.ROUND).  A score is off by at most (D + 8) 2^-24 scale sum |q k|,
its exp by that much relative, and so is the sum of exps: twice in the quotient.
Sums over n cached tokens are serial additions, n 2^-24; exp2 and the
rescalings, 64 2^-24.  exp(s - max) is rounded once to a 16-bit type, u of itself,
and in f16 by half of its smallest step at 2^14 times it, 2^-39 of the largest, for each of n tokens.  All of
these weigh values of at most max |v|.  Last, the result is rounded, u of itself.
"""
import math

import torch

from mlx_amd import abi
from serving_util import F16, F32, ROUND, TORCH, Device

CHUNK_WEIGHT = {F32: 0.0, F16: 2.0 ** -11, 2: 2.0 ** -8}


def chunk_reference(q, kc, vc, table, starts, seq, lens, H, window=0, scale=1.0, softcap=0.0, dtype=F32):
    """(out [T, H, D], lse [T, H], tolerance [T, H] in units of max |v|, which rows are a request's) in 64 bits."""
    R, cols = table.shape
    pages, Hk, page, D = kc.shape
    G, T = H // Hk, q.shape[0]
    out = torch.zeros(T, H, D, dtype=torch.float64)
    lse = torch.full((T, H), -math.inf, dtype=torch.float64)
    tol = torch.zeros(T, H, dtype=torch.float64)
    mine = torch.zeros(T, dtype=torch.bool)
    cap = cols * page if pages else 0
    for r in range(R):
        n, s0, s1 = min(max(int(lens[r]), 0), cap), int(starts[r]), min(int(starts[r + 1]), T)
        mine[s0:s1] = True
        if n == 0 or s1 <= s0:
            continue
        t = torch.arange(n)
        ids = table[r].long()[t // page]
        there = (ids >= 0) & (ids < pages)
        ids = torch.where(there, ids, 0)
        pos = min(max(int(seq[r]), 0), cols * page) + torch.arange(s1 - s0)
        seen = there & (t <= pos[:, None]) & ((t > pos[:, None] - window) if window else True)
        for h in range(H):
            k, v = kc[ids, h // G, t % page].double(), vc[ids, h // G, t % page].double()
            qq = q[s0:s1, h * D:(h + 1) * D].double()
            s = scale * (qq @ k.t())
            if softcap > 0:
                s = softcap * torch.tanh(s / softcap)
            s = torch.where(seen, s, -math.inf)
            lse[s0:s1, h] = torch.logsumexp(s, -1)
            some = seen.any(-1)
            p = torch.where(seen, torch.exp(s - s.amax(-1, keepdim=True)), 0.0)
            # a row's own tokens alone: 0 times a value that is not finite is no part of it
            if torch.isfinite(v[there]).all():
                o = p @ torch.where(there[:, None], v, 0.0)
            else:
                o = torch.stack([(p[i][:, None] * v)[seen[i]].sum(0) for i in range(p.shape[0])])
            out[s0:s1, h] = torch.where(some[:, None], o / p.sum(-1, keepdim=True), 0.0)
            size = torch.where(seen, qq.abs() @ k.abs().t(), 0.0).amax(-1)
            ds = (D + 8) * 2.0 ** -24 * abs(scale) * size + 4 * 2.0 ** -24 * torch.where(seen, s.abs(), 0.0).amax(-1)
            if softcap > 0:
                ds = ds + 8 * 2.0 ** -24 * softcap
            tol[s0:s1, h] = 2 * ds + (64 + n) * 2.0 ** -24 + (n * 2.0 ** -39 if dtype == F16 else 0)
    return out, lse, tol, mine


def check_chunk(got, lse, ref, v_max, dtype, what, filled=None):
    """Rows of requests against the definition, the others against what was there (`filled`)."""
    out, want_lse, tol, mine = ref
    T, H, D = out.shape
    got = got.double().view(T, H, D)
    if filled is not None:
        assert (got[~mine] == filled).all(), f"{what}: rows of no request were written"
    want, got, tol = out[mine], got[mine], tol[mine]
    finite = torch.isfinite(want)
    assert torch.equal(torch.isfinite(got), finite), f"{what}: {int((torch.isfinite(got) != finite).sum())} values finite or not"
    assert torch.equal(torch.isnan(got), torch.isnan(want)) and torch.equal(got[~finite].nan_to_num(0, 1, -1), want[~finite].nan_to_num(0, 1, -1)), what
    bound = (tol + CHUNK_WEIGHT[dtype])[..., None] * v_max + ROUND[dtype] * want.abs()
    if dtype == F16:
        bound = bound + 2.0 ** -25
    bound = torch.where(finite, bound, 1.0)
    off = torch.where(finite, (got - want).abs(), 0.0)
    assert (off <= bound).all(), f"{what}: {int((off > bound).sum())} of {off.numel()} values off, worst {float((off / bound).max()):.3g} of the bound"
    if lse is not None:
        got_lse, want_lse = lse.double()[mine], want_lse[mine]
        if filled is not None:
            assert (lse[~mine] == filled).all(), what
        flat = torch.isfinite(want_lse)
        assert torch.equal(got_lse[~flat].nan_to_num(5, 1, -1), want_lse[~flat].nan_to_num(5, 1, -1)), what
        d = (got_lse - want_lse)[flat].abs()
        assert (d <= tol[flat] + 4 * 2.0 ** -24 * want_lse[flat].abs()).all(), f"{what}: lse off by {float(d.max()):.3g}"


def starts_of(new):
    s = [0]
    for n in new:
        s.append(s[-1] + n)
    return torch.tensor(s, dtype=torch.int32)


def table_of(gen, lens, page, cols=None, extra=2):
    """(block table of pages in any order, pages of the pool)"""
    held = [-(-max(n, 0) // page) for n in lens]
    cols = cols or max(1, *held)
    pool = sum(held) + extra
    order = torch.randperm(pool, generator=gen).to(torch.int32)
    table = torch.full((len(lens), cols), -1, dtype=torch.int32)
    at = 0
    for r, n in enumerate(held):
        table[r, :n] = order[at:at + n]
        at += n
    return table, pool


def run_chunk(ctx, dtype, q, kc, vc, table, starts, seq, lens, H, /, window=0, scale=1.0, softcap=0.0, fill=3.0, lse=True, expect=None, **over):
    """One call on uploaded arrays: (out, lse), or the error it returned."""
    pages, Hk, page, D = kc.shape
    T = q.shape[0]
    with Device(ctx) as d:
        out, get = d.new(T, H * D, dtype=TORCH[dtype], fill=fill)
        lse_h, get_lse = d.new(T, H, dtype=torch.float32, fill=fill) if lse else (None, lambda: None)
        a = abi.PagedChunkArgs(
            requests=table.shape[0], tokens=T, heads=H, kv_heads=Hk, head_dim=D, page_size=page, num_pages=pages, max_pages=table.shape[1],
            window=window, dtype=dtype, scale=scale, softcap=softcap, q=d.up(q), k_cache=d.up(kc), v_cache=d.up(vc), block_table=d.up(table),
            token_starts=d.up(starts), seq_lens=d.up(seq), kv_lens=d.up(lens), out=out, lse=lse_h)
        for k, v in over.items():
            setattr(a, k, v)
        rc = ctx.p.op_paged_chunk_attention(ctx.handle, a)
        if expect is not None:
            assert rc == expect, rc
            return None
        assert rc == 0, rc
        return get(), get_lse()


# --- pages in use -------------------------------------------------------------------------


def cut(n, cols, page):
    return min(max(int(n), 0), cols * page)


def up(n, page):
    return -(-n // page)


def ints(v, *shape):
    t = torch.tensor(v, dtype=torch.int32)
    return t.reshape(*shape) if shape else t


def fork_reference(src, dst, lens, table, shares, free, head, page):
    src, dst, lens, shares, free = (list(map(int, x)) for x in (src, dst, lens, shares, free))
    table = [list(map(int, row)) for row in table]
    R, cols, pool, F = len(lens), len(table[0]), len(shares), len(free)
    before, made = list(lens), set()
    head = at = min(max(int(head), 0), F)
    copy_src, copy_dst, taken, shared, missing, out = [], [], 0, 0, 0, 0
    for s, d in zip(src, dst):
        copy_src.append(-1)
        copy_dst.append(-1)
        if not (0 <= s < R and 0 <= d < R and s != d and before[d] <= 0) or d in made:
            out += 1
            continue
        made.add(d)
        n = cut(before[s], cols, page)
        full = n // page
        for c in range(full):
            table[d][c] = table[s][c]
            if 0 <= table[s][c] < pool:
                shares[table[s][c]] += 1
        shared += full
        if n % page:
            last = table[s][full]
            table[d][full] = last
            if 0 <= last < pool:
                if at < F:
                    table[d][full], copy_src[-1], copy_dst[-1] = free[at], last, free[at]
                    taken += 1
                else:
                    table[d][full], n = -1, full * page
                    missing += 1
                at += 1
        lens[d] = n
    return {"lens": ints(lens), "block_table": ints(table), "shares": ints(shares), "copy_src": ints(copy_src), "copy_dst": ints(copy_dst),
            "counts": ints([head + taken, shared, missing, out])}


def release_reference(lens, keep, table, shares, free, head, page):
    shares, free = list(map(int, shares)), list(map(int, free))
    pool, cols = len(shares), table.shape[1]
    head = min(max(int(head), 0), len(free))
    kv, back, entries = [], set(), 0
    for r in range(len(lens)):
        n = cut(lens[r], cols, page)
        kept = min(n, max(0, int(keep[r])))
        kv.append(kept)
        for c in range(up(kept, page), up(n, page)):
            p = int(table[r, c])
            if 0 <= p < pool:
                entries += 1
                if shares[p] == 0:
                    back.add(p)
                else:
                    shares[p] -= 1
    back = sorted(back)
    lost = max(0, len(back) - head)
    free[head - (len(back) - lost):head] = back[lost:]
    return {"kv_lens": ints(kv), "shares": ints(shares), "free_pages": ints(free),
            "counts": ints([max(0, head - len(back)), len(back), entries - len(back), lost])}


def compact_reference(lens, table, shares, free, limit, max_moves, page):
    pool, cols = len(shares), table.shape[1]
    held = [up(cut(n, cols, page), page) for n in lens]
    live = {int(table[r, c]) for r in range(len(lens)) for c in range(held[r]) if 0 <= int(table[r, c]) < pool}
    high, room = sorted(p for p in live if p >= limit), [p for p in range(limit) if p not in live]
    moves = min(len(high), len(room), max_moves)
    name = dict(zip(high[:moves], room))
    new_table, new_shares = table.clone(), list(map(int, shares))
    for r in range(len(lens)):
        for c in range(held[r]):
            new_table[r, c] = name.get(int(table[r, c]), int(table[r, c]))
    for a, b in name.items():
        new_shares[b], new_shares[a] = int(shares[a]), 0
    left, free = room[moves:], list(map(int, free))
    first = max(0, len(free) - len(left))
    free[first:] = left[len(left) - (len(free) - first):]
    fill = lambda v: ints(v + [-1] * (max_moves - moves))  # noqa: E731
    return {"table_out": new_table, "shares_out": ints(new_shares), "free_pages": ints(free), "copy_src": fill(high[:moves]),
            "copy_dst": fill(room[:moves]), "counts": ints([first, moves, len(high) - moves, len(live)])}


# --- log probabilities --------------------------------------------------------------------


def logprobs_reference(logits, tokens, top, scale):
    """Scores in 64 bits of rows without NaN and +infinity, and the absolute tolerance of each kind.  A row of
    n logits: each exp is off by 2^-24 (4 + 2 y) of itself, y its distance to the largest one by log2 e (the
    factor's rounding and that of y), its share of the sum at most 2^-y, so 8 2^-24 in all; a thread adds
    n / 512 and then 70 of them one by one; log and the products round 4 times at the result's size.
    The entropy's second sum weighs each error by y, at most log2 n + 1 on average."""
    x = logits.double() * scale
    T, V = x.shape
    lse = torch.logsumexp(x, -1)
    every = x - lse[:, None]
    p = torch.exp(every)
    p = torch.where(torch.isneginf(x), 0.0, p)
    entropy = torch.where(torch.isneginf(lse), 0.0, -torch.where(p > 0, p * every, 0.0).sum(-1))
    every = torch.where(torch.isneginf(lse)[:, None], -math.inf, every)
    log_p = torch.tensor([float(every[t, i]) if 0 <= i < V else -math.inf for t, i in enumerate(map(int, tokens))], dtype=torch.float64)
    # -0 is 0, ties go to the lowest place
    order = torch.argsort(logits.double() + 0.0, dim=-1, descending=True, stable=True)[:, :top]
    unit = 2.0 ** -24
    base = unit * (12 + V / 512 + 70 + math.log2(V) * 4)
    size = 4 * unit * (scale * logits.double()).masked_fill(torch.isinf(logits.double()), 0).abs().amax(-1)
    return {"lse": lse, "logprobs": log_p, "entropy": entropy, "top_ids": order.to(torch.int32), "top_logprobs": every.gather(1, order)}, \
        {"lse": base + size, "logprobs": base + size, "top_logprobs": (base + size)[:, None], "entropy": (base + size) * (math.log2(V) + 2)}


def run_logprobs(ctx, dtype, logits, tokens, top, /, scale=1.0, offset=0, pad=0, expect=None, **over):
    T, V = logits.shape
    wide = torch.full((T * (V + pad) + offset,), math.nan, dtype=logits.dtype)
    wide[offset:].view(T, V + pad)[:, :V] = logits
    with Device(ctx) as d:
        outs = {k: d.new(*s, dtype=t, fill=9) for k, s, t in [
            ("logprobs", (T,), torch.float32), ("entropy", (T,), torch.float32), ("lse", (T,), torch.float32),
            ("top_ids", (T, top), torch.int32), ("top_logprobs", (T, top), torch.float32)]}
        a = abi.TokenLogprobsArgs(rows=T, vocab=V, top=top, dtype=dtype, scale=scale, logits_offset=offset, row_stride=V + pad,
                                  logits=d.up(wide), tokens=d.up(tokens), **{k: v[0] for k, v in outs.items()})
        for k, v in over.items():
            setattr(a, k, v)
        rc = ctx.p.op_token_logprobs(ctx.handle, a)
        if expect is not None:
            assert rc == expect, rc
            return None
        assert rc == 0, rc
        return {k: v[1]() for k, v in outs.items()}
