"""One attention block of a decoder, step by step over a paged cache: norm,
quantized projection, plan of pages and slots, append, attention, quantized
output projection, norm with residual, all on one context's stream, with
nothing read back between steps.  Then a beam search over the same block: the
prompt in one step, its tokens' log probabilities, beams that fork and are given
back, and a pool that is made smaller at the end.

    python examples/paged_decode.py            # a few requests, checked on the CPU

The lengths, the free list's head and the block table stay on the device: a
step's kv_lens are the next one's seq_lens, its counts the next one's head.

Rows.  The plan numbers a step's new tokens, the attention its requests.  Here row
r is both, so the requests that take a token in a step stand in front of those
that pause (feed()); a program with any other order gathers the rows of k and v by
token_request, or those of q by token_starts.
"""
import os
import sys

import numpy as np

sys.path.insert(0, os.path.dirname(os.path.dirname(os.path.abspath(__file__))))
from mlx_amd import abi, runtime  # noqa: E402
from oracle import oracle as O  # noqa: E402

F16, F32 = abi.FLOAT16, abi.FLOAT32


class Linear:
    """A quantized layer on the device, and its weights on the host."""

    def __init__(self, ctx, N, K, seed, bits=4, group=64):
        _, w, s, b, _ = O.make_problem(1, K, N, bits, group, F16, F16, seed=seed)
        self.ctx, self.N, self.K, self.bits, self.group = ctx, N, K, bits, group
        self.bufs = [ctx.upload(a) for a in (w, s, b)]
        self.weights = O.dequantize(w, s, b, K, group, bits, F16, F32)

    def __call__(self, x, out, M):
        self.ctx.quantized_matmul(x, *self.bufs, out, M, self.K, self.N, self.group, self.bits, F16, F16, F16)


class Block:
    """norm -> qkv -> paged attention -> output projection -> residual and the next norm, in f16."""

    def __init__(self, ctx, dim, heads, kv_heads, head_dim, requests, pages, page, max_pages, seed=1, tokens=None):
        self.ctx, self.dim, self.H, self.Hk, self.D = ctx, dim, heads, kv_heads, head_dim
        self.R, self.pages, self.page, self.cols = requests, pages, page, max_pages
        self.q_len, self.kv_len = heads * head_dim, kv_heads * head_dim
        rng = np.random.default_rng(seed)
        self.qkv = Linear(ctx, self.q_len + 2 * self.kv_len, dim, seed + 1)
        self.proj = Linear(ctx, dim, self.q_len, seed + 2)
        self.norm_w = [(1 + 0.1 * rng.standard_normal(dim)).astype(np.float16) for _ in range(3)]
        self.norms = [ctx.upload(w.view(np.uint16)) for w in self.norm_w]
        f16 = lambda *shape: ctx.alloc(int(np.prod(shape)) * 2)  # noqa: E731
        i32 = lambda n: ctx.alloc(n * 4)  # noqa: E731
        R, T = requests, tokens or requests
        self.T = T
        self.x, self.normed, self.fused = f16(T, dim), f16(T, dim), f16(T, self.qkv.N)
        self.att, self.out, self.h, self.next = f16(T, self.q_len), f16(T, dim), f16(T, dim), f16(T, dim)
        self.kc, self.vc = (f16(pages, kv_heads, page, head_dim) for _ in range(2))
        self.free = ctx.upload(np.arange(pages, dtype=np.int32)[::-1].copy())
        self.table = ctx.upload(np.full((R, max_pages), -1, np.int32))
        self.new = i32(R)
        self.lens, self.counts = [i32(R), i32(R)], [i32(4), i32(4)]  # this step's and the next one's
        self.slots, self.starts = i32(T), i32(R + 1)

        h = lambda b: b.handle  # noqa: E731
        self.plans = [abi.PagedPlanArgs(
            requests=R, max_tokens=T, max_pages=max_pages, page_size=page, num_pages=pages, free_count=pages,
            seq_lens=h(self.lens[i]), new_lens=h(self.new), free_pages=h(self.free), free_head=h(self.counts[i]),
            block_table=h(self.table), slots=h(self.slots), token_starts=h(self.starts), kv_lens=h(self.lens[1 - i]),
            counts=h(self.counts[1 - i])) for i in range(2)]
        self.append = abi.PagedAppendArgs(
            tokens=T, kv_heads=kv_heads, head_dim=head_dim, page_size=page, num_pages=pages, in_dtype=F16, cache_dtype=F16,
            k_offset=self.q_len, k_row_stride=self.qkv.N, v_offset=self.q_len + self.kv_len, v_row_stride=self.qkv.N,
            k=h(self.fused), v=h(self.fused), slots=h(self.slots), k_cache=h(self.kc), v_cache=h(self.vc))
        self.attention = [abi.PagedAttentionArgs(
            requests=R, heads=heads, kv_heads=kv_heads, head_dim=head_dim, page_size=page, num_pages=pages, max_pages=max_pages,
            dtype=F16, scale=head_dim ** -0.5, q_row_stride=self.qkv.N, q=h(self.fused), k_cache=h(self.kc), v_cache=h(self.vc),
            block_table=h(self.table), kv_lens=h(self.lens[1 - i]), out=h(self.att)) for i in range(2)]
        self.chunks = [abi.PagedChunkArgs(
            requests=R, tokens=T, heads=heads, kv_heads=kv_heads, head_dim=head_dim, page_size=page, num_pages=pages, max_pages=max_pages,
            dtype=F16, scale=head_dim ** -0.5, q_row_stride=self.qkv.N, q=h(self.fused), k_cache=h(self.kc), v_cache=h(self.vc),
            block_table=h(self.table), token_starts=h(self.starts), seq_lens=h(self.lens[i]), kv_lens=h(self.lens[1 - i]),
            out=h(self.att)) for i in range(2)]
        self.first = abi.BlockNormArgs(rows=T, dim=dim, pre_norm=abi.NORM_RMS, x_dtype=F16, residual_dtype=F16, weight_dtype=F16,
                                       residual_scale=1.0, eps=1e-5, residual=h(self.x), pre_weight=h(self.norms[0]), out=h(self.normed))
        self.last = abi.BlockNormArgs(rows=T, dim=dim, post_norm=abi.NORM_RMS, pre_norm=abi.NORM_RMS, x_dtype=F16, residual_dtype=F16,
                                      weight_dtype=F16, residual_scale=1.0, eps=1e-5, x=h(self.out), residual=h(self.x),
                                      post_weight=h(self.norms[1]), pre_weight=h(self.norms[2]), residual_out=h(self.h), out=h(self.next))
        self.turn = 0

    def feed(self, x, new=None):
        """A step's inputs, a row per request, and which of them take a token: all, or 1s and then 0s."""
        new = np.ones(self.R, np.int32) if new is None else np.asarray(new, np.int32)
        if new.shape != (self.R,) or ((new != 0) & (new != 1)).any() or (np.diff(new) > 0).any():
            raise ValueError(f"one token or none per request, those with one first: {new.tolist()}")
        self.x.upload(x.view(np.uint16))
        self.new.upload(new)

    def feed_rows(self, x, new):
        """Inputs of a step in chunks: a row per new token, request after request, new[r] of them for request r."""
        rows = np.zeros((self.T, self.dim), np.float16)
        rows[:len(x)] = x
        self.x.upload(rows.view(np.uint16))
        self.new.upload(np.asarray(new, np.int32))

    def step(self, chunks=False):
        """One token for each request that feed() gave one; the others' rows are computed and thrown away.  chunks: the rows of
        feed_rows(); rows of att behind them are what they were."""
        c, i = self.ctx, self.turn
        c.block_norm(self.first)
        self.qkv(self.normed, self.fused, self.T)
        c.paged_plan(self.plans[i])
        c.paged_append(self.append)
        if chunks:
            c.paged_chunk_attention(self.chunks[i])
        else:
            c.paged_attention(self.attention[i])
        self.proj(self.att, self.out, self.T)
        c.block_norm(self.last)
        self.turn = 1 - i

    def reference(self, x, past, new):
        """The same step in 64 bits, rows that take no token 0; `past`: each request's keys and values so far, extended in place."""
        def rms(v, w):
            return v / np.sqrt((v * v).mean(-1, keepdims=True) + 1e-5) * w.astype(np.float64)

        x = x.astype(np.float64)
        fused = rms(x, self.norm_w[0]) @ self.qkv.weights.astype(np.float64).T
        att = np.zeros((self.R, self.q_len))
        on = np.asarray(new, bool)
        for r in np.flatnonzero(on):
            k, v = (fused[r, at:at + self.kv_len].reshape(self.Hk, 1, self.D) for at in (self.q_len, self.q_len + self.kv_len))
            past[r] = (k, v) if past[r] is None else tuple(np.concatenate([o, n], 1) for o, n in zip(past[r], (k, v)))
            q = fused[r, :self.q_len].reshape(self.Hk, -1, self.D)
            s = q @ past[r][0].transpose(0, 2, 1) / np.sqrt(self.D)
            p = np.exp(s - s.max(-1, keepdims=True))
            att[r] = ((p / p.sum(-1, keepdims=True)) @ past[r][1]).reshape(-1)
        h = x + rms(att @ self.proj.weights.astype(np.float64).T, self.norm_w[1])
        return h * on[:, None], rms(h, self.norm_w[2]) * on[:, None]

    def free_all(self):
        for b in [*self.qkv.bufs, *self.proj.bufs, *self.norms, *self.lens, *self.counts, self.x, self.normed, self.fused, self.att, self.out,
                  self.h, self.next, self.kc, self.vc, self.free, self.table, self.new, self.slots, self.starts]:
            b.free()


def run(ctx, steps=20, requests=3, dim=512, heads=8, kv_heads=2, head_dim=64, page=4, seed=7, running=None):
    """Decodes `steps` tokens for each request; returns the worst error of a step, relative to its largest value.
    running: at which steps only that many requests take a token ({step: n})."""
    pages = requests * -(-steps // page) + 2
    block = Block(ctx, dim, heads, kv_heads, head_dim, requests, pages, page, -(-steps // page), seed)
    rng, past, worst, lens = np.random.default_rng(seed), [None] * requests, 0.0, np.zeros(requests, np.int32)
    try:
        for i in range(steps):
            x = rng.standard_normal((requests, dim)).astype(np.float16)
            new = (np.arange(requests) < (running or {}).get(i, requests)).astype(np.int32)
            block.feed(x, new)
            block.step()
            lens += new
            for buf, want in zip((block.h, block.next), block.reference(x, past, new)):
                got = buf.download(np.uint16, want.shape).view(np.float16).astype(np.float64) * new[:, None]
                worst = max(worst, float(np.abs(got - want).max() / max(np.abs(want).max(), 1e-30)))
        got = block.lens[block.turn].download(np.int32, (requests,))
        assert (got == lens).all(), (got, lens)
        return worst
    finally:
        block.free_all()


class Beams:
    """Beams over a Block and a layer of logits: two halves of `width` requests, one of which holds the beams.  A step's
    winners fork from it into the other half, their last pages are copied, and the half that lost is given back."""

    def __init__(self, ctx, block, head, width):
        self.ctx, self.block, self.head, self.width = ctx, block, head, width
        R, T, N, pool = block.R, block.T, head.N, block.pages
        i32 = lambda n: ctx.alloc(n * 4)  # noqa: E731
        h = lambda b: b.handle  # noqa: E731
        self.logits = ctx.alloc(T * N * 2)
        self.tokens, self.scores, self.ids, self.top = i32(T), i32(T), i32(T * width), i32(T * width)
        self.shares = ctx.upload(np.zeros(pool, np.int32))
        self.src, self.dst, self.keep, self.counts = i32(width), i32(width), i32(R), i32(4)
        self.from_, self.to = i32(pool), i32(pool)
        self.score = abi.TokenLogprobsArgs(rows=T, vocab=N, top=width, dtype=F16, scale=1.0, logits=h(self.logits), tokens=h(self.tokens),
                                           logprobs=h(self.scores), top_ids=h(self.ids), top_logprobs=h(self.top))
        where = dict(requests=R, max_pages=block.cols, page_size=block.page, num_pages=pool, free_count=pool, block_table=h(block.table),
                     shares=h(self.shares), free_pages=h(block.free))
        # after a step of turn i the lengths and the list's head are in lens[1 - i] and counts[1 - i], where the next one reads them
        self.forks = [abi.PagedForkArgs(forks=width, src=h(self.src), dst=h(self.dst), lens=h(block.lens[i]), free_head=h(block.counts[i]),
                                        copy_src=h(self.from_), copy_dst=h(self.to), counts=h(self.counts), **where) for i in range(2)]
        self.releases = [abi.PagedReleaseArgs(lens=h(block.lens[i]), keep_lens=h(self.keep), free_head=h(self.counts), kv_lens=h(block.lens[i]),
                                              counts=h(block.counts[i]), **where) for i in range(2)]
        self.compacts = [abi.PagedCompactArgs(max_moves=pool, lens=h(block.lens[i]), table_out=h(block.table), shares_out=h(self.shares),
                                              copy_src=h(self.from_), copy_dst=h(self.to), counts=h(block.counts[i]), **where) for i in range(2)]
        self.copy = abi.PagedCopyArgs(layers=1, kv_heads=block.Hk, head_dim=block.D, page_size=block.page, num_pages=pool, dtype=F16,
                                      copy_src=h(self.from_), copy_dst=h(self.to), k_cache=h(block.kc), v_cache=h(block.vc))

    def step(self, x, new, tokens):
        """The new rows' cache entries, logits and scores: (log probability of each row's token, the best tokens, their log probabilities)."""
        b, n = self.block, len(x)
        b.feed_rows(x, new)
        rows = np.full(b.T, -1, np.int32)
        rows[:len(tokens)] = tokens
        self.tokens.upload(rows)
        b.step(chunks=True)
        self.head(b.next, self.logits, b.T)
        self.ctx.token_logprobs(self.score)
        return (self.scores.download(np.float32, (b.T,))[:n], self.ids.download(np.int32, (b.T, self.width))[:n],
                self.top.download(np.float32, (b.T, self.width))[:n])

    def move(self, src, dst):
        """Requests dst begin as src are; all others end."""
        keep = np.zeros(self.block.R, np.int32)
        keep[dst] = np.iinfo(np.int32).max
        for buf, v in ((self.src, src), (self.dst, dst)):
            buf.upload(np.asarray(v, np.int32))
        self.keep.upload(keep)
        i = self.block.turn
        self.ctx.paged_fork(self.forks[i])
        self.copy.pages = self.width
        self.ctx.paged_copy(self.copy)
        self.ctx.paged_release(self.releases[i])

    def shrink(self, limit):
        """Pages from `limit` on move below it; returns the moves, the pages that stayed behind, and all in use."""
        i = self.block.turn
        self.compacts[i].limit = limit
        self.ctx.paged_compact(self.compacts[i])
        self.copy.pages = self.block.pages
        self.ctx.paged_copy(self.copy)
        return self.block.counts[i].download(np.int32, (4,))[1:].tolist()

    def free_all(self):
        for b in (self.logits, self.tokens, self.scores, self.ids, self.top, self.shares, self.src, self.dst, self.keep, self.counts, self.from_, self.to):
            b.free()


def beams(ctx, prompt=45, width=3, steps=8, dim=512, heads=8, kv_heads=2, head_dim=64, page=4, vocab=1000, seed=11):
    """A prompt and `steps` tokens of `width` beams; returns the worst error of a step's logits, relative to the largest one, and
    of the log probabilities of the best tokens, both against 64 bits."""
    R, cols = 2 * width, -(-(prompt + steps + 1) // page)
    pages = prompt // page + R * (2 + -(-steps // page)) + 2
    block = Block(ctx, dim, heads, kv_heads, head_dim, R, pages, page, cols, seed, tokens=max(prompt, width))
    head = Linear(ctx, vocab, dim, seed + 5)
    search = Beams(ctx, block, head, width)
    rng = np.random.default_rng(seed)
    table = rng.standard_normal((vocab, dim)).astype(np.float16)  # a token's input
    past, worst, worst_log = [None] * R, 0.0, 0.0
    live = list(range(width))  # the half that holds the beams

    def check(x, rows_of, top):
        """The rows' logits in 64 bits, token by token; `past` takes the new keys and values."""
        nonlocal worst, worst_log
        got = search.logits.download(np.uint16, (block.T, vocab)).view(np.float16).astype(np.float64)
        for i, r in enumerate(rows_of):
            one, on = np.zeros((R, dim), np.float16), np.zeros(R, np.int32)
            one[r], on[r] = x[i], 1
            want = block.reference(one, past, on)[1][r] @ head.weights.astype(np.float64).T
            worst = max(worst, float(np.abs(got[i] - want).max() / np.abs(want).max()))
            best = np.sort(got[i])[::-1][:width]
            lse = best[0] + np.log(np.exp(got[i] - best[0]).sum())
            worst_log = max(worst_log, float(np.abs(top[i] - (best - lse)).max()))

    try:
        tokens = rng.integers(0, vocab, prompt)
        _, ids, top = search.step(table[tokens], [prompt] + [0] * (R - 1), tokens[1:])
        check(table[tokens], [0] * prompt, top)
        live, other = list(range(width, R)), list(range(width))
        search.move([0] * width, live)
        for r in live:
            past[r] = past[0]
        beam_tokens, total = ids[-1], top[-1].astype(np.float64)
        for _ in range(steps):
            new = np.zeros(R, np.int32)
            new[live] = 1
            x = table[beam_tokens]
            _, ids, top = search.step(x, new, [])
            check(x, live, top)
            every = total[:, None] + top
            chosen = np.argsort(-every, axis=None, kind="stable")[:width]
            src, beam_tokens, total = chosen // width, ids.reshape(-1)[chosen], every.reshape(-1)[chosen]
            search.move([live[s] for s in src], other)
            for s, r in zip(src, other):
                past[r] = past[live[s]]
            live, other = other, live
        held = (prompt + steps) // page
        used_limit = held + width * (2 + -(-steps // page))
        moves, behind, used = search.shrink(used_limit)
        assert behind == 0 and used <= used_limit and (moves == 0 or used <= pages), (moves, behind, used, used_limit)
        new = np.zeros(R, np.int32)
        new[live] = 1
        x = table[beam_tokens]
        check(x, live, search.step(x, new, [])[2])
        lens = block.lens[block.turn].download(np.int32, (R,))
        assert (lens[live] == prompt + steps + 1).all() and lens.sum() == width * (prompt + steps + 1), lens
        assert block.table.download(np.int32, (R, cols))[live].max() < used_limit
        return worst, worst_log
    finally:
        search.free_all()
        block.free_all()
        for b in head.bufs:
            b.free()


if __name__ == "__main__":
    context = runtime.Context(0)
    error = run(context)
    beam_error, log_error = beams(context)
    context.close()
    print(f"20 steps, 3 requests: largest error {error:.2e} of the largest value")
    print(f"45 tokens of prompt and 9 of 3 beams: logits off by {beam_error:.2e} of the largest, log probabilities by {log_error:.2e}")
    sys.exit(0 if max(error, beam_error) < 1e-2 else 1)
