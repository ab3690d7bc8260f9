"""One attention block of a decoder, step by step over a paged cache: norm,
quantized projection, plan of pages and slots, append, attention, quantized
output projection, norm with residual, all on one context's stream, with
nothing read back between steps.

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

    def __init__(self, ctx, dim, heads, kv_heads, head_dim, requests, pages, page, max_pages, seed=1):
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
        R, T = requests, requests
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

    def step(self):
        """One token for each request that feed() gave one; the others' rows are computed and thrown away."""
        c, i = self.ctx, self.turn
        c.block_norm(self.first)
        self.qkv(self.normed, self.fused, self.R)
        c.paged_plan(self.plans[i])
        c.paged_append(self.append)
        c.paged_attention(self.attention[i])
        self.proj(self.att, self.out, self.R)
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


if __name__ == "__main__":
    context = runtime.Context(0)
    error = run(context)
    context.close()
    print(f"20 steps, 3 requests: largest error {error:.2e} of the largest value")
    sys.exit(0 if error < 1e-2 else 1)
