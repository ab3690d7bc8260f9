"""The operators of prompts and of pages in use together, with the plan, the
append, the norms and the quantized matmul, as examples/paged_decode.py runs
them; the same captured in a graph; on two contexts at once; beside the products
that use the same workspace; and past 32 bits.

Errors of the logits: the roundings of a decoding step (12 2^-11 of the largest
value, test_gpu_decode_step.py), the weights of the attention, rounded once
(averaged over the tokens), and the logits themselves: 14 2^-11.  The log
probabilities are those of the downloaded logits: serial sums of V / 512 terms
in fp32 and some ten roundings at the size of lse, at most 16."""
import ctypes
import os
import sys

import numpy as np
import pytest
import torch

from mlx_amd import abi, runtime
from prompt_util import check_chunk, chunk_reference, run_chunk, run_logprobs
from serving_util import BF16, F16, F32, Device, randn
from test_gpu_paged_chunk import problem

pytestmark = pytest.mark.gpu

sys.path.insert(0, os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "examples"))


@pytest.mark.parametrize("prompt,width,steps,heads,kv_heads,head_dim,page", [(45, 3, 8, 8, 2, 64, 4), (64, 1, 5, 4, 4, 128, 16), (7, 6, 12, 16, 2, 64, 1),
                                                                             (130, 4, 3, 8, 1, 64, 24)])
def test_beams_against_64_bits(ctx, prompt, width, steps, heads, kv_heads, head_dim, page):
    import paged_decode
    error, log_error = paged_decode.beams(ctx, prompt, width, steps, 512, heads, kv_heads, head_dim, page, vocab=1000, seed=prompt)
    assert error <= 14 * 2.0 ** -11, error
    assert log_error <= 2.0 ** -24 * 16 * (1000 / 512 + 70 + 10), log_error


class Pass:
    """A chunk for some requests, its scores, forks, copies, cuts, a second chunk, the end of all, and the pool made anew."""

    def __init__(self, ctx, seed):
        import paged_decode
        self.ctx, self.R, self.T, self.V = ctx, 6, 40, 600
        self.block = paged_decode.Block(ctx, 512, 8, 2, 64, self.R, 64, 4, 12, seed, tokens=self.T)
        self.head = paged_decode.Linear(ctx, self.V, 512, seed + 5)
        self.beams = paged_decode.Beams(ctx, self.block, self.head, 3)
        up = lambda v: ctx.upload(np.asarray(v, np.int32))  # noqa: E731
        self.bufs = [up([0, 0, 1]), up([3, 4, 5]), up([0, 5, 9, 0, 11, 2]), up([0] * 6)]
        h = [b.handle for b in self.bufs]
        for f in self.beams.forks:
            f.src, f.dst = h[0], h[1]
        # one pass: turn 0, then turn 1; after the first step the lengths are in lens[1]
        self.cut, self.end = self.beams.releases[1], self.beams.releases[0]
        self.cut.keep_lens, self.end.keep_lens = h[2], h[3]
        self.beams.compacts[0].limit = 50
        self.beams.copy.pages = 3

    def feed(self, x, new, tokens):
        self.block.feed_rows(x, new)
        rows = np.full(self.T, -1, np.int32)
        rows[:len(tokens)] = tokens
        self.beams.tokens.upload(rows)

    def run(self):
        c, b = self.ctx, self.beams
        assert self.block.turn == 0
        self.block.step(chunks=True)
        self.head(self.block.next, b.logits, self.T)
        c.token_logprobs(b.score)
        c.paged_fork(b.forks[1])
        c.paged_copy(b.copy)
        c.paged_release(self.cut)
        self.block.step(chunks=True)
        self.head(self.block.next, b.logits, self.T)
        c.token_logprobs(b.score)
        c.paged_release(self.end)
        c.paged_compact(b.compacts[0])
        c.paged_copy(b.copy)

    def state(self):
        b, s, R, T = self.block, self.beams, self.R, self.T
        new = int(b.starts.download(np.int32, (R + 1,))[-1])
        shapes = [("att", b.att, np.uint16, (T, b.q_len)), ("next", b.next, np.uint16, (T, b.dim)), ("kc", b.kc, np.uint16, (64 * 2 * 4 * 64,)),
                  ("vc", b.vc, np.uint16, (64 * 2 * 4 * 64,)), ("table", b.table, np.int32, (R * 12,)), ("free", b.free, np.int32, (64,)),
                  ("shares", s.shares, np.int32, (64,)), ("lens", b.lens[0], np.int32, (R,)), ("counts", b.counts[0], np.int32, (4,)),
                  ("scores", s.scores, np.uint32, (T,)), ("ids", s.ids, np.int32, (T, 3)), ("top", s.top, np.uint32, (T, 3))]
        return {k: (v.download(t, n)[:new] if k in ("att", "next", "scores", "ids", "top") else v.download(t, n)) for k, v, t, n in shapes}

    def free_all(self):
        self.beams.free_all()
        self.block.free_all()
        for b in [*self.head.bufs, *self.bufs]:
            b.free()


def test_pass_in_a_graph(ctx):
    """Captured once and replayed with other inputs, with other calls of the same context between, against the calls made one by one."""
    hip = ctypes.CDLL("libamdhip64.so", mode=os.RTLD_NOW | os.RTLD_GLOBAL)

    def ck(rc):
        assert rc == 0, f"hipError {rc}"

    a, b = Pass(ctx, 3), Pass(ctx, 3)
    stream, graph, ready = ctypes.c_void_p(ctx.stream), ctypes.c_void_p(), ctypes.c_void_p()
    rng = np.random.default_rng(5)
    other = problem(21, BF16, [60, 1, 30], [300, 90, 0], 8, 2, 128, 16)
    want = run_chunk(ctx, BF16, *other, 8, scale=0.1)
    logits = torch.randn(3, 40000, generator=torch.Generator().manual_seed(2))
    want_scores = run_logprobs(ctx, F32, logits, torch.tensor([1, 2, 3], dtype=torch.int32), 5)
    try:
        first = rng.standard_normal((2, 512)).astype(np.float16)
        for p in (a, b):
            p.feed(first, [2, 0, 0, 0, 0, 0], [1])
            p.run()
        ctx.sync()
        ck(hip.hipStreamBeginCapture(stream, 2))
        try:
            a.run()
        finally:
            ck(hip.hipStreamEndCapture(stream, ctypes.byref(graph)))
        ck(hip.hipGraphInstantiate(ctypes.byref(ready), graph, None, None, ctypes.c_size_t(0)))
        for new in ([7, 9, 1, 0, 0, 0], [1, 0, 0, 0, 0, 0], [0] * 6, [9, 12, 6, 0, 0, 0], [12, 4, 4, 0, 0, 0]):
            x = rng.standard_normal((sum(new), 512)).astype(np.float16)
            tokens = rng.integers(0, 600, sum(new))
            for p in (a, b):
                p.feed(x, new, tokens)
            ck(hip.hipGraphLaunch(ready, stream))
            again = run_chunk(ctx, BF16, *other, 8, scale=0.1)
            assert torch.equal(again[0].view(torch.int16), want[0].view(torch.int16)) and torch.equal(again[1], want[1])
            scores = run_logprobs(ctx, F32, logits, torch.tensor([1, 2, 3], dtype=torch.int32), 5)
            assert all(torch.equal(scores[k], want_scores[k]) for k in scores)
            b.run()
            one, two = a.state(), b.state()
            for k in one:
                assert np.array_equal(one[k], two[k]), (new, k)
            assert (one["lens"] == 0).all() and (one["shares"] == 0).all() and one["counts"][1:].tolist() == [0, 0, 0], one["counts"]
    finally:
        if ready:
            hip.hipGraphExecDestroy(ready)
        if graph:
            hip.hipGraphDestroy(graph)
        a.free_all()
        b.free_all()


def test_two_contexts_at_once(ctx):
    """Calls on two streams, none waiting for the other: each context has its own workspace."""
    small = problem(31, F16, [40, 1], [2000, 700], 8, 2, 64, 16)
    large = problem(32, F16, [300, 20], [100, 900], 48, 2, 64, 16)
    logits = [torch.randn(2, 50000, generator=torch.Generator().manual_seed(i)) for i in (1, 2)]
    with runtime.Context(0) as other:
        want = [run_chunk(ctx, F16, *small, 8, scale=0.1), run_chunk(ctx, F16, *large, 48, scale=0.1)]
        scores = [run_logprobs(ctx, F32, x, torch.tensor([5, 7], dtype=torch.int32), 10) for x in logits]
        calls = []
        with Device(ctx) as d0, Device(other) as d1:
            for n, d in enumerate((d0, d1)):
                args, H = ((small, 8), (large, 48))[n]
                q, kc, vc, table, starts, seq, lens = args
                out, get = d.new(q.shape[0], q.shape[1], dtype=torch.float16)
                chunk = abi.PagedChunkArgs(
                    requests=2, tokens=q.shape[0], heads=H, kv_heads=2, head_dim=64, page_size=16, num_pages=kc.shape[0], max_pages=table.shape[1],
                    dtype=F16, scale=0.1, q=d.up(q), k_cache=d.up(kc), v_cache=d.up(vc), block_table=d.up(table), token_starts=d.up(starts),
                    seq_lens=d.up(seq), kv_lens=d.up(lens), out=out)
                outs = {k: d.new(2, *s, dtype=t) for k, s, t in [("lse", (), torch.float32), ("top_ids", (10,), torch.int32),
                                                                 ("top_logprobs", (10,), torch.float32)]}
                score = abi.TokenLogprobsArgs(rows=2, vocab=50000, top=10, dtype=F32, scale=1.0, logits=d.up(logits[n]),
                                              **{k: v[0] for k, v in outs.items()})
                calls.append(((ctx, other)[n], chunk, score, get, outs))
            for _ in range(20):
                for c, chunk, score, _, _ in calls:
                    c.paged_chunk_attention(chunk)
                    c.token_logprobs(score)
            for n, (_, _, _, get, outs) in enumerate(calls):
                assert torch.equal(get().view(torch.int16), want[n][0].view(torch.int16))
                for k, v in outs.items():
                    assert torch.equal(v[1](), scores[n][k]), k


def test_products_between_keep_their_results(ctx, oracle):
    """A split-K product before, between and after calls that use the workspace."""
    x, w, s, b, _ = oracle.make_problem(64, 3584, 4096, 3, 64, F16, F16, seed=3)
    args = problem(41, BF16, [200, 3], [900, 2000], 8, 2, 128, 16)
    logits = torch.randn(4, 100000, generator=torch.Generator().manual_seed(3))
    gen = torch.Generator().manual_seed(4)
    R, cols, page, pool = 40, 16, 4, 9000
    table = torch.randperm(pool, generator=gen)[:R * cols].view(R, cols).to(torch.int32)
    ys, outs, scores, lists = [], [], [], []
    for _ in range(3):
        ys.append(runtime.run_quantized_matmul(ctx, x, w, s, b, 64, 3584, 4096, 64, 3, F16, F16, F16))
        outs.append(run_chunk(ctx, BF16, *args, 8, scale=0.1))
        scores.append(run_logprobs(ctx, F32, logits, torch.tensor([1, 2, 3, 4], dtype=torch.int32), 9))
        with Device(ctx) as d:
            free, get = d.out(torch.arange(pool, dtype=torch.int32))
            counts, get_counts = d.new(4)
            ctx.paged_release(abi.PagedReleaseArgs(
                requests=R, max_pages=cols, page_size=page, num_pages=pool, free_count=pool, lens=d.up(torch.full((R,), 61, dtype=torch.int32)),
                keep_lens=d.up(torch.arange(R, dtype=torch.int32)), block_table=d.up(table), shares=d.up(torch.zeros(pool, dtype=torch.int32)),
                free_pages=free, free_head=d.up(torch.tensor([pool], dtype=torch.int32)), kv_lens=d.new(R)[0], counts=counts))
            lists.append((get(), get_counts()))
    ys.append(runtime.run_quantized_matmul(ctx, x, w, s, b, 64, 3584, 4096, 64, 3, F16, F16, F16))
    assert all(np.array_equal(y, ys[0]) for y in ys)
    assert all(torch.equal(o[0].view(torch.int16), outs[0][0].view(torch.int16)) for o in outs)
    assert all(torch.equal(o[k], scores[0][k]) for o in scores for k in o)
    assert all(torch.equal(p, q) for o in lists for p, q in zip(o, lists[0]))
    back = sorted(int(table[r, c]) for r in range(R) for c in range(-(-min(r, 61) // page), 16))
    assert lists[0][0][pool - len(back):].tolist() == back and lists[0][1].tolist() == [pool - len(back), len(back), 0, 0]


def test_caches_past_32_bits(ctx):
    """Pages at the end of a cache of more than 4 GiB: attention, and copies into it and out of it."""
    Hk, page, D, pages = 8, 64, 256, 17000
    bytes_ = pages * Hk * page * D * 2
    assert bytes_ > 2 ** 32
    kb, vb = ctx.alloc(bytes_), ctx.alloc(bytes_)
    try:
        gen = torch.Generator().manual_seed(4)
        part = randn(gen, F16, 3, 2, Hk, page, D)  # three pages' keys and values
        rows = part.transpose(2, 3).reshape(3, 2, page, Hk * D)
        at = torch.tensor([pages - 1, 3, 5], dtype=torch.int32)
        slots = (at[:, None] * page + torch.arange(page, dtype=torch.int32)).reshape(-1)
        with Device(ctx) as dev:
            ctx.paged_append(abi.PagedAppendArgs(
                tokens=3 * page, kv_heads=Hk, head_dim=D, page_size=page, num_pages=pages, in_dtype=F16, cache_dtype=F16,
                k=dev.up(rows[:, 0].reshape(-1, Hk * D)), v=dev.up(rows[:, 1].reshape(-1, Hk * D)), slots=dev.up(slots),
                k_cache=kb.handle, v_cache=vb.handle))
            # the last page to 7, page 3 to the one before the last
            ctx.paged_copy(abi.PagedCopyArgs(pages=2, layers=1, kv_heads=Hk, head_dim=D, page_size=page, num_pages=pages, dtype=F16,
                                             copy_src=dev.up(torch.tensor([pages - 1, 3], dtype=torch.int32)),
                                             copy_dst=dev.up(torch.tensor([7, pages - 2], dtype=torch.int32)), k_cache=kb.handle, v_cache=vb.handle))
            n = torch.tensor([3 * page], dtype=torch.int32)
            small = torch.arange(3, dtype=torch.int32)[None]
            for T, H, table in [(5, 16, [pages - 1, pages - 2, 5]), (150, 128, [7, pages - 2, 5])]:
                q = randn(gen, F16, T, H * D)
                out_h, out_get = dev.new(T, H * D, dtype=torch.float16)
                ctx.paged_chunk_attention(abi.PagedChunkArgs(
                    requests=1, tokens=T, heads=H, kv_heads=Hk, head_dim=D, page_size=page, num_pages=pages, max_pages=3, dtype=F16, scale=D ** -0.5,
                    q=dev.up(q), k_cache=kb.handle, v_cache=vb.handle, block_table=dev.up(torch.tensor([table], dtype=torch.int32)),
                    token_starts=dev.up(torch.tensor([0, T], dtype=torch.int32)), seq_lens=dev.up(n - T), kv_lens=dev.up(n), out=out_h))
                ref = chunk_reference(q, part[:, 0].contiguous(), part[:, 1].contiguous(), small, torch.tensor([0, T]), n - T, n, H,
                                      scale=D ** -0.5, dtype=F16)
                check_chunk(out_get(), None, ref, float(part.double().abs().max()), F16, f"past 32 bits, {T}")
    finally:
        kb.free()
        vb.free()


def test_rows_past_32_bits(ctx):
    """Rows of q, out and logits whose elements lie beyond 2^32."""
    H, D, stride = 2, 64, 2 ** 31 + 8
    q = ctx.alloc((2 * stride + H * D) * 2)
    out = ctx.alloc((2 * stride + H * D) * 2)
    try:
        gen = torch.Generator().manual_seed(6)
        rows = randn(gen, F16, 3, H * D)
        kc, vc = randn(gen, F16, 2, 1, 16, D), randn(gen, F16, 2, 1, 16, D)
        base = [ctypes.c_void_p.from_address(b.handle).value for b in (q, out)]
        parts = [[ctx.wrap(p + i * stride * 2, H * D * 2) for i in range(3)] for p in base]
        try:
            for b, x in zip(parts[0], rows):
                b.upload(x.view(torch.int16).numpy())
            with Device(ctx) as d:
                i = lambda *v: d.up(torch.tensor(v, dtype=torch.int32))  # noqa: E731
                ctx.paged_chunk_attention(abi.PagedChunkArgs(
                    requests=1, tokens=3, heads=H, kv_heads=1, head_dim=D, page_size=16, num_pages=2, max_pages=2, dtype=F16, scale=0.125,
                    q_row_stride=stride, out_row_stride=stride, q=q.handle, k_cache=d.up(kc), v_cache=d.up(vc), block_table=i(1, 0),
                    token_starts=i(0, 3), seq_lens=i(17), kv_lens=i(20), out=out.handle))
                got = torch.stack([torch.from_numpy(b.download(np.int16, (H * D,))).view(torch.float16) for b in parts[1]])
                lse, get = d.new(3, dtype=torch.float32)
                ctx.token_logprobs(abi.TokenLogprobsArgs(rows=3, vocab=H * D, dtype=F16, scale=1.0, row_stride=stride, logits=q.handle, lse=lse))
                assert (get().double() - torch.logsumexp(rows.double(), -1)).abs().max() < 1e-5
            ref = chunk_reference(rows, kc, vc, torch.tensor([[1, 0]]), torch.tensor([0, 3]), torch.tensor([17]), torch.tensor([20]), H,
                                  scale=0.125, dtype=F16)
            check_chunk(got, None, ref, float(vc.abs().max()), F16, "rows")
        finally:
            for b in [*parts[0], *parts[1]]:
                b.free()
    finally:
        q.free()
        out.free()


def test_wrapped_memory(ctx):
    """Operands that start on any element of an allocation and end with it."""
    hip = ctypes.CDLL("libamdhip64.so", mode=os.RTLD_NOW | os.RTLD_GLOBAL)
    size, p = 2 << 20, ctypes.c_void_p()
    assert hip.hipMalloc(ctypes.byref(p), ctypes.c_size_t(size)) == 0
    try:
        args = problem(51, F16, [20, 1], [40, 9], 4, 2, 64, 16)
        want = run_chunk(ctx, F16, *args, 4, scale=0.125)
        for shift in (2, 6):
            n = args[0].numel() * 2
            b = ctx.wrap(p.value + size - n, n)
            o = ctx.wrap(p.value + shift, n)
            b.upload(args[0].view(torch.int16).numpy())
            run_chunk(ctx, F16, *args, 4, scale=0.125, q=b.handle, out=o.handle)
            assert np.array_equal(o.download(np.int16, (21, 256)), want[0].view(torch.int16).numpy())
            b.free()
            o.free()
        logits = torch.randn(3, 5001, generator=torch.Generator().manual_seed(9)).half()
        scores = run_logprobs(ctx, F16, logits, torch.tensor([1, 2, 5000], dtype=torch.int32), 7)
        b = ctx.wrap(p.value + size - logits.numel() * 2, logits.numel() * 2)
        b.upload(logits.view(torch.int16).numpy())
        again = run_logprobs(ctx, F16, logits, torch.tensor([1, 2, 5000], dtype=torch.int32), 7, logits=b.handle)
        assert all(torch.equal(again[k], scores[k]) for k in again)
        b.free()
    finally:
        ctx.sync()
        assert hip.hipFree(p) == 0
