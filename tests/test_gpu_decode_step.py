"""The decoding step's operators together with the quantized matmul, as
examples/paged_decode.py runs them, and the same captured in a graph.

Errors: f16 activations round at every stage (normed input, fused projection,
attention, output projection, both results: 6 roundings of 2^-11, each carried
on by products whose rows average it), so 12 2^-11 = 6e-3 of the largest value."""
import ctypes
import os
import sys

import numpy as np
import pytest

from mlx_amd import abi

pytestmark = pytest.mark.gpu

sys.path.insert(0, os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "examples"))


@pytest.mark.parametrize("requests,heads,kv_heads,head_dim,page,steps", [(3, 8, 2, 64, 4, 20), (1, 4, 4, 128, 16, 35), (9, 16, 2, 64, 1, 6)])
def test_steps_against_64_bits(ctx, requests, heads, kv_heads, head_dim, page, steps):
    import paged_decode
    error = paged_decode.run(ctx, steps, requests, 512, heads, kv_heads, head_dim, page, seed=steps)
    assert error <= 12 * 2.0 ** -11, error


def test_step_in_a_graph(ctx):
    """Plan, append, attention and norms captured once, replayed with other inputs, against the same calls made one by one."""
    import paged_decode
    hip = ctypes.CDLL("libamdhip64.so", mode=os.RTLD_NOW | os.RTLD_GLOBAL)

    def ck(rc):
        assert rc == 0, f"hipError {rc}"

    requests, steps, dim = 5, 6, 512
    blocks = [paged_decode.Block(ctx, dim, 8, 2, 64, requests, 64, 4, 8, seed=3) for _ in range(2)]
    stream, graph, ready = ctypes.c_void_p(ctx.stream), ctypes.c_void_p(), ctypes.c_void_p()
    rng = np.random.default_rng(5)

    def feed():
        x = rng.standard_normal((requests, dim)).astype(np.float16).view(np.uint16)
        new = rng.integers(0, 2, requests).astype(np.int32)
        for b in blocks:
            b.x.upload(x)
            b.new.upload(new)

    try:
        # two steps, so that lengths and counts are back in their first buffers
        blocks[0].step()
        blocks[0].step()
        blocks[1].step()
        blocks[1].step()
        ctx.sync()
        ck(hip.hipStreamBeginCapture(stream, 2))
        try:
            blocks[0].step()
            blocks[0].step()
        finally:
            ck(hip.hipStreamEndCapture(stream, ctypes.byref(graph)))
        ck(hip.hipGraphInstantiate(ctypes.byref(ready), graph, None, None, ctypes.c_size_t(0)))
        for _ in range(steps):
            feed()
            ck(hip.hipGraphLaunch(ready, stream))
            blocks[1].step()
            blocks[1].step()
            for name, dt, n in [("h", np.uint16, requests * dim), ("next", np.uint16, requests * dim), ("table", np.int32, requests * 8),
                                ("slots", np.int32, requests), ("kc", np.uint16, 64 * 2 * 4 * 64)]:
                got, want = (getattr(b, name).download(dt, (n,)) for b in blocks)
                assert np.array_equal(got, want), name
            assert np.array_equal(blocks[0].lens[0].download(np.int32, (requests,)), blocks[1].lens[0].download(np.int32, (requests,)))
    finally:
        if ready:
            hip.hipGraphExecDestroy(ready)
        if graph:
            hip.hipGraphDestroy(graph)
        for b in blocks:
            b.free_all()


def test_rows_short_of_pages_leave_the_others_alone(ctx):
    """A pool of two pages for three requests: the third gets none, and its attention is zero."""
    import paged_decode
    block = paged_decode.Block(ctx, 512, 8, 2, 64, 3, 2, 4, 4, seed=9)
    block.new.upload(np.ones(3, np.int32))
    x = np.random.default_rng(1).standard_normal((3, 512)).astype(np.float16)
    block.x.upload(x.view(np.uint16))
    try:
        block.step()
        assert block.counts[1].download(np.int32, (4,)).tolist() == [2, 3, 1, 1]
        assert block.lens[1].download(np.int32, (3,)).tolist() == [1, 1, 0]
        assert block.slots.download(np.int32, (3,)).tolist() == [4, 0, -1]
        att = block.att.download(np.uint16, (3, 512)).view(np.float16)
        assert (att[2] == 0).all() and np.abs(att[:2]).max() > 0
    finally:
        block.free_all()


def test_misaligned_cache_is_refused(ctx):
    b = ctx.alloc(4096)
    address = ctypes.c_void_p.from_address(b.handle).value
    off = ctx.wrap(address + 2, 2048)
    small = ctx.alloc(64)
    q, out = ctx.alloc(64 * 2), ctx.alloc(64 * 2)
    a = abi.PagedAttentionArgs(requests=1, heads=1, kv_heads=1, head_dim=64, page_size=1, num_pages=1, max_pages=1, dtype=abi.FLOAT16,
                               scale=1.0, q=q.handle, k_cache=off.handle, v_cache=b.handle, block_table=small.handle, kv_lens=small.handle,
                               out=out.handle)
    assert ctx.s.op_paged_attention(ctx.handle, a) == abi.ERR_INVALID_ARGUMENT
    for x in (off, b, small, q, out):
        x.free()
