"""The chunk attention's workspace: contexts that make no such call go without it, and
the first one may be captured."""
import ctypes
import os

import pytest
import torch

from mlx_amd import abi, runtime
from prompt_util import run_chunk
from serving_util import F16, Device
from test_gpu_paged_chunk import problem

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def hip():
    return ctypes.CDLL("libamdhip64.so", mode=os.RTLD_NOW | os.RTLD_GLOBAL)


def ck(rc):
    assert rc == 0, f"hipError {rc}"


def free_bytes(hip):
    free, total = ctypes.c_size_t(), ctypes.c_size_t()
    ck(hip.hipMemGetInfo(ctypes.byref(free), ctypes.byref(total)))
    return free.value


def test_contexts_without_prompts_are_small(ctx, hip):
    """Products and decoding steps need 32 MB of a context; the parts of cut tiles are 102 MB."""
    args = problem(61, F16, [40], [900], 4, 2, 64, 16)
    run_chunk(ctx, F16, *args, 4, scale=0.125)
    before = free_bytes(hip)
    with runtime.Context(0) as c:
        assert before - free_bytes(hip) < 64 << 20
        run_chunk(c, F16, *args, 4, scale=0.125, requests=0)
        assert before - free_bytes(hip) < 64 << 20
        got = run_chunk(c, F16, *args, 4, scale=0.125)
        held = before - free_bytes(hip)
        run_chunk(c, F16, *args, 4, scale=0.125)
        assert 64 << 20 < held and before - free_bytes(hip) <= held
    want = run_chunk(ctx, F16, *args, 4, scale=0.125)
    assert torch.equal(got[0].view(torch.int16), want[0].view(torch.int16)) and torch.equal(got[1], want[1])


@pytest.mark.parametrize("mode", [0, 1, 2])
def test_first_call_captured(ctx, hip, mode):
    """In each of the runtime's capture modes; replayed with eager calls between."""
    args = problem(62, F16, [40, 1], [2000, 700], 8, 2, 64, 16)
    want = run_chunk(ctx, F16, *args, 8, scale=0.1)
    q, kc, vc, table, starts, seq, lens = args
    with runtime.Context(0) as c, Device(c) as d:
        out, get = d.new(41, 8 * 64, dtype=torch.float16)
        a = abi.PagedChunkArgs(requests=2, tokens=41, heads=8, kv_heads=2, head_dim=64, page_size=16, num_pages=kc.shape[0], max_pages=table.shape[1],
                               dtype=F16, scale=0.1, q=d.up(q), k_cache=d.up(kc), v_cache=d.up(vc), block_table=d.up(table), token_starts=d.up(starts),
                               seq_lens=d.up(seq), kv_lens=d.up(lens), out=out)
        c.sync()
        stream, graph, ready = ctypes.c_void_p(c.stream), ctypes.c_void_p(), ctypes.c_void_p()
        ck(hip.hipStreamBeginCapture(stream, mode))
        try:
            c.paged_chunk_attention(a)
        finally:
            ck(hip.hipStreamEndCapture(stream, ctypes.byref(graph)))
        try:
            ck(hip.hipGraphInstantiate(ctypes.byref(ready), graph, None, None, ctypes.c_size_t(0)))
            for _ in range(3):
                ck(hip.hipGraphLaunch(ready, stream))
                assert torch.equal(get().view(torch.int16), want[0].view(torch.int16))
                again = run_chunk(c, F16, *args, 8, scale=0.1)
                assert torch.equal(again[0].view(torch.int16), want[0].view(torch.int16))
        finally:
            if ready:
                hip.hipGraphExecDestroy(ready)
            hip.hipGraphDestroy(graph)
