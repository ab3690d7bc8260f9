"""Chunk attention of requests that end just below 2^31 tokens: one page, named by
every entry of the row, so that its places count alike.  With a window the same
chunk further in front has the same result (prompt_util.py has the tolerances)."""
import numpy as np
import pytest
import torch

from mlx_amd import abi
from prompt_util import check_chunk, chunk_reference
from serving_util import F16, F32, ROUND, TORCH, Device, randn

pytestmark = pytest.mark.gpu

D = 8


def call(ctx, d, table, columns, dtype, q, kc, vc, H, seq, n, window):
    T, Hk, page = q.shape[0], kc.shape[1], kc.shape[2]
    out, get = d.new(T, H * D, dtype=TORCH[dtype], fill=3.0)
    lse, get_lse = d.new(T, H, dtype=torch.float32, fill=3.0)
    one = lambda *v: d.up(torch.tensor(v, dtype=torch.int32))  # noqa: E731
    ctx.paged_chunk_attention(abi.PagedChunkArgs(
        requests=1, tokens=T, heads=H, kv_heads=Hk, head_dim=D, page_size=page, num_pages=1, max_pages=columns, window=window, dtype=dtype,
        scale=D ** -0.5, q=d.up(q), k_cache=d.up(kc), v_cache=d.up(vc), block_table=table.handle, token_starts=one(0, T), seq_lens=one(seq),
        kv_lens=one(n), out=out, lse=lse))
    return get(), get_lse()


# (page, columns): up to 2^31 - 16 and 2^31 - 8; pages that hold whole runs of tokens and pages that do not
@pytest.mark.parametrize("page,columns", [(16, 2 ** 27 - 1), (12, 178956970)])
def test_windows_just_below_31_bits(ctx, page, columns):
    """The tiles and stages of few rows, of many, and of many heads of keys with few rows each."""
    most = page * columns
    assert 2 ** 31 - 17 < most < 2 ** 31
    table = ctx.upload(np.zeros(columns, np.int32))
    try:
        for dtype in (F32, F16):
            for H, Hk, T in [(1, 1, 1), (4, 2, 5), (1792, 1, 7), (1792, 1792, 7)]:
                gen = torch.Generator().manual_seed(H + T)
                q, kc, vc = randn(gen, dtype, T, H * D), randn(gen, dtype, 1, Hk, page, D), randn(gen, dtype, 1, Hk, page, D)
                for window, short in [(1, 0), (16, 0), (100, 0), (100, 3), (700, 1)]:
                    print(f"[case] page {page}, type {dtype}, heads {H} on {Hk}, {T} tokens, window {window}, {short} short", flush=True)
                    with Device(ctx) as d:
                        got, lse = call(ctx, d, table, columns, dtype, q, kc, vc, H, most - T, most - short, window)
                    shift = most - 60 * page
                    small = torch.zeros(1, 60, dtype=torch.int32)
                    ref = chunk_reference(q, kc, vc, small, torch.tensor([0, T]), torch.tensor([most - T - shift]), torch.tensor([most - short - shift]),
                                          H, window=window, scale=D ** -0.5, dtype=dtype)
                    check_chunk(got, lse, ref, float(vc.abs().max()), dtype, f"{page} {dtype} {H} {Hk} {window} {short}")
    finally:
        table.free()


def test_length_just_below_31_bits(ctx):
    """All 2^31 - 16 tokens.  Each of 256 ranges has four groups of waves, of whose tokens a lane adds every second weight
    one by one: 2^20 roundings of 2^-24 of the sum; the values' sums are 2^17 additions of 16 products."""
    page, columns, H = 16, 2 ** 27 - 1, 2
    table = ctx.upload(np.zeros(columns, np.int32))
    try:
        gen = torch.Generator().manual_seed(1)
        q, kc, vc = randn(gen, F16, 1, H * D), 0.5 * randn(gen, F16, 1, 1, page, D), (0.5 * randn(gen, F16, 1, 1, page, D)).abs() + 1
        print("[case] 2^31 - 16 tokens", flush=True)
        with Device(ctx) as d:
            got, lse = call(ctx, d, table, columns, F16, q, kc, vc, H, page * columns - 1, page * columns, 0)
    finally:
        table.free()
    s = q.double().view(H, D) @ kc[0, 0].double().t() / D ** 0.5
    want = torch.softmax(s, -1) @ vc[0, 0].double()
    bound = 2.0 ** -4 + 2.0 ** -6
    assert ((got.double().view(H, D) - want).abs() <= (bound + ROUND[F16]) * want).all()
    assert ((lse.double()[0] - torch.logsumexp(s, -1) - np.log(float(columns))).abs() <= bound).all()
