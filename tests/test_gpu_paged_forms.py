"""The paged operators' forms that depend on sizes: attention's padded channels
and pages that no run of 16 tokens fits, its loads for large pools, the append's
stores past the caches, and a plan of more tokens than its threads."""
import pytest
import torch

from mlx_amd import abi
from serving_util import BF16, F16, F32, TORCH, Device, attention_reference, check_attention, randn
from test_gpu_paged_attention import check, problem
from test_gpu_paged_cache import append, append_reference, check_plan, same_bits

pytestmark = pytest.mark.gpu

LENS = [0, 1, 15, 17, 33, 64, 130, 257]


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("D", [56, 72, 120, 136, 160, 176, 184, 200, 248])
def test_padded_channels(ctx, dtype, D):
    check(ctx, 500 + D + dtype, dtype, LENS, 6, 2, D, 16)


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("D", [40, 64, 96, 128, 160, 192, 248, 256])
@pytest.mark.parametrize("page", [5, 24])
def test_pages_that_end_inside_a_tile(ctx, dtype, D, page):
    check(ctx, 800 + D + dtype + page, dtype, LENS, 4, 2, D, page)
    check(ctx, 900 + D + dtype + page, dtype, [1500, 3], 2, 1, D, page, window=1003)


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("D", [64, 128, 192, 256])
def test_large_pools(ctx, dtype, D):
    """Pools past 256 MB, of which a few pages are in use: ranges that cut pairs, and short requests."""
    H, Hk, page, lens = 8, 2, 16, [3000, 70, 900, 1, 0]
    q, kc, vc, table, n = problem(1100 + D + dtype, dtype, lens, H, Hk, D, page, spare=0, poison=False)
    size = TORCH[dtype].itemsize
    pages = (256 << 20) // (2 * D * size * page * Hk) + 3
    assert pages > kc.shape[0]
    gen = torch.Generator().manual_seed(D)
    place = torch.randperm(pages, generator=gen)[:kc.shape[0]].to(torch.int32)  # of the small pool's pages in the large one
    print(f"[case] dtype={dtype} D={D} pages={pages}", flush=True)
    kb, vb = (ctx.alloc(pages * Hk * page * D * size) for _ in range(2))
    try:
        with Device(ctx) as dev:
            slots = (place[:, None] * page + torch.arange(page, dtype=torch.int32)).reshape(-1)
            rows = [c.transpose(1, 2).reshape(-1, Hk * D) for c in (kc, vc)]
            ctx.paged_append(abi.PagedAppendArgs(
                tokens=len(slots), kv_heads=Hk, head_dim=D, page_size=page, num_pages=pages, in_dtype=dtype, cache_dtype=dtype,
                k=dev.up(rows[0]), v=dev.up(rows[1]), slots=dev.up(slots), k_cache=kb.handle, v_cache=vb.handle))
            far = torch.where(table >= 0, place[table.clamp(min=0).long()], -1)
            out_h, out_get = dev.new(len(lens), H * D, dtype=TORCH[dtype])
            lse_h, lse_get = dev.new(len(lens), H, dtype=torch.float32)
            ctx.paged_attention(abi.PagedAttentionArgs(
                requests=len(lens), heads=H, kv_heads=Hk, head_dim=D, page_size=page, num_pages=pages, max_pages=table.shape[1], dtype=dtype,
                scale=D ** -0.5, q=dev.up(q), k_cache=kb.handle, v_cache=vb.handle, block_table=dev.up(far), kv_lens=dev.up(n), out=out_h,
                lse=lse_h))
            got, lse = out_get(), lse_get()
    finally:
        kb.free()
        vb.free()
    ref = attention_reference(q, kc, vc, table, n, H, scale=D ** -0.5)
    check_attention(got, lse, ref, float(vc.double().abs().max()), dtype, "large pool")


@pytest.mark.parametrize("in_dt,cache_dt", [(F32, F16), (F32, BF16), (F16, F16), (BF16, BF16), (F16, BF16)])
def test_append_past_the_caches(ctx, in_dt, cache_dt):
    """32 MB of 16-bit results and more."""
    Hk, D, page, T = 8, 128, 16, 8200
    gen = torch.Generator().manual_seed(in_dt + 3 * cache_dt)
    pages = -(-T // page) + 3
    slots = torch.randperm(pages * page, generator=gen)[:T].to(torch.int32)
    slots[::7] = -1
    k, v = randn(gen, in_dt, T, Hk * D), randn(gen, in_dt, T, Hk * D)
    kc, vc = randn(gen, cache_dt, pages, Hk, page, D), randn(gen, cache_dt, pages, Hk, page, D)
    gk, gv = append(ctx, k, v, slots, kc, vc, in_dt, cache_dt)
    assert same_bits(gk, append_reference(k, slots, kc)) and same_bits(gv, append_reference(v, slots, vc))


def test_plan_of_many_tokens(ctx):
    """More tokens than 1024 blocks of 256 threads, with entries for all of them and for some."""
    check_plan(ctx, [5, 0, 100], [200000, 1, 150003], 64, 6000, seed=1)
    check_plan(ctx, [5, 0, 100], [200000, 1, 150003], 64, 6000, max_tokens=270001, spare=-100, seed=2)
    check_plan(ctx, [3] * 2500, [130] * 2500, 16, 20, seed=3)


@pytest.mark.parametrize("R", [2047, 2048, 2049, 4095, 4096, 4097])
def test_plan_of_very_many_requests(ctx, R):
    """On both sides of what one launch takes, each thread's stretch of requests ragged at its end."""
    gen = torch.Generator().manual_seed(R)
    seq, new = torch.randint(0, 60, (R,), generator=gen).tolist(), torch.randint(0, 2, (R,), generator=gen).tolist()
    new[-1], new[R // 3] = 70, 300
    check_plan(ctx, seq, new, 16, 24, spare=-2, head=5, seed=R)
    new[0] = 300000
    check_plan(ctx, seq, new, 16, 24, max_tokens=280000, seed=R)
