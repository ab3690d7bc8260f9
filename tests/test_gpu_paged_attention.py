"""Paged attention of one token per request against its definition in 64 bits:
types, head layouts, lengths around tiles and pages, page sizes that end inside
tiles, windows, softcap, strided rows, empty requests, pages that are none, and
cache places that hold NaN and infinities."""
import numpy as np
import pytest
import torch

from mlx_amd import abi
from serving_util import BF16, F16, F32, TORCH, Device, attention_reference, check_attention, randn

pytestmark = pytest.mark.gpu


def attend(ctx, q, kc, vc, table, lens, H, dtype, window=0, scale=None, softcap=0.0, lse=True, q_offset=0, q_stride=None,
           out_offset=0, out_stride=None):
    """q: [R, q_stride] storage; out comes back as [R, H * D]."""
    R, cols = table.shape
    pages, Hk, page, D = kc.shape
    out_stride = out_stride or H * D
    with Device(ctx) as dev:
        store = torch.full((out_offset + max(R, 1) * out_stride,), 7.0, dtype=TORCH[dtype])
        out_h, out_get = dev.out(store)
        lse_h, lse_get = dev.new(R, H, dtype=torch.float32) if lse else (None, None)
        args = abi.PagedAttentionArgs(
            requests=R, heads=H, kv_heads=Hk, head_dim=D, page_size=page, num_pages=pages, max_pages=cols, window=window,
            scale=D ** -0.5 if scale is None else scale, softcap=softcap, dtype=dtype, q_offset=q_offset,
            q_row_stride=q_stride or H * D, out_offset=out_offset, out_row_stride=out_stride, q=dev.up(q), k_cache=dev.up(kc),
            v_cache=dev.up(vc), block_table=dev.up(table), kv_lens=dev.up(lens), out=out_h, lse=lse_h)
        ctx.paged_attention(args)
        got = out_get()
        # places between the rows stay
        mask = torch.ones_like(store, dtype=torch.bool)
        rows = torch.as_strided(got, (R, H * D), (out_stride, 1), out_offset).clone()
        if R:
            torch.as_strided(mask, (R, H * D), (out_stride, 1), out_offset).fill_(False)
        assert (got[mask] == 7.0).all()
        return rows, lse_get() if lse else None


def problem(seed, dtype, lens, H, Hk, D, page, spare=3, poison=True):
    """Pages in any order; places that no position names hold NaN and infinities."""
    gen = torch.Generator().manual_seed(seed)
    R, cols = len(lens), max(1, -(-max(list(lens) + [1]) // page)) + 1
    pages = sum(-(-n // page) for n in lens if n > 0) + spare
    order = torch.randperm(pages, generator=gen).to(torch.int32)
    table = torch.full((R, cols), -1, dtype=torch.int32)
    at = 0
    for r, n in enumerate(lens):
        c = max(0, -(-n // page))
        table[r, :c] = order[at:at + c]
        at += c
    kc, vc = randn(gen, dtype, pages, Hk, page, D), randn(gen, dtype, pages, Hk, page, D)
    if poison:
        used = torch.zeros(pages, page, dtype=torch.bool)
        for r, n in enumerate(lens):
            for t in range(max(n, 0)):
                used[table[r, t // page], t % page] = True
        junk = torch.tensor([float("nan"), float("inf"), -float("inf")])
        for c in (kc, vc):
            bad = junk[torch.randint(0, 3, c.shape, generator=gen)].to(c.dtype)
            c[:] = torch.where(used[:, None, :, None], c, bad)
    q = randn(gen, dtype, R, H * D)
    return q, kc, vc, table, torch.tensor(list(lens), dtype=torch.int32)


def check(ctx, seed, dtype, lens, H, Hk, D, page, window=0, softcap=0.0, scale=None, poison=True):
    print(f"[case] seed={seed} dtype={dtype} lens={list(lens)[:12]} H={H} Hk={Hk} D={D} page={page} window={window} softcap={softcap}", flush=True)
    q, kc, vc, table, n = problem(seed, dtype, lens, H, Hk, D, page, poison=poison)
    got, lse = attend(ctx, q, kc, vc, table, n, H, dtype, window, scale, softcap)
    ref = attention_reference(q, kc, vc, table, n, H, window, D ** -0.5 if scale is None else scale, softcap)
    v_max = float(torch.nan_to_num(vc.double(), 0, 0, 0).abs().max())
    check_attention(got, lse, ref, v_max, dtype, f"seed {seed}")


LENS = [0, 1, 2, 15, 16, 17, 31, 32, 33, 63, 64, 65, 127, 128, 129, 257, 400]


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("H,Hk,D", [(4, 4, 64), (8, 2, 128), (16, 1, 256), (6, 2, 80), (3, 3, 8), (10, 2, 192)])
def test_lengths_around_tiles_and_pages(ctx, dtype, H, Hk, D):
    check(ctx, 1 + D + dtype, dtype, LENS, H, Hk, D, 16)


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("page", [1, 3, 8, 24, 32, 100, 128])
def test_page_sizes(ctx, dtype, page):
    check(ctx, 50 + page + dtype, dtype, [1, page - 1, page, page + 1, 3 * page, 211], 8, 2, 64, page)


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("H,Hk", [(1, 1), (5, 1), (17, 1), (40, 2), (33, 1), (24, 8), (64, 1)])
def test_query_groups(ctx, dtype, H, Hk):
    check(ctx, 100 + H + dtype, dtype, [1, 30, 300, 0, 129], H, Hk, 128, 16)


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("window", [1, 2, 31, 32, 100, 1000])
def test_windows(ctx, dtype, window):
    check(ctx, 150 + window + dtype, dtype, [0, 1, 32, 33, 100, 101, 385, 500], 8, 4, 64, 24, window=window)


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
def test_softcap_and_scales(ctx, dtype):
    check(ctx, 200 + dtype, dtype, [1, 50, 333], 8, 2, 128, 16, softcap=2.0)
    check(ctx, 203 + dtype, dtype, [1, 50, 333], 8, 2, 128, 16, softcap=30.0, scale=1.0)
    check(ctx, 206 + dtype, dtype, [1, 50, 333], 8, 2, 128, 16, scale=-0.3)
    check(ctx, 209 + dtype, dtype, [1, 50, 333], 8, 2, 128, 16, scale=0.0)


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
def test_long_and_ragged(ctx, dtype):
    """Ranges that cut pairs: long beside short, and one request alone over many ranges."""
    check(ctx, 250 + dtype, dtype, [5000, 1, 0, 2900, 130], 8, 2, 64, 16, poison=False)
    check(ctx, 253 + dtype, dtype, [9000], 4, 1, 128, 32, poison=False)
    check(ctx, 256 + dtype, dtype, [1500, 3, 700], 4, 2, 256, 16, poison=False)


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
def test_pairs_of_very_many_parts(ctx, dtype):
    """Wide partial results of one pair over most of the card's ranges, alone and beside short requests."""
    check(ctx, 260 + dtype, dtype, [9000], 16, 1, 256, 32, poison=False)
    check(ctx, 263 + dtype, dtype, [5, 0, 20000, 17, 1, 300] + [40] * 20, 12, 1, 256, 16, poison=False)
    check(ctx, 266 + dtype, dtype, [30000, 2], 16, 2, 128, 64, poison=False)


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
def test_many_short_requests(ctx, dtype):
    gen = torch.Generator().manual_seed(9)
    check(ctx, 270 + dtype, dtype, torch.randint(0, 90, (700,), generator=gen).tolist(), 2, 1, 64, 16)


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
def test_pages_that_are_none(ctx, dtype):
    """-1, and numbers past the pool, in the middle of a request and for all of one."""
    q, kc, vc, table, n = problem(300 + dtype, dtype, [200, 64, 300], 8, 2, 64, 16, poison=False)
    table[0, 3], table[0, 12], table[1, :4] = -1, kc.shape[0], torch.tensor([-1, 2 ** 30, -5, 2 ** 31 - 1], dtype=torch.int32)
    got, lse = attend(ctx, q, kc, vc, table, n, 8, dtype)
    check_attention(got, lse, attention_reference(q, kc, vc, table, n, 8, scale=0.125), float(vc.double().abs().max()), dtype, "none pages")
    assert (got[1] == 0).all() and torch.isneginf(lse[1]).all()


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
def test_lengths_past_the_table_and_below_zero(ctx, dtype):
    q, kc, vc, table, n = problem(320 + dtype, dtype, [64, 48, 20], 4, 4, 64, 16, poison=False)
    table = table[:, :3].contiguous()
    n = torch.tensor([10 ** 9, -4, 20], dtype=torch.int32)
    got, lse = attend(ctx, q, kc, vc, table, n, 4, dtype)
    check_attention(got, lse, attention_reference(q, kc, vc, table, n, 4, scale=0.125), float(vc.double().abs().max()), dtype, "lengths")


def test_empty_pool_and_no_requests(ctx):
    q, lens = torch.ones(2, 4 * 64), torch.tensor([5, 0], dtype=torch.int32)
    empty = torch.zeros(0, 2, 16, 64)
    got, lse = attend(ctx, q, empty, empty, torch.zeros(2, 3, dtype=torch.int32), lens, 4, F32)
    assert (got == 0).all() and torch.isneginf(lse).all()
    got, _ = attend(ctx, torch.ones(0, 4 * 64), torch.ones(1, 2, 16, 64), torch.ones(1, 2, 16, 64), torch.zeros(0, 3, dtype=torch.int32),
                    torch.zeros(0, dtype=torch.int32), 4, F32)
    assert got.numel() == 0


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("q_offset,q_stride,out_offset,out_stride", [(0, 8 * 64 + 2 * 4 * 64, 0, 0), (3, 8 * 64 + 5, 1, 8 * 64 + 7)])
def test_strided_rows(ctx, dtype, q_offset, q_stride, out_offset, out_stride):
    """q out of a fused projection, and rows at odd places."""
    lens = [70, 1, 300]
    q, kc, vc, table, n = problem(340 + dtype, dtype, lens, 8, 4, 64, 16)
    store = torch.full((q_offset + len(lens) * q_stride,), float("nan"), dtype=TORCH[dtype])
    torch.as_strided(store, (len(lens), 8 * 64), (q_stride, 1), q_offset).copy_(q)
    got, lse = attend(ctx, store, kc, vc, table, n, 8, dtype, q_offset=q_offset, q_stride=q_stride, out_offset=out_offset,
                      out_stride=out_stride, lse=False)
    v_max = float(torch.nan_to_num(vc.double(), 0, 0, 0).abs().max())
    check_attention(got, None, attention_reference(q, kc, vc, table, n, 8, scale=0.125), v_max, dtype, "strided")


def test_infinite_and_nan_scores_that_count(ctx):
    """A key of -infinity direction takes weight 0; NaN in a counted place makes its heads NaN and no other."""
    q, kc, vc, table, n = problem(360, F32, [50, 50], 4, 2, 64, 16, poison=False)
    kc[table[0, 1], 0, 3] = -float("inf") * torch.sign(q[0, :64])  # head 0's score there: -infinity
    kc[table[1, 2], 1, 5, 0] = float("nan")
    got, _ = attend(ctx, q, kc, vc, table, n, 4, F32)
    got = got.view(2, 4, 64)
    assert torch.isfinite(got[0, 0]).all() and torch.isfinite(got[1, :2]).all()
    assert torch.isnan(got[1, 2:]).all()
    one = torch.cat([torch.arange(19), torch.arange(20, 50)])
    k, v = (c[table[0, one // 16].long(), 0, one % 16].double() for c in (kc, vc))
    p = torch.softmax(k @ q[0, :64].double() / 8, 0)
    assert (got[0, 0].double() - p @ v).abs().max() < 1e-5


def test_cache_past_32_bits(ctx):
    """Rows beyond 4 GiB of a cache: pages at its end."""
    Hk, page, D, pages = 8, 64, 256, 17000
    bytes_ = pages * Hk * page * D * 2
    assert bytes_ > 2 ** 32
    kb, vb = ctx.alloc(bytes_), ctx.alloc(bytes_)
    try:
        gen = torch.Generator().manual_seed(4)
        table = torch.tensor([[pages - 1, pages - 2, 5]], dtype=torch.int32)
        part = randn(gen, F16, 3, 2, Hk, page, D)  # the three pages' keys and values
        with Device(ctx) as dev:
            # the pages are written by the append operator
            slots = (table[0, :, None] * page + torch.arange(page, dtype=torch.int32)).reshape(-1)
            rows = part.transpose(2, 3).reshape(3, 2, page, Hk * D)
            ctx.paged_append(abi.PagedAppendArgs(
                tokens=3 * page, kv_heads=Hk, head_dim=D, page_size=page, num_pages=pages, in_dtype=F16, cache_dtype=F16,
                k=dev.up(rows[:, 0].reshape(-1, Hk * D)), v=dev.up(rows[:, 1].reshape(-1, Hk * D)), slots=dev.up(slots),
                k_cache=kb.handle, v_cache=vb.handle))
            q, lens = randn(gen, F16, 1, 16 * D), torch.tensor([3 * page], dtype=torch.int32)
            out_h, out_get = dev.new(1, 16 * D, dtype=torch.float16)
            ctx.paged_attention(abi.PagedAttentionArgs(
                requests=1, heads=16, kv_heads=Hk, head_dim=D, page_size=page, num_pages=pages, max_pages=3, dtype=F16, scale=D ** -0.5,
                q=dev.up(q), k_cache=kb.handle, v_cache=vb.handle, block_table=dev.up(table), kv_lens=dev.up(lens), out=out_h))
            got = out_get()
        small = torch.arange(3, dtype=torch.int32)[None]
        ref = attention_reference(q, part[:, 0].contiguous(), part[:, 1].contiguous(), small, lens, 16, scale=D ** -0.5)
        check_attention(got, None, ref, float(part.double().abs().max()), F16, "past 32 bits")
    finally:
        kb.free()
        vb.free()


def test_repeats_are_the_same_and_leave_the_gemm_workspace(ctx, oracle):
    """The same bits on every launch, and a split-K product before, between and after."""
    from mlx_amd import runtime
    x, w, s, b, _ = oracle.make_problem(64, 3584, 4096, 3, 64, F16, F16, seed=3)
    q, kc, vc, table, n = problem(400, BF16, [3000, 70, 900, 1], 8, 2, 128, 16, poison=False)
    ys, outs = [], []
    for _ in range(3):
        ys.append(runtime.run_quantized_matmul(ctx, x, w, s, b, 64, 3584, 4096, 64, 3, F16, F16, F16))
        outs.append(attend(ctx, q, kc, vc, table, n, 8, BF16))
    ys.append(runtime.run_quantized_matmul(ctx, x, w, s, b, 64, 3584, 4096, 64, 3, F16, F16, F16))
    assert all(np.array_equal(y, ys[0]) for y in ys)
    assert all(torch.equal(o[0].view(torch.int16), outs[0][0].view(torch.int16)) and torch.equal(o[1], outs[0][1]) for o in outs)


def _record(dev, **over):
    r = dict(requests=2, heads=4, kv_heads=2, head_dim=64, page_size=16, num_pages=8, max_pages=4, dtype=F16, scale=0.125)
    bufs = dict(q=torch.zeros(2, 256), k_cache=torch.zeros(8, 2, 16, 64), v_cache=torch.zeros(8, 2, 16, 64), out=torch.zeros(2, 256))
    r.update({k: dev.up(v.to(torch.float16)) for k, v in bufs.items()})
    r.update(block_table=dev.up(torch.zeros(2, 4, dtype=torch.int32)), kv_lens=dev.up(torch.zeros(2, dtype=torch.int32)))
    r.update(over)
    return abi.PagedAttentionArgs(**r)


def test_refusals(ctx):
    I, N = abi.ERR_INVALID_ARGUMENT, abi.ERR_NOT_SUPPORTED
    with Device(ctx) as dev:
        call = lambda a: ctx.s.op_paged_attention(ctx.handle, a)  # noqa: E731
        assert call(_record(dev)) == abi.OK
        for over, want in [(dict(requests=-1), I), (dict(requests=3), I), (dict(heads=5), I), (dict(heads=0), I), (dict(kv_heads=0), I),
                           (dict(head_dim=0), I), (dict(head_dim=60), N), (dict(head_dim=264), N), (dict(page_size=0), I),
                           (dict(num_pages=-1), I), (dict(num_pages=9), I), (dict(max_pages=0), I), (dict(max_pages=5), I),
                           (dict(window=-1), I), (dict(softcap=-1.0), I), (dict(softcap=float("nan")), I), (dict(dtype=3), N),
                           (dict(dtype=F32), I), (dict(q_row_stride=255), I), (dict(q_row_stride=257), I), (dict(q_offset=1), I),
                           (dict(q_offset=-1), I), (dict(out_row_stride=1), I), (dict(q=None), I), (dict(k_cache=None), I),
                           (dict(block_table=None), I), (dict(kv_lens=None), I), (dict(out=None), I),
                           (dict(max_pages=2 ** 30, page_size=4), N)]:
            assert call(_record(dev, **over)) == want, over
        for pair in [("out", "q"), ("out", "k_cache"), ("lse", "kv_lens")]:
            a = _record(dev)
            setattr(a, pair[0], getattr(a, pair[1]))
            assert call(a) == I, pair
        a = _record(dev)
        a.struct_size = 8
        assert call(a) == I
        assert ctx.s.op_paged_attention(None, _record(dev)) == I and ctx.s.op_paged_attention(ctx.handle, None) == I
