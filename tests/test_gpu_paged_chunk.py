"""Chunk attention over a paged cache against its definition in 64 bits
(prompt_util.py has the tolerances)."""
import math

import pytest
import torch

from mlx_amd import abi
from prompt_util import check_chunk, chunk_reference, run_chunk, starts_of, table_of
from serving_util import BF16, F16, F32, TORCH, randn

pytestmark = pytest.mark.gpu


def problem(seed, dtype, new, held, H, Hk, D, page, cols=None, short=None, rows=0):
    """q, caches, table, starts, seq, lens; short: how many of a request's last tokens have no page; rows: behind the last one"""
    gen = torch.Generator().manual_seed(seed)
    lens = [n + h - ((short or {}).get(r, 0)) for r, (n, h) in enumerate(zip(new, held))]
    table, pool = table_of(gen, lens, page, cols)
    q = randn(gen, dtype, sum(new) + rows, H * D)
    kc, vc = randn(gen, dtype, pool, Hk, page, D), randn(gen, dtype, pool, Hk, page, D)
    i = lambda v: torch.tensor(v, dtype=torch.int32)  # noqa: E731
    return q, kc, vc, table, starts_of(new), i(held), i(lens)


def check(ctx, dtype, args, H, what, **kw):
    D = args[1].shape[-1]
    kw.setdefault("scale", D ** -0.5)
    out, lse = run_chunk(ctx, dtype, *args, H, **kw)
    ref = chunk_reference(*args, H, dtype=dtype, **{k: v for k, v in kw.items() if k in ("window", "scale", "softcap")})
    v = args[2].double()
    check_chunk(out, lse, ref, float(v[torch.isfinite(v)].abs().max()), dtype, what, filled=3.0)


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("H,Hk,D,page", [(8, 2, 64, 16), (4, 4, 128, 16), (10, 2, 80, 24), (8, 1, 256, 32), (6, 2, 192, 8), (3, 3, 8, 4),
                                         (7, 1, 136, 5), (40, 1, 64, 16), (300, 1, 16, 16), (5, 5, 128, 1), (32, 2, 96, 7)])
def test_ragged_batch(ctx, dtype, H, Hk, D, page):
    """Chunks and single tokens, with and without tokens held before, an empty request among them."""
    new, held = [5, 1, 0, 70, 1, 33], [0, 0, 9, 130, 77, 1]
    check(ctx, dtype, problem(H * D, dtype, new, held, H, Hk, D, page, rows=3), H, f"{H} {Hk} {D} {page}")


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("new,held", [([1], [0]), ([1], [1]), ([64], [0]), ([65], [63]), ([2], [2000]), ([700], [0]), ([1] * 70, [3] * 70),
                                      ([0, 0, 1, 0], [5, 0, 300, 2]), ([257, 31], [64, 1500])])
@pytest.mark.parametrize("D", [64, 128, 256])
def test_lengths(ctx, dtype, new, held, D):
    """From one token to several tiles, and few rows whose cached tokens are cut into many parts."""
    check(ctx, dtype, problem(len(new), dtype, new, held, 4, 2, D, 16), 4, f"{new} {held}")


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("window", [1, 7, 16, 100, 100000])
def test_window(ctx, dtype, window):
    check(ctx, dtype, problem(window, dtype, [40, 1, 200], [0, 500, 90], 4, 2, 64, 16), 4, f"window {window}", window=window)


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("scale,softcap", [(0.125, 30.0), (1.0, 0.5), (-0.2, 0.0), (0.0, 0.0), (-0.3, 5.0), (2.0, 0.0)])
def test_scale_and_cap(ctx, dtype, scale, softcap):
    check(ctx, dtype, problem(3, dtype, [30, 2], [100, 7], 4, 1, 64, 16), 4, f"{scale} {softcap}", scale=scale, softcap=softcap)


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
def test_pages_that_are_none(ctx, dtype):
    """Holes of -1, of ids past the pool and below it, inside and at the ends, and a request without any page."""
    args = problem(5, dtype, [50, 20, 9], [100, 40, 30], 4, 2, 128, 16)
    table = args[3]
    table[0, 2], table[0, 5], table[0, 9] = -1, args[1].shape[0], -5
    table[1, 0] = 1 << 30
    table[2, :] = -1
    check(ctx, dtype, args, 4, "holes")
    check(ctx, dtype, args, 4, "holes and window", window=20)


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_tokens_past_the_cache(ctx, dtype):
    """Pages ran out: new tokens whose positions are at or past kv_lens see what there is."""
    check(ctx, dtype, problem(6, dtype, [20, 5, 3], [30, 0, 16], 2, 1, 64, 16, cols=4, short={0: 4, 1: 5, 2: 3}), 2, "short")
    check(ctx, dtype, problem(6, dtype, [20, 5, 3], [30, 0, 16], 2, 1, 64, 16, cols=4, short={0: 4, 1: 5, 2: 3}), 2, "short", window=3)


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
def test_lengths_outside_the_table(ctx, dtype):
    """seq_lens and kv_lens below 0 and above the table's capacity."""
    q, kc, vc, table, starts, seq, lens = problem(7, dtype, [4, 4, 4], [20, 20, 20], 2, 2, 64, 8)
    seq[0], lens[1], lens[2] = -3, -9, 1 << 30
    seq[2] = table.shape[1] * 8 - 2
    check(ctx, dtype, (q, kc, vc, table, starts, seq, lens), 2, "outside")


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("D", [64, 128])
def test_values_that_do_not_count(ctx, dtype, D):
    """NaN and infinities in every place that no row sees, and in pages of nobody."""
    new, held, page = [30, 1, 5], [70, 33, 0], 16
    args = problem(8, dtype, new, held, 4, 2, D, page)
    q, kc, vc, table = args[:4]
    seen = torch.zeros(kc.shape[0], page, dtype=torch.bool)
    for r, n in enumerate(a + b for a, b in zip(new, held)):
        t = torch.arange(n)
        seen[table[r].long()[t // page], t % page] = True
    bad = torch.tensor([math.nan, math.inf, -math.inf])
    for c in (kc, vc):
        at = (~seen)[:, None, :, None].expand(c.shape)
        c[at] = bad[torch.arange(int(at.sum())) % 3].to(c.dtype)
    check(ctx, dtype, args, 4, "garbage")


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("held", [0, 40, 2000])
def test_infinite_values(ctx, dtype, held):
    """An infinite value counts for the rows that see it, and for no other: those before it in the chunk."""
    args = problem(9, dtype, [90, 3], [held, 10], 4, 2, 64, 16)
    vc, table = args[2], args[3]

    def place(t, r=0):
        return int(table[r, t // 16]), t % 16
    for t, h, d, x in [(held + 20, 0, 3, math.inf), (held + 41, 1, 60, -math.inf), (held + 50, 1, 60, math.inf), (held + 70, 0, 9, math.nan)]:
        pg, at = place(t)
        vc[pg, h, at, d] = x
    check(ctx, dtype, args, 4, "infinite")


@pytest.mark.parametrize("dtype", [F16, BF16])
def test_keys_that_are_not_finite(ctx, dtype):
    """A key of NaN makes the rows that see it NaN, and no other."""
    q, kc, vc, table, starts, seq, lens = args = problem(10, dtype, [40], [24], 2, 1, 64, 8)
    kc[int(table[0, 50 // 8]), 0, 50 % 8, 7] = math.nan
    out, lse = run_chunk(ctx, dtype, *args, 2, scale=0.125)
    rows = torch.arange(40) + 24 >= 50
    assert torch.isnan(out.float()[rows]).all() and torch.isnan(lse[rows]).all()
    kc[int(table[0, 50 // 8]), 0, 50 % 8, 7] = 0.5
    ref = chunk_reference(q, kc, vc, table, starts, seq, lens, 2, scale=0.125, dtype=dtype)
    cut = tuple(x[~rows] for x in ref)
    check_chunk(out[~rows], lse[~rows], cut, float(vc.abs().max()), dtype, "before it")


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
def test_large_scores_and_small_weights(ctx, dtype):
    """Scores that fall or rise over the cache, and thousands of small weights beside a large one."""
    q, kc, vc, table, starts, seq, lens = args = problem(11, dtype, [3], [3000], 1, 1, 64, 16)
    q.fill_(0)
    q[:, 0] = 1.0
    kc.fill_(0)
    flat = torch.empty(3008)
    for what, line in [("rise", torch.arange(3003) / 100.0), ("fall", -torch.arange(3003) / 100.0),
                       ("one", torch.where(torch.arange(3003) == 1234, 0.0, -16.0)), ("late", torch.where(torch.arange(3003) == 2990, 60.0, 0.0))]:
        flat[:3003] = line
        kc[table[0].long(), 0, :, 0] = flat.view(-1, 16).to(TORCH[dtype])
        check(ctx, dtype, args, 1, what, scale=1.0)


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("q_off,q_pad,o_off,o_pad", [(0, 5, 0, 3), (7, 0, 1, 0), (3, 9, 5, 1)])
def test_strides_and_offsets(ctx, dtype, q_off, q_pad, o_off, o_pad):
    H, D = 4, 64
    q, kc, vc, table, starts, seq, lens = problem(12, dtype, [20, 3], [50, 0], H, 2, D, 16)
    T, row = q.shape
    wide = torch.full((T * (row + q_pad) + q_off,), math.nan, dtype=q.dtype)
    wide[q_off:].view(T, row + q_pad)[:, :row] = q
    from serving_util import Device
    with Device(ctx) as d:
        n = T * (row + o_pad) + o_off
        out, get = d.new(n, dtype=q.dtype, fill=3.0)
        a = abi.PagedChunkArgs(
            requests=2, tokens=T, heads=H, kv_heads=2, head_dim=D, page_size=16, num_pages=kc.shape[0], max_pages=table.shape[1], dtype=dtype,
            scale=0.125, q_offset=q_off, q_row_stride=row + q_pad, out_offset=o_off, out_row_stride=row + o_pad, q=d.up(wide), k_cache=d.up(kc),
            v_cache=d.up(vc), block_table=d.up(table), token_starts=d.up(starts), seq_lens=d.up(seq), kv_lens=d.up(lens), out=out)
        ctx.paged_chunk_attention(a)
        got = get()
    ref = chunk_reference(q, kc, vc, table, starts, seq, lens, H, scale=0.125, dtype=dtype)
    body = got[o_off:].view(T, row + o_pad)
    check_chunk(body[:, :row].contiguous(), None, ref, float(vc.abs().max()), dtype, "strides")
    assert (got[:o_off] == 3).all() and (body[:, row:] == 3).all()


def test_rows_in_front_and_behind(ctx):
    """token_starts that begin past row 0 and end before the last row, and past the last row."""
    q, kc, vc, table, starts, seq, lens = problem(13, F16, [20, 30], [10, 0], 4, 2, 64, 16, rows=9)
    check(ctx, F16, (q, kc, vc, table, starts + 4, seq, lens), 4, "in front")
    out, _ = run_chunk(ctx, F16, q[:45], kc, vc, table, starts, seq, lens, 4, scale=0.125)
    ref = chunk_reference(q[:45], kc, vc, table, starts, seq, lens, 4, scale=0.125, dtype=F16)
    check_chunk(out, None, ref, float(vc.abs().max()), F16, "cut short")


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
def test_many_requests(ctx, dtype):
    gen = torch.Generator().manual_seed(14)
    new = torch.randint(0, 4, (1500,), generator=gen).tolist()
    held = torch.randint(0, 30, (1500,), generator=gen).tolist()
    check(ctx, dtype, problem(14, dtype, new, held, 2, 1, 64, 8), 2, "many")
    check(ctx, dtype, problem(14, dtype, [0] * 900 + [5] + [0] * 900 + [7], [3] * 1802, 2, 1, 64, 8), 2, "empty ones")


def test_same_result_each_time(ctx):
    args = problem(15, BF16, [100, 1, 3], [900, 2000, 0], 8, 2, 128, 16)
    first = run_chunk(ctx, BF16, *args, 8, scale=0.1)
    for _ in range(5):
        again = run_chunk(ctx, BF16, *args, 8, scale=0.1)
        assert torch.equal(first[0].view(torch.int16), again[0].view(torch.int16)) and torch.equal(first[1], again[1])


REFUSED = [
    (abi.ERR_INVALID_ARGUMENT, dict(struct_size=1)), (abi.ERR_INVALID_ARGUMENT, dict(requests=-1)), (abi.ERR_INVALID_ARGUMENT, dict(tokens=-1)),
    (abi.ERR_INVALID_ARGUMENT, dict(heads=3)), (abi.ERR_INVALID_ARGUMENT, dict(heads=0)), (abi.ERR_INVALID_ARGUMENT, dict(page_size=0)),
    (abi.ERR_INVALID_ARGUMENT, dict(max_pages=0)), (abi.ERR_INVALID_ARGUMENT, dict(window=-1)), (abi.ERR_INVALID_ARGUMENT, dict(softcap=-1.0)),
    (abi.ERR_INVALID_ARGUMENT, dict(softcap=1e-35)), (abi.ERR_INVALID_ARGUMENT, dict(softcap=math.nan)), (abi.ERR_INVALID_ARGUMENT, dict(q=None)),
    (abi.ERR_INVALID_ARGUMENT, dict(out=None)), (abi.ERR_INVALID_ARGUMENT, dict(token_starts=None)), (abi.ERR_INVALID_ARGUMENT, dict(seq_lens=None)),
    (abi.ERR_INVALID_ARGUMENT, dict(tokens=8)), (abi.ERR_INVALID_ARGUMENT, dict(requests=3)), (abi.ERR_INVALID_ARGUMENT, dict(num_pages=100)),
    (abi.ERR_INVALID_ARGUMENT, dict(q_row_stride=100)), (abi.ERR_INVALID_ARGUMENT, dict(q_offset=1)), (abi.ERR_INVALID_ARGUMENT, dict(out_offset=-1)),
    (abi.ERR_NOT_SUPPORTED, dict(dtype=3)), (abi.ERR_NOT_SUPPORTED, dict(head_dim=60)), (abi.ERR_NOT_SUPPORTED, dict(head_dim=264)),
    (abi.ERR_NOT_SUPPORTED, dict(max_pages=1 << 27)), (abi.ERR_NOT_SUPPORTED, dict(num_pages=1 << 27)),
]


@pytest.mark.parametrize("code,over", REFUSED)
def test_refusals(ctx, code, over):
    args = problem(16, F16, [4, 2], [3, 0], 4, 2, 64, 16)
    run_chunk(ctx, F16, *args, 4, expect=code, **over)


def test_overlaps_are_refused(ctx):
    args = problem(17, F16, [4, 2], [3, 0], 4, 2, 64, 16)
    q, kc, vc, table, starts, seq, lens = args
    from serving_util import Device
    with Device(ctx) as d:
        b = d.up(q)
        run_chunk(ctx, F16, *args, 4, expect=abi.ERR_INVALID_ARGUMENT, q=b, out=b)


def test_nothing_to_do(ctx):
    q, kc, vc, table, starts, seq, lens = problem(18, F16, [4, 2], [3, 0], 4, 2, 64, 16)
    out, lse = run_chunk(ctx, F16, q, kc, vc, table, torch.zeros(3, dtype=torch.int32), seq, lens, 4)
    assert (out == 3).all() and (lse == 3).all()
    out, _ = run_chunk(ctx, F16, q, kc, vc, table, starts, seq, lens, 4, requests=0)
    assert (out == 3).all()
    out, lse = run_chunk(ctx, F16, q, kc, vc, table, starts, seq, lens, 4, num_pages=0)
    assert (out == 0).all() and torch.isneginf(lse).all()
