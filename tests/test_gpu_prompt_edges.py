"""Calls of the prompt operators that their documentation allows at the edges, and
arguments that they refuse or survive."""
import math

import pytest
import torch

from mlx_amd import abi
from prompt_util import ints, run_chunk
from serving_util import BF16, F16, F32, Device
from test_gpu_paged_chunk import check, problem

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("front", [1, 63, 64, 65, 300, 1000])
@pytest.mark.parametrize("new,held,H", [([20, 1, 30], [10, 300, 0], 4), ([0, 0, 40, 0, 7], [5, 0, 9, 3, 0], 4), ([200, 90], [30, 100], 64)])
def test_rows_far_in_front(ctx, front, new, held, H):
    """token_starts that begin tiles past row 0: the rows before stay as they were."""
    q, kc, vc, table, starts, seq, lens = problem(front, F16, new, held, H, 2, 64, 16, rows=front + 5)
    check(ctx, F16, (q, kc, vc, table, starts + front, seq, lens), H, f"{front} rows in front")


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
def test_one_column_and_one_page(ctx, dtype):
    check(ctx, dtype, problem(1, dtype, [3, 1], [0, 2], 2, 1, 64, 16), 2, "one page each")
    check(ctx, dtype, problem(2, dtype, [200], [0], 2, 1, 128, 200), 2, "a page for all")
    check(ctx, dtype, problem(3, dtype, [5], [1000], 2, 1, 8, 1005), 2, "a page that is no multiple of a run")


@pytest.mark.parametrize("page", [2, 4, 6, 8, 12, 40, 64])
@pytest.mark.parametrize("dtype", [F32, BF16])
def test_page_sizes(ctx, page, dtype):
    """Pages that end within a run of tokens, and runs that fill them; heads of 96 and 128 channels."""
    for D in (96, 128):
        check(ctx, dtype, problem(page, dtype, [70, 1, 9], [130, 55, 0], 4, 2, D, page), 4, f"pages of {page}, {D}")
        check(ctx, dtype, problem(page, dtype, [150, 60], [200, 3], 64, 4, D, page), 64, f"pages of {page}, {D}, wide", window=90)


@pytest.mark.parametrize("scale", [math.nan, math.inf, -math.inf])
def test_scales_that_are_not_finite(ctx, scale):
    run_chunk(ctx, F16, *problem(4, F16, [4, 2], [3, 0], 4, 2, 64, 16), 4, scale=scale, expect=abi.ERR_INVALID_ARGUMENT)


@pytest.mark.parametrize("R", [3, 40])
def test_counts_below_zero(ctx, R):
    """shares that no program of pages leaves behind: the list is written where it may be, and nowhere else."""
    pool, cols = 500, 4
    table = torch.arange(R * cols, dtype=torch.int32).view(R, cols)
    shares = torch.zeros(pool, dtype=torch.int32)
    shares[200:] = -1
    with Device(ctx) as d:
        free, get = d.out(torch.full((pool,), -9, dtype=torch.int32))
        counts, get_counts = d.new(4)
        ctx.paged_release(abi.PagedReleaseArgs(
            requests=R, max_pages=cols, page_size=1, num_pages=pool, free_count=100, lens=d.up(torch.full((R,), cols, dtype=torch.int32)),
            keep_lens=d.up(torch.zeros(R, dtype=torch.int32)), block_table=d.up(table), shares=d.up(shares), free_pages=free,
            free_head=d.up(ints([60])), kv_lens=d.new(R)[0], counts=counts))
        assert (get()[60:] == -9).all()


def test_the_same_page_many_times(ctx):
    """One page in every column of every request: a chunk over it, its release by all, and a compaction."""
    R, cols, page = 5, 7, 16
    q, kc, vc, table, starts, seq, lens = problem(5, BF16, [9] * R, [cols * page - 9] * R, 4, 2, 64, page)
    table[:] = 3
    check(ctx, BF16, (q, kc, vc, table, starts, seq, lens), 4, "one page")
    pool = 40
    with Device(ctx) as d:
        shares, get_shares = d.out(torch.where(torch.arange(pool) == 3, R * cols - 1, 0).to(torch.int32))
        free, get_free = d.out(torch.full((pool,), -9, dtype=torch.int32))
        counts, get_counts = d.new(4)
        where = dict(requests=R, max_pages=cols, page_size=page, num_pages=pool, free_count=pool, lens=d.up(lens), block_table=d.up(table), shares=shares,
                     free_pages=free, counts=counts)
        src, get_src = d.new(4)
        dst, get_dst = d.new(4)
        out, get_out = d.new(R, cols)
        ctx.paged_compact(abi.PagedCompactArgs(limit=2, max_moves=4, table_out=out, shares_out=d.new(pool)[0], copy_src=src, copy_dst=dst, **where))
        assert (get_out() == 0).all() and get_src().tolist() == [3, -1, -1, -1] and get_dst().tolist() == [0, -1, -1, -1]
        assert get_counts().tolist() == [pool - 1, 1, 0, 1] and get_free()[-1] == 1
        ctx.paged_release(abi.PagedReleaseArgs(keep_lens=d.up(torch.zeros(R, dtype=torch.int32)), free_head=d.up(ints([pool])), kv_lens=d.new(R)[0], **where))
        assert get_counts().tolist() == [pool - 1, 1, R * cols - 1, 0] and get_free()[-1] == 3 and (get_shares() == 0).all()
