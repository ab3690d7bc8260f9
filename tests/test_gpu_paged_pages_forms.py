"""Forks, releases and compactions at the sizes where their launches change: forks
of one launch and of two, of a thread each and of several; pools and tables of one
block and of many."""
import pytest
import torch

from prompt_util import ints
from test_gpu_paged_pages import compact, fork, held, release

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("forks", [63, 64, 65, 1023, 1024, 1025, 2049])
@pytest.mark.parametrize("page,cols", [(4, None), (1, 300)])
def test_forks(ctx, forks, page, cols):
    """Every second dst twice, pages that run out, tables of several rounds of a wave."""
    gen = torch.Generator().manual_seed(forks)
    lens, table, shares, free, head = held(forks, torch.randint(0, 290 // (1 if page == 1 else 2), (20,), generator=gen).tolist(), forks, page, cols,
                                           extra=forks // 3)
    src = torch.randint(0, 22, (forks,), generator=gen).to(torch.int32)
    dst = 20 + torch.arange(forks, dtype=torch.int32) // 2 * 2 + (torch.arange(forks) % 5 == 0)
    fork(ctx, src, dst, lens, table, shares, free, head, page, f"{forks} forks")


@pytest.mark.parametrize("requests", [15, 16, 17, 33])
@pytest.mark.parametrize("cols,extra", [(20, 0), (300, 0), (600, 0), (200, 4097)])
def test_releases(ctx, requests, cols, extra):
    """Tables of up to three rounds of a wave, pools around one run of pages."""
    gen = torch.Generator().manual_seed(requests + cols)
    page = 2
    lens = torch.randint(0, 2 * cols + 3, (requests,), generator=gen).tolist()
    lens[0], lens[-1] = 2 * cols, 0
    lens_t, table, shares, free, head = held(requests, [min(n, 2 * cols) for n in lens], 0, page, cols, extra=max(1, extra))
    for r in range(1, requests, 3):  # pages that the request before holds too
        n = -(-min(int(lens_t[r]), int(lens_t[r - 1])) // page) // 2
        lost = table[r, :n].clone()
        table[r, :n] = table[r - 1, :n]
        shares[table[r, :n].long()] += 1
        assert len(lost) == n
    keep = torch.randint(-2, 2 * cols, (requests,), generator=gen).to(torch.int32)
    keep[::4] = 0
    release(ctx, lens_t, keep, table, shares, free, head, page, f"{requests} requests of {cols}")
    release(ctx, lens_t, keep, table, shares, free, head, page, "in place", in_place=True)
    release(ctx, lens_t, torch.zeros_like(keep), table, shares, free, head, page, "all of them")


@pytest.mark.parametrize("pool", [1, 31, 32, 33, 4096, 4097, 8191, 8192, 8193])
def test_releases_of_pools(ctx, pool):
    requests, cols = 12, max(1, min(pool // 12, 900))
    used = torch.randperm(pool, generator=torch.Generator().manual_seed(pool))[:requests * cols]
    table = torch.full((requests * cols,), -1, dtype=torch.int32)
    table[:len(used)] = used.to(torch.int32)
    lens = torch.full((requests,), cols, dtype=torch.int32)
    release(ctx, lens, torch.arange(requests, dtype=torch.int32), table.view(requests, cols), torch.zeros(pool, dtype=torch.int32),
            torch.full((pool,), -9, dtype=torch.int32), pool, 1, f"pool of {pool}")


@pytest.mark.parametrize("in_place", [False, True])
@pytest.mark.parametrize("pool,requests,cols", [(8192, 64, 256), (8193, 64, 256), (8192, 65, 256), (8191, 1, 16384), (8192, 1, 16385), (1, 1, 1),
                                                (33, 2, 3), (8192, 16384, 1), (4096, 7, 301)])
def test_compactions(ctx, pool, requests, cols, in_place):
    """One block's bits and entries, and one more; ids that are none, names that several requests hold, tables without any."""
    gen = torch.Generator().manual_seed(pool + requests)
    page = 2
    table = torch.randint(-1, pool + 1, (requests, cols), generator=gen).to(torch.int32)
    lens = torch.randint(-2, 2 * cols + 3, (requests,), generator=gen).to(torch.int32)
    shares = torch.randint(0, 3, (pool,), generator=gen).to(torch.int32)
    for limit, free, moves in [(pool, pool, 0), (pool // 2, pool, pool), (pool // 3 + 1, 50, 40), (0, pool, 3), (pool - 1, 0, pool)]:
        compact(ctx, lens, table, shares, torch.full((free,), -7, dtype=torch.int32), limit, moves, page, f"limit {limit}, {moves} moves", in_place)
    compact(ctx, torch.zeros_like(lens), table, shares, torch.full((pool,), -7, dtype=torch.int32), pool // 2, 5, page, "nothing held", in_place)


def test_releases_of_long_tables(ctx):
    """A request of a hundred thousand pages beside short ones."""
    cols = 100000
    table = torch.full((3, cols), -1, dtype=torch.int32)
    order = torch.randperm(cols + 40, generator=torch.Generator().manual_seed(1)).to(torch.int32)
    table[0], table[1, :20], table[2, :20] = order[:cols], order[cols:cols + 20], order[cols + 20:]
    lens = ints([cols, 20, 20])
    release(ctx, lens, ints([17, 0, 20]), table, torch.zeros(cols + 40, dtype=torch.int32), torch.full((cols + 40,), -1, dtype=torch.int32),
            cols + 40, 1, "long")
