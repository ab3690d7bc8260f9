"""Forks, releases, compactions and copies of pages against their definitions
(prompt_util.py): whole numbers, equal in every place."""
import itertools

import pytest
import torch

from mlx_amd import abi
from prompt_util import compact_reference, fork_reference, ints, release_reference, table_of
from serving_util import BF16, F16, F32, Device, randn

pytestmark = pytest.mark.gpu


def run(ctx, op, record, arrays, outs, expect=None, **over):
    """One call: `arrays` by field, those named in `outs` downloaded after it."""
    with Device(ctx) as d:
        get = {}
        fields = {}
        for k, t in arrays.items():
            h, g = d.out(t)
            fields[k] = h
            if k in outs:
                get[k] = g
        a = record(**fields)
        for k, v in over.items():
            setattr(a, k, v)
        rc = getattr(ctx.p, op)(ctx.handle, a)
        if expect is not None:
            assert rc == expect, rc
            return None
        assert rc == 0, rc
        return {k: g() for k, g in get.items()}


def same(got, want, what):
    for k, v in want.items():
        assert torch.equal(got[k], v), f"{what}: {k}\n{got[k]}\n{v}"


def fork(ctx, src, dst, lens, table, shares, free, head, page, what, /, **kw):
    F, n = len(src), dict(forks=len(src), requests=len(lens), max_pages=table.shape[1], page_size=page, num_pages=len(shares), free_count=len(free))
    n.update(kw)
    new = lambda k: torch.full((k,), -7, dtype=torch.int32)  # noqa: E731
    got = run(ctx, "op_paged_fork", abi.PagedForkArgs,
              dict(src=src, dst=dst, lens=lens, block_table=table, shares=shares, free_pages=free, free_head=ints([head]), copy_src=new(F),
                   copy_dst=new(F), counts=new(4)), ("lens", "block_table", "shares", "copy_src", "copy_dst", "counts", "free_pages"), **n)
    if got is not None:
        same(got, fork_reference(src, dst, lens, table, shares, free, head, page), what)
        assert torch.equal(got["free_pages"], free)
    return got


def held(seed, lens, rows, page, cols=None, extra=9):
    """Requests with tables, `rows` empty ones behind them: lens, table, shares, free list, its head"""
    gen = torch.Generator().manual_seed(seed)
    table, pool = table_of(gen, lens, page, cols, extra)
    table = torch.cat([table, torch.full((rows, table.shape[1]), -1, dtype=torch.int32)])
    named = set(table.view(-1).tolist())
    rest = [p for p in torch.randperm(pool, generator=gen).tolist() if p not in named]
    used = [p for p in range(pool) if p in named]
    return ints(list(lens) + [0] * rows), table, torch.zeros(pool, dtype=torch.int32), ints(used + rest), len(used)


@pytest.mark.parametrize("page", [1, 4, 16, 7])
def test_forks(ctx, page):
    lens, table, shares, free, head = held(1, [0, 1, 5, 16, 33, 64, 100], 12, page)
    src = ints([4, 4, 4, 2, 6, 0, 5, 3, 1])
    fork(ctx, src, ints(list(range(7, 16))), lens, table, shares, free, head, page, f"page {page}")


def test_forks_that_are_left_out(ctx):
    """Numbers outside, a request onto itself, one that holds something, the same one twice, one that another fork fills."""
    lens, table, shares, free, head = held(2, [20, 7, 33], 6, 8)
    lens[4] = -3
    src, dst = ints([0, 0, -1, 9, 1, 0, 2, 1, 3, 2, 2]), ints([3, 1, 4, 4, 1, 9, 3, 4, 5, 5, -1])
    got = fork(ctx, src, dst, lens, table, shares, free, head, 8, "left out")
    assert got["counts"][3] == 8


def test_forks_without_pages(ctx):
    """The list ends after two of the forks; heads below 0 and past the list; holes in the source's table."""
    lens, table, shares, free, head = held(3, [20, 17], 8, 8, extra=2)
    table[1, 1] = -1
    for h in (head, len(free), len(free) + 5):
        fork(ctx, ints([0, 1, 0, 0]), ints([2, 3, 4, 5]), lens, table, shares, free, h, 8, f"head {h}")
    fork(ctx, ints([0]), ints([2]), lens, table, shares, free, -4, 8, "head -4")
    table[1, 2], table[0, 0] = -1, 1 << 29
    fork(ctx, ints([0, 1, 0, 0]), ints([2, 3, 4, 5]), lens, table, shares, free, head, 8, "holes")


def test_many_forks(ctx):
    """More than one block's, and tables of more than one launch: some of them of the same request."""
    gen = torch.Generator().manual_seed(4)
    lens, table, shares, free, head = held(4, torch.randint(0, 200, (50,), generator=gen).tolist(), 3000, 4, extra=2500)
    src = torch.randint(0, 50, (2700,), generator=gen).to(torch.int32)
    dst = torch.randint(50, 3050, (2700,), generator=gen).to(torch.int32)
    fork(ctx, src, dst, lens, table, shares, free, head, 4, "many")


@pytest.mark.parametrize("n", [0, 1])
def test_few_forks(ctx, n):
    lens, table, shares, free, head = held(5, [9], 2, 4)
    fork(ctx, ints([0] * n), ints([1] * n), lens, table, shares, free, head, 4, f"{n} forks")


def release(ctx, lens, keep, table, shares, free, head, page, what, in_place=False, **kw):
    n = dict(requests=len(lens), max_pages=table.shape[1], page_size=page, num_pages=len(shares), free_count=len(free))
    n.update(kw)
    with Device(ctx) as d:
        kv, get_kv = d.out(lens if in_place else torch.full_like(lens, -7))
        sh, get_shares = d.out(shares)
        fr, get_free = d.out(free)
        ct, get_counts = d.new(4)
        a = abi.PagedReleaseArgs(lens=kv if in_place else d.up(lens), keep_lens=d.up(keep), block_table=d.up(table), shares=sh, free_pages=fr,
                                 free_head=d.up(ints([head])), kv_lens=kv, counts=ct, **n)
        ctx.paged_release(a)
        got = {"kv_lens": get_kv(), "shares": get_shares(), "free_pages": get_free(), "counts": get_counts()}
    same(got, release_reference(lens, keep, table, shares, free, head, page), what)
    return got


@pytest.mark.parametrize("in_place", [False, True])
@pytest.mark.parametrize("page", [1, 4, 16])
def test_releases(ctx, page, in_place):
    lens, table, shares, free, head = held(6, [0, 1, 5, 16, 33, 64, 100, 50], 2, page)
    keep = ints([0, 0, 5, 1, 20, 1000, -5, 48, 7, 0])
    release(ctx, lens, keep, table, shares, free, head, page, f"page {page}", in_place)


@pytest.mark.parametrize("requests", [30, 3000])
def test_releases_of_shared_pages(ctx, requests):
    """Pages with several holders: some let go, all let go, more than hold them; small and large pools."""
    gen = torch.Generator().manual_seed(7)
    page, cols = 4, 10
    pool = requests * 14
    table = torch.randint(0, pool // 3, (requests, cols), generator=gen).to(torch.int32)
    table[:, 7] = pool // 3 + torch.arange(requests)
    table[::5, 3] = -1
    table[1::7, 2] = pool
    lens = torch.randint(-3, 50, (requests,), generator=gen).to(torch.int32)
    keep = torch.where(torch.rand(requests, generator=gen) < 0.5, 0, torch.randint(-3, 50, (requests,), generator=gen)).to(torch.int32)
    holders = torch.zeros(pool, dtype=torch.int32)
    for r in range(requests):
        for c in range(min(cols, -(-max(0, int(lens[r])) // page))):
            if 0 <= int(table[r, c]) < pool:
                holders[int(table[r, c])] += 1
    shares = (holders - 1).clamp(min=0)
    free = torch.arange(pool, dtype=torch.int32)
    release(ctx, lens, keep, table, shares, free, pool - 5, page, "shared")
    release(ctx, lens, keep, table, (shares - 1).clamp(min=0), free, pool - 5, page, "held less often than named")


@pytest.mark.parametrize("requests", [10, 5000])
def test_lists_without_room(ctx, requests):
    page = 2
    table = torch.arange(requests * 3, dtype=torch.int32).flip(0).view(requests, 3).contiguous()
    lens, keep = torch.full((requests,), 6, dtype=torch.int32), torch.full((requests,), 1, dtype=torch.int32)
    shares = torch.zeros(requests * 3 + 5, dtype=torch.int32)
    for free, head in [(8, 3), (8, 0), (0, 0), (8, -4), (8, 100), (requests * 3, requests * 3)]:
        release(ctx, lens, keep, table, shares, torch.full((free,), 77, dtype=torch.int32), head, page, f"list of {free} from {head}")


def compact(ctx, lens, table, shares, free, limit, moves, page, what, in_place=False):
    n = dict(requests=len(lens), max_pages=table.shape[1], page_size=page, num_pages=len(shares), free_count=len(free), limit=limit, max_moves=moves)
    with Device(ctx) as d:
        new = lambda t: torch.full_like(t, -7)  # noqa: E731
        t_out, get_table = d.out(table if in_place else new(table))
        s_out, get_shares = d.out(shares if in_place else new(shares))
        fr, get_free = d.out(free)
        cs, get_src = d.new(moves)
        cd, get_dst = d.new(moves)
        ct, get_counts = d.new(4)
        ctx.paged_compact(abi.PagedCompactArgs(
            lens=d.up(lens), block_table=t_out if in_place else d.up(table), shares=s_out if in_place else d.up(shares), table_out=t_out,
            shares_out=s_out, free_pages=fr, copy_src=cs, copy_dst=cd, counts=ct, **n))
        got = {"table_out": get_table(), "shares_out": get_shares(), "free_pages": get_free(), "copy_src": get_src(), "copy_dst": get_dst(),
               "counts": get_counts()}
    same(got, compact_reference(lens, table, shares, free, limit, moves, page), what)
    return got


@pytest.mark.parametrize("in_place", [False, True])
@pytest.mark.parametrize("page,extra", [(1, 30), (4, 100), (16, 70)])
def test_compactions(ctx, page, extra, in_place):
    lens, table, shares, free, _ = held(8, [0, 1, 5, 16, 33, 64, 100, 50], 2, page, extra=extra)
    pool = len(shares)
    table[5, 0] = table[6, 0]
    shares[int(table[6, 0])] = 1
    for limit, moves in itertools.product((0, 1, pool // 3, pool // 2 + 1, pool - 1, pool), (0, 5, pool)):
        compact(ctx, lens, table, shares, free, limit, moves, page, f"limit {limit}, {moves} moves", in_place)


def test_compactions_of_large_pools(ctx):
    gen = torch.Generator().manual_seed(9)
    pool, page = 100003, 2
    table = torch.randint(-1, pool + 1, (900, 40), generator=gen).to(torch.int32)
    lens = torch.randint(-2, 90, (900,), generator=gen).to(torch.int32)
    shares = torch.randint(0, 3, (pool,), generator=gen).to(torch.int32)
    for limit, free in [(50000, pool), (50000, 1000), (20000, pool), (99999, 0)]:
        compact(ctx, lens, table, shares, torch.full((free,), -7, dtype=torch.int32), limit, pool, page, f"limit {limit}")


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("layers,Hk,page,D,extra", [(1, 2, 16, 64, 0), (3, 8, 16, 128, 0), (2, 1, 3, 7, 0), (2, 3, 5, 24, 11), (1, 1, 1, 1, 0), (2, 16, 64, 128, 64)])
def test_copies(ctx, dtype, layers, Hk, page, D, extra):
    gen = torch.Generator().manual_seed(10)
    pool = 20
    one = pool * Hk * page * D
    caches = [randn(gen, dtype, layers * (one + extra)) for _ in range(2)]
    src, dst = ints([3, -1, 5, 7, 3, 20, 1, 9]), ints([0, 4, 19, -1, 11, 6, 25, 9])
    want = [c.clone() for c in caches]
    for c in want:
        for x in range(layers):
            pages = c[x * (one + extra):x * (one + extra) + one].view(pool, -1)
            for s, d in ((3, 0), (5, 19), (3, 11)):
                pages[d] = pages[s].clone()
    got = run(ctx, "op_paged_copy", abi.PagedCopyArgs, dict(copy_src=src, copy_dst=dst, k_cache=caches[0], v_cache=caches[1]), ("k_cache", "v_cache"),
              pages=len(src), layers=layers, kv_heads=Hk, head_dim=D, page_size=page, num_pages=pool, dtype=dtype, layer_stride=one + extra)
    for name, w in zip(("k_cache", "v_cache"), want):
        assert torch.equal(got[name].view(-1).view(torch.uint8), w.view(torch.uint8)), name


def test_copies_into_wrapped_caches(ctx):
    """Caches that start on any element."""
    for off in (1, 3, 8):
        t = torch.arange(off + 10 * 64, device="cuda").to(torch.float16)
        u = t.clone()
        s, d = (torch.tensor(v, dtype=torch.int32, device="cuda") for v in ([1, 2], [5, 9]))
        torch.cuda.synchronize()
        bufs = [ctx.wrap(x.data_ptr() + o * x.element_size(), (x.numel() - o) * x.element_size()) for x, o in ((t, off), (u, off), (s, 0), (d, 0))]
        ctx.paged_copy(abi.PagedCopyArgs(pages=2, layers=1, kv_heads=1, head_dim=8, page_size=8, num_pages=10, dtype=F16, copy_src=bufs[2].handle,
                                         copy_dst=bufs[3].handle, k_cache=bufs[0].handle, v_cache=bufs[1].handle))
        ctx.sync()
        want = torch.arange(off + 640).to(torch.float16)
        pages = want[off:].view(10, 64)
        pages[5], pages[9] = pages[1].clone(), pages[2].clone()
        assert torch.equal(t.cpu(), want) and torch.equal(u.cpu(), want)
        for b in bufs:
            b.free()


BAD_PAGES = [dict(struct_size=5), dict(requests=-1), dict(max_pages=0), dict(page_size=0), dict(num_pages=-1), dict(free_count=-1), dict(shares=None),
             dict(block_table=None), dict(counts=None), dict(lens=None), dict(num_pages=1000), dict(requests=100), dict(free_count=1000)]


@pytest.mark.parametrize("over", BAD_PAGES + [dict(forks=-1), dict(forks=9), dict(src=None), dict(copy_dst=None)])
def test_fork_refusals(ctx, over):
    lens, table, shares, free, head = held(11, [9], 2, 4)
    fork(ctx, ints([0]), ints([1]), lens, table, shares, free, head, 4, "", expect=abi.ERR_INVALID_ARGUMENT, **over)


@pytest.mark.parametrize("over", BAD_PAGES + [dict(keep_lens=None), dict(kv_lens=None)])
def test_release_refusals(ctx, over):
    lens, table, shares, free, head = held(11, [9], 2, 4)
    n = dict(requests=3, max_pages=table.shape[1], page_size=4, num_pages=len(shares), free_count=len(free))
    run(ctx, "op_paged_release", abi.PagedReleaseArgs,
        dict(lens=lens, keep_lens=lens, block_table=table, shares=shares, free_pages=free, free_head=ints([head]), kv_lens=lens.clone(),
             counts=ints([0] * 4)), (), expect=abi.ERR_INVALID_ARGUMENT, **{**n, **over})


@pytest.mark.parametrize("over", BAD_PAGES + [dict(limit=-1), dict(limit=1000), dict(max_moves=-1), dict(max_moves=9), dict(table_out=None)])
def test_compact_refusals(ctx, over):
    lens, table, shares, free, head = held(11, [9], 2, 4)
    n = dict(requests=3, max_pages=table.shape[1], page_size=4, num_pages=len(shares), free_count=len(free), limit=3, max_moves=2)
    run(ctx, "op_paged_compact", abi.PagedCompactArgs,
        dict(lens=lens, block_table=table, shares=shares, table_out=table.clone(), shares_out=shares.clone(), free_pages=free, copy_src=ints([0] * 2),
             copy_dst=ints([0] * 2), counts=ints([0] * 4)), (), expect=abi.ERR_INVALID_ARGUMENT, **{**n, **over})


@pytest.mark.parametrize("code,over", [(abi.ERR_INVALID_ARGUMENT, o) for o in (
    dict(struct_size=0), dict(pages=-1), dict(pages=9), dict(layers=-1), dict(layers=9), dict(kv_heads=0), dict(num_pages=99), dict(layer_stride=7),
    dict(copy_src=None), dict(k_cache=None))] + [(abi.ERR_NOT_SUPPORTED, dict(dtype=9)), (abi.ERR_NOT_SUPPORTED, dict(num_pages=1 << 30))])
def test_copy_refusals(ctx, code, over):
    n = dict(pages=2, layers=1, kv_heads=2, head_dim=8, page_size=4, num_pages=6, dtype=F32)
    run(ctx, "op_paged_copy", abi.PagedCopyArgs, dict(copy_src=ints([1, 2]), copy_dst=ints([3, 4]), k_cache=torch.zeros(6 * 64), v_cache=torch.zeros(6 * 64)),
        (), expect=code, **{**n, **over})


def test_outputs_over_others_are_refused(ctx):
    lens, table, shares, free, head = held(11, [9], 2, 4)
    with Device(ctx) as d:
        b = {k: d.up(t) for k, t in dict(lens=lens, block_table=table, shares=shares, free_pages=free, free_head=ints([head]), counts=ints([0] * 4)).items()}
        n = dict(requests=3, max_pages=table.shape[1], page_size=4, num_pages=len(shares), free_count=len(free))
        rc = ctx.p.op_paged_release(ctx.handle, abi.PagedReleaseArgs(**n, **{**b, "counts": b["shares"]}, keep_lens=d.up(lens), kv_lens=d.up(lens)))
        assert rc == abi.ERR_INVALID_ARGUMENT
        keep = d.up(lens)
        rc = ctx.p.op_paged_release(ctx.handle, abi.PagedReleaseArgs(**n, **b, keep_lens=keep, kv_lens=keep))
        assert rc == abi.ERR_INVALID_ARGUMENT
        rc = ctx.p.op_paged_fork(ctx.handle, abi.PagedForkArgs(forks=1, **n, **{**b, "counts": b["free_head"]}, src=d.up(ints([0])), dst=d.up(ints([1])),
                                                               copy_src=d.up(ints([0])), copy_dst=d.up(ints([0]))))
        assert rc == abi.ERR_INVALID_ARGUMENT
