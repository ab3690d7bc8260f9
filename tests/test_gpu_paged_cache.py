"""The paged plan (whole numbers, against a walk over requests and tokens) and
the append (every bit, against torch's rounding)."""
import pytest
import torch

from mlx_amd import abi
from serving_util import BF16, F16, F32, TORCH, Device, plan_reference, randn

pytestmark = pytest.mark.gpu

OUT = ["block_table", "slots", "positions", "token_request", "token_starts", "kv_lens", "counts"]


def plan(ctx, seq, new, free, head, table, page, pool, max_tokens, some_null=False):
    R = len(seq)
    i32 = lambda v: torch.as_tensor(v, dtype=torch.int32)  # noqa: E731
    with Device(ctx) as dev:
        h, get = {}, {}
        h["block_table"], get["block_table"] = dev.out(table)
        for k, n in [("slots", max_tokens), ("positions", max_tokens), ("token_request", max_tokens), ("token_starts", R + 1),
                     ("kv_lens", R), ("counts", 4)]:
            h[k], get[k] = dev.new(n)
        if some_null:
            h["positions"] = h["token_request"] = None
        args = abi.PagedPlanArgs(requests=R, max_tokens=max_tokens, max_pages=table.shape[1], page_size=page, num_pages=pool,
                                 free_count=len(free), seq_lens=dev.up(i32(seq)), new_lens=dev.up(i32(new)), free_pages=dev.up(i32(free)),
                                 free_head=dev.up(i32([head])), **h)
        ctx.paged_plan(args)
        first = {k: get[k]() for k in OUT}
        ctx.paged_plan(args)  # the same record again: the same plan
        assert all(torch.equal(get[k](), first[k]) for k in OUT)
        return first


def check_plan(ctx, seq, new, page, cols, spare=0, head=0, max_tokens=None, seed=0, pool=None, some_null=False):
    gen = torch.Generator().manual_seed(seed)
    R = len(seq)
    held = [-(-min(max(s, 0), cols * page) // page) for s in seq]
    want = sum(max(0, min(-(-(min(max(s, 0), cols * page) + max(n, 0)) // page), cols) - h) for s, n, h in zip(seq, new, held))
    pages = torch.randperm(sum(held) + head + want + 8, generator=gen).tolist()
    table = torch.full((R, cols), -1, dtype=torch.int32)
    at = 0
    for r in range(R):
        table[r, :held[r]] = torch.tensor(pages[at:at + held[r]], dtype=torch.int32)
        at += held[r]
    free = pages[at:][:max(0, head + want + spare)]
    T = max_tokens if max_tokens is not None else sum(max(n, 0) for n in new) + 5
    print(f"[case] R={R} page={page} cols={cols} T={T} head={head} spare={spare}", flush=True)
    got = plan(ctx, seq, new, free, head, table, page, pool or len(pages), T, some_null)
    ref = plan_reference(seq, new, free, head, table, page, pool or len(pages), T)
    for k in OUT:
        if not (some_null and k in ("positions", "token_request")):
            assert torch.equal(got[k], ref[k]), (k, got[k], ref[k])


@pytest.mark.parametrize("page", [1, 3, 16, 64])
def test_plan_lengths(ctx, page):
    seq = [0, 0, 1, page - 1, page, page + 1, 5 * page, 7, 0, 100]
    new = [0, 1, 1, 1, 1, 1, 3 * page + 1, 0, 2 * page, 33]
    check_plan(ctx, seq, new, page, 200, head=3, seed=page)
    check_plan(ctx, seq, new, page, 200, head=0, spare=-2, seed=page + 1)   # the last pages are not there
    check_plan(ctx, seq, new, page, 200, head=2, spare=-400, seed=page + 2)  # nothing is left
    check_plan(ctx, seq, new, page, 6, head=1, seed=page + 3)                # rows of the table that are too short
    check_plan(ctx, seq, new, page, 200, max_tokens=10, seed=page + 4)       # more tokens than entries
    check_plan(ctx, seq, new, page, 200, max_tokens=0, seed=page + 5)
    check_plan(ctx, seq, new, page, 200, pool=9, seed=page + 6)              # pages outside the pool
    check_plan(ctx, seq, new, page, 200, some_null=True, seed=page + 7)


def test_plan_negative_lengths_and_head(ctx):
    check_plan(ctx, [-5, 3, 10 ** 6], [4, -2, 7], 16, 9, seed=1)
    table = torch.full((1, 4), -1, dtype=torch.int32)
    got = plan(ctx, [0], [20], [7, 3, 1], -9, table, 16, 8, 20)
    assert got["block_table"].tolist() == [[7, 3, -1, -1]] and got["counts"].tolist() == [2, 20, 0, 0]
    got = plan(ctx, [0], [20], [7, 3, 1], 5, table, 16, 8, 20)  # a head past the list
    assert got["block_table"].tolist() == [[-1, -1, -1, -1]] and got["counts"].tolist() == [5, 20, 2, 20]


@pytest.mark.parametrize("R", [1, 2, 63, 64, 65, 255, 256, 257, 1023, 1024, 1025, 3000, 5000])
def test_plan_many_requests(ctx, R):
    gen = torch.Generator().manual_seed(R)
    seq = torch.randint(0, 100, (R,), generator=gen).tolist()
    new = (torch.randint(0, 3, (R,), generator=gen) * (torch.rand(R, generator=gen) < 0.7)).int().tolist()
    new[R // 2] += 300
    check_plan(ctx, seq, new, 16, 40, spare=-3 if R % 2 else 4, seed=R)


def test_plan_no_requests(ctx):
    got = plan(ctx, [], [], [1, 2], 1, torch.zeros(0, 3, dtype=torch.int32), 16, 4, 3)
    assert got["token_starts"].tolist() == [0] and got["counts"].tolist() == [1, 0, 0, 0] and got["slots"].tolist() == [-1] * 3


def test_plan_refusals(ctx):
    I, N = abi.ERR_INVALID_ARGUMENT, abi.ERR_NOT_SUPPORTED
    z = lambda n: torch.zeros(n, dtype=torch.int32)  # noqa: E731
    with Device(ctx) as dev:
        def record(**over):
            r = dict(requests=2, max_tokens=4, max_pages=3, page_size=16, num_pages=8, free_count=5)
            r.update({k: dev.up(z(n)) for k, n in [("seq_lens", 2), ("new_lens", 2), ("free_pages", 5), ("free_head", 1), ("block_table", 6),
                                                  ("slots", 4), ("positions", 4), ("token_request", 4), ("token_starts", 3),
                                                  ("kv_lens", 2), ("counts", 4)]})
            r.update(over)
            return abi.PagedPlanArgs(**r)
        call = lambda a: ctx.s.op_paged_plan(ctx.handle, a)  # noqa: E731
        assert call(record()) == abi.OK
        for over, want in [(dict(requests=-1), I), (dict(requests=3), I), (dict(max_tokens=-1), I), (dict(max_tokens=5), I),
                           (dict(max_pages=0), I), (dict(max_pages=4), I), (dict(page_size=0), I), (dict(num_pages=-1), I),
                           (dict(free_count=6), I), (dict(free_count=-1), I), (dict(page_size=2 ** 30), N),
                           (dict(seq_lens=None), I), (dict(slots=None), I), (dict(counts=None), I), (dict(free_head=None), I)]:
            assert call(record(**over)) == want, over
        for a, b in [("counts", "free_head"), ("kv_lens", "seq_lens"), ("slots", "positions"), ("block_table", "free_pages")]:
            r = record()
            setattr(r, a, getattr(r, b))
            assert call(r) == I, (a, b)
        r = record()
        r.struct_size += 8
        assert call(r) == I


def append(ctx, k, v, slots, kc, vc, in_dt, cache_dt, k_off=0, k_stride=0, v_off=0, v_stride=0, handles=None):
    pages, Hk, page, D = kc.shape
    with Device(ctx) as dev:
        kh, kget = dev.out(kc)
        vh, vget = dev.out(vc)
        kin = dev.up(k)
        vin = kin if v is None else dev.up(v)
        ctx.paged_append(abi.PagedAppendArgs(
            tokens=len(slots), kv_heads=Hk, head_dim=D, page_size=page, num_pages=pages, in_dtype=in_dt, cache_dtype=cache_dt,
            k_offset=k_off, k_row_stride=k_stride, v_offset=v_off, v_row_stride=v_stride, k=kin, v=vin,
            slots=dev.up(slots), k_cache=kh, v_cache=vh))
        return kget(), vget()


def append_reference(rows, slots, cache):
    cache = cache.clone()
    pages, Hk, page, D = cache.shape
    for t, s in enumerate(slots.tolist()):
        if 0 <= s < pages * page:
            cache[s // page, :, s % page] = rows[t].view(Hk, D).to(cache.dtype)
    return cache


def same_bits(a, b):
    i = torch.int16 if a.element_size() == 2 else torch.int32
    nan = torch.isnan(a) & torch.isnan(b)
    return bool(((a.view(i) == b.view(i)) | nan).all())


@pytest.mark.parametrize("in_dt", [F32, F16, BF16])
@pytest.mark.parametrize("cache_dt", [F32, F16, BF16])
@pytest.mark.parametrize("Hk,D,page,T", [(8, 128, 16, 37), (1, 64, 24, 100), (3, 80, 1, 9), (2, 5, 7, 33), (5, 256, 32, 1), (1, 1, 3, 11),
                                         (16, 256, 8, 40)])
def test_append(ctx, in_dt, cache_dt, Hk, D, page, T):
    gen = torch.Generator().manual_seed(T + D + 10 * in_dt + cache_dt)
    pages = -(-T // page) + 3
    slots = torch.randperm(pages * page, generator=gen)[:T].to(torch.int32)
    slots[::5] = torch.tensor([-1, pages * page, -2 ** 31, 2 ** 31 - 1])[torch.randint(0, 4, (len(slots[::5]),), generator=gen)].to(torch.int32)
    k, v = randn(gen, in_dt, T, Hk * D), randn(gen, in_dt, T, Hk * D)
    k[0, 0], v[-1, -1] = float("inf"), float("nan")
    k[T // 2] *= 1e5  # past f16
    v[T // 2] *= 1e-7
    kc, vc = randn(gen, cache_dt, pages, Hk, page, D), randn(gen, cache_dt, pages, Hk, page, D)
    print(f"[case] in={in_dt} cache={cache_dt} Hk={Hk} D={D} page={page} T={T}", flush=True)
    gk, gv = append(ctx, k, v, slots, kc, vc, in_dt, cache_dt)
    assert same_bits(gk, append_reference(k, slots, kc)) and same_bits(gv, append_reference(v, slots, vc))


@pytest.mark.parametrize("in_dt,cache_dt", [(F32, F32), (F16, F16), (BF16, F16), (F32, BF16)])
@pytest.mark.parametrize("q,odd", [(4 * 64, 0), (3, 1), (8, 4)])
def test_append_out_of_a_fused_projection(ctx, in_dt, cache_dt, q, odd):
    """Queries, keys and values side by side in one buffer, at even and odd places."""
    Hk, D, page, T = 2, 64, 16, 21
    gen = torch.Generator().manual_seed(q)
    stride = q + 2 * Hk * D + odd
    store = randn(gen, in_dt, T * stride)
    slots = torch.randperm(64, generator=gen)[:T].to(torch.int32)
    kc, vc = randn(gen, cache_dt, 4, Hk, page, D), randn(gen, cache_dt, 4, Hk, page, D)
    rows = lambda off: torch.as_strided(store, (T, Hk * D), (stride, 1), off)  # noqa: E731
    # the last row of v ends at or before the buffer's end
    gk, gv = append(ctx, store, None, slots, kc, vc, in_dt, cache_dt, k_off=q, k_stride=stride, v_off=q + Hk * D, v_stride=stride)
    assert same_bits(gk, append_reference(rows(q), slots, kc)) and same_bits(gv, append_reference(rows(q + Hk * D), slots, vc))


def test_append_refusals(ctx):
    I, N = abi.ERR_INVALID_ARGUMENT, abi.ERR_NOT_SUPPORTED
    with Device(ctx) as dev:
        def record(**over):
            r = dict(tokens=3, kv_heads=2, head_dim=8, page_size=4, num_pages=5, in_dtype=F32, cache_dtype=F16,
                     k=dev.up(torch.zeros(3, 16)), v=dev.up(torch.zeros(3, 16)), slots=dev.up(torch.zeros(3, dtype=torch.int32)),
                     k_cache=dev.up(torch.zeros(5, 2, 4, 8, dtype=torch.float16)), v_cache=dev.up(torch.zeros(5, 2, 4, 8, dtype=torch.float16)))
            r.update(over)
            return abi.PagedAppendArgs(**r)
        call = lambda a: ctx.s.op_paged_append(ctx.handle, a)  # noqa: E731
        assert call(record()) == abi.OK and call(record(tokens=0)) == abi.OK and call(record(num_pages=0)) == abi.OK
        for over, want in [(dict(tokens=-1), I), (dict(tokens=4), I), (dict(kv_heads=0), I), (dict(head_dim=9), I), (dict(page_size=0), I),
                           (dict(num_pages=6), I), (dict(in_dtype=4), N), (dict(cache_dtype=9), N), (dict(cache_dtype=F32), I),
                           (dict(k_row_stride=15), I), (dict(k_row_stride=17), I), (dict(v_offset=1), I), (dict(v_offset=-1), I),
                           (dict(k=None), I), (dict(v_cache=None), I), (dict(slots=None), I),
                           (dict(num_pages=2 ** 30, page_size=2), N)]:
            assert call(record(**over)) == want, over
        r = record()
        r.v_cache = r.k_cache
        assert call(r) == I
        r = record(cache_dtype=F32, in_dtype=F32)
        r.struct_size = 0
        assert call(r) == I
