"""More rows, tokens or pairs than one launch may have threads (2^32)."""
import pytest
import torch

from mlx_amd import abi
from serving_util import F16, F32

pytestmark = pytest.mark.gpu


@pytest.fixture
def wrapped(ctx):
    """Buffers over tensors on the card, freed with the test."""
    bufs = []

    def wrap(*tensors):
        torch.cuda.synchronize()
        bufs.extend(ctx.wrap(t.data_ptr(), t.numel() * t.element_size()) for t in tensors)
        return [b.handle for b in bufs[-len(tensors):]]

    yield wrap
    for b in bufs:
        b.free()
    torch.cuda.empty_cache()


def test_norm_of_many_short_rows(ctx, wrapped):
    T, D = 2 ** 26 + 3, 4
    r = torch.randn(T, D, device="cuda")
    out = torch.full_like(r, float("nan"))
    br, bo = wrapped(r, out)
    ctx.block_norm(abi.BlockNormArgs(rows=T, dim=D, pre_norm=abi.NORM_RMS, residual_scale=1.0, eps=0.01, x_dtype=F32, residual_dtype=F32,
                                     residual=br, out=bo))
    ctx.sync()
    want = r * torch.rsqrt(r.square().mean(-1, keepdim=True) + 0.01)
    assert ((out - want).abs() <= 2.0 ** -20 * (1 + want.abs())).all()


@pytest.mark.parametrize("D,dtype", [(1, F32), (3, F16)])
def test_append_of_many_tokens(ctx, wrapped, D, dtype):
    """A block per token where rows allow no vectors."""
    T, page = 2 ** 24 + 7, 16
    pages = T // page + 1
    t = {F32: torch.float32, F16: torch.float16}[dtype]
    k, v = (torch.randn(T, D, device="cuda").to(t) for _ in range(2))
    kc, vc = (torch.full((pages * page, D), 7.0, dtype=t, device="cuda") for _ in range(2))
    slots = torch.arange(T, dtype=torch.int32, device="cuda").flip(0)
    bk, bv, bs, bkc, bvc = wrapped(k, v, slots, kc, vc)
    ctx.paged_append(abi.PagedAppendArgs(tokens=T, kv_heads=1, head_dim=D, page_size=page, num_pages=pages, in_dtype=dtype, cache_dtype=dtype,
                                         k=bk, v=bv, slots=bs, k_cache=bkc, v_cache=bvc))
    ctx.sync()
    for new, cache in ((k, kc), (v, vc)):
        assert torch.equal(cache[:T], new.flip(0)) and (cache[T:] == 7).all()


def test_attention_of_many_pairs(ctx, wrapped):
    """A block per pair of request and head of keys; a token each, so that out is its value."""
    R, H, D, page = 2 ** 20 + 3, 16, 8, 4
    pages = 1000
    gen = torch.Generator(device="cuda").manual_seed(1)
    kc, vc = (torch.randn(pages, H, page, D, device="cuda", generator=gen).half() for _ in range(2))
    q = torch.randn(R, H * D, device="cuda", generator=gen).half()
    table = torch.randint(0, pages, (R, 1), device="cuda", generator=gen, dtype=torch.int32)
    lens = torch.randint(0, 2, (R,), device="cuda", generator=gen, dtype=torch.int32)
    out, lse = torch.full_like(q, 7.0), torch.full((R, H), 7.0, device="cuda")
    bq, bk, bv, bt, bl, bo, be = wrapped(q, kc, vc, table, lens, out, lse)
    ctx.paged_attention(abi.PagedAttentionArgs(requests=R, heads=H, kv_heads=H, head_dim=D, page_size=page, num_pages=pages, max_pages=1, dtype=F16,
                                               scale=1.0, q=bq, k_cache=bk, v_cache=bv, block_table=bt, kv_lens=bl, out=bo, lse=be))
    ctx.sync()
    on = lens[:, None, None] > 0
    want = torch.where(on, vc[table[:, 0].long(), :, 0], torch.zeros((), dtype=torch.float16, device="cuda"))
    assert torch.equal(out.view(R, H, D), want)
    score = (q.view(R, H, D).float() * kc[table[:, 0].long(), :, 0].float()).sum(-1)
    # 8 products and sums, the factor log2 e and back: 16 roundings of the largest term, and of the score
    bound = 16 * 2.0 ** -24 * (1 + (q.view(R, H, D).float() * kc[table[:, 0].long(), :, 0].float()).abs().sum(-1))
    assert torch.where(on[..., 0], (lse - score).abs() <= bound, lse == -float("inf")).all()
