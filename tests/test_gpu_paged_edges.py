"""Paged attention at the edges of its numbers, against 64 bits."""
import pytest
import torch

from serving_util import BF16, F16, F32, ROUND, TORCH
from test_gpu_paged_attention import attend

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("far", [10, 16, 18, 22, 30])
def test_very_many_small_weights(ctx, dtype, far):
    """One token of value 0 and 20000 of weight exp(-far) beside it: together they are the result."""
    D, page, N, R = 64, 64, 20000, 512  # so many requests that few waves share one
    gen = torch.Generator().manual_seed(far)
    pages = -(-N // page)
    kc = torch.zeros(pages, 1, page, D, dtype=TORCH[dtype])
    vc = (1 + 0.25 * torch.rand(pages, 1, page, D, generator=gen)).to(TORCH[dtype])
    kc[0, 0, 7, 0], vc[0, 0, 7] = far, 0
    q = torch.zeros(R, D, dtype=TORCH[dtype])
    q[:, 0] = 8
    table, n = torch.randperm(pages, generator=gen).to(torch.int32).expand(R, pages).contiguous(), torch.full((R,), N, dtype=torch.int32)
    got, lse = attend(ctx, q, kc, vc, table, n, 1, dtype)
    t = torch.arange(N)
    pg = table[0, t // page].long()
    s = kc[pg, 0, t % page, 0].double()
    p = torch.exp(s - far)
    want = (p @ vc[pg, 0, t % page].double()) / p.sum()
    # the weights are off by what 3 roundings move a score of `far`, and by 64 more of the exp2, and sums of N / 16 terms
    # by as many; as they enter the product with v they are off by 2^-16 (bf16) or 2^-21 (f16) of themselves and, in f16, 2^-36
    own = {F32: 0.0, F16: 2.0 ** -21, BF16: 2.0 ** -16}[dtype]
    bound = want * ((3 * far + 64 + N / 16) * 2.0 ** -24 + own + ROUND[dtype])
    if dtype == F16:
        bound = bound + 1.25 * N * 2.0 ** -36 / p.sum() + 2.0 ** -25
    assert ((got.double() - want).abs() <= bound).all(), float(((got.double() - want).abs() / bound).max())
    assert ((lse.double() - (far + torch.log(p.sum()))).abs() <= (3 * far + 64 + N / 16) * 2.0 ** -24).all()
