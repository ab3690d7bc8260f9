"""Paged attention at the edges of its numbers, against 64 bits."""
import pytest
import torch

from mlx_amd import abi
from serving_util import BF16, F16, F32, ROUND, TORCH, Device, attention_reference, check_attention, randn
from test_gpu_paged_attention import _record, attend, problem

pytestmark = pytest.mark.gpu
INF = float("inf")


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


def check_with_infinities(got, lse, ref, v_max, dtype, what):
    """Infinities and NaN where the definition has them; the rest as in the other tests."""
    out, want_lse, tol = ref
    got = got.double().view(out.shape)
    assert torch.equal(torch.isnan(got), torch.isnan(out)), what
    odd = ~torch.isfinite(out)
    assert torch.equal(torch.isinf(got), torch.isinf(out)) and torch.equal(got[torch.isinf(out)], out[torch.isinf(out)]), what
    check_attention(torch.where(odd, 0.0, got).to(TORCH[dtype]), lse, (torch.where(odd, 0.0, out), want_lse, tol), v_max, dtype, what)


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("lens", [[1, 1, 2, 40], [3000, 1, 500, 33]])
def test_infinite_values(ctx, dtype, lens):
    """The weight of a counted token is above 0, so an infinite value is the channel's result, and two opposite ones NaN."""
    H, Hk, D, page = 8, 2, 64, 16
    q, kc, vc, table, n = problem(600 + dtype, dtype, lens, H, Hk, D, page, poison=False)
    at = lambda r, t: (int(table[r, t // page]), slice(None), t % page)  # noqa: E731
    v_max = float(vc.double().abs().max())
    vc[at(0, 0)][:, 3], vc[at(1, 0)][:, 5] = INF, -INF
    vc[at(2, 1)][:, 0], vc[at(3, 17)][:, 9], vc[at(3, 20)][:, 9], vc[at(3, 30)][0, 10] = INF, INF, -INF, -INF
    got, lse = attend(ctx, q, kc, vc, table, n, H, dtype)
    ref = attention_reference(q, kc, vc, table, n, H, scale=D ** -0.5)
    assert torch.isinf(ref[0]).sum() == 8 + 8 + 8 + 4 and torch.isnan(ref[0]).sum() == 8
    check_with_infinities(got, lse, ref, v_max, dtype, "infinite values")


@pytest.mark.parametrize("dtype,far", [(F32, 60), (F16, 12), (F16, 20), (F16, 60), (BF16, 20), (BF16, 60)])
def test_infinite_values_of_small_weight(ctx, dtype, far):
    """An infinite value whose weight is exp(-far) of the largest."""
    D, page = 64, 16
    q, kc, vc, table, n = problem(630, dtype, [100], 1, 1, D, page, poison=False)
    q[0] = 0
    q[0, 0] = 8
    kc[..., 0] = 0
    kc[int(table[0, 2]), 0, 5, 0] = far  # its score: far; all others 0
    v_max = float(vc.double().abs().max())
    vc[int(table[0, 0]), 0, 1, 7] = -INF
    got, lse = attend(ctx, q, kc, vc, table, n, 1, dtype)
    ref = attention_reference(q, kc, vc, table, n, 1, scale=D ** -0.5)
    assert torch.isinf(ref[0]).sum() == 1
    check_with_infinities(got, lse, ref, v_max, dtype, "small weight")


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("cap", [2.0 ** -60, 0.01, 1.0, 50.0, 1e3, 1e5, 1e6, 1e9, 2.0 ** 90])
def test_caps_of_any_size(ctx, dtype, cap):
    """A score far below its cap is itself, whatever the cap: nothing may be off by a share of the cap."""
    D, H = 64, 8
    q, kc, vc, table, n = problem(660 + dtype, dtype, [1, 60, 333, 1500], H, 2, D, 16, poison=False)
    got, lse = attend(ctx, q, kc, vc, table, n, H, dtype, softcap=cap)
    out, want_lse, _ = attention_reference(q, kc, vc, table, n, H, scale=D ** -0.5, softcap=cap)
    tol = attention_reference(q, kc, vc, table, n, H, scale=D ** -0.5)[2]
    # the cap's own steps: at most 16 roundings of the capped score, none of which is above 8 here or above the cap
    tol = tol + 2 * 16 * 2.0 ** -24 * min(cap, 8.0)
    check_attention(got, lse, (out, want_lse, tol), float(vc.double().abs().max()), dtype, f"cap {cap}")


def test_caps_that_are_refused(ctx):
    """Infinite ones, whose scores would be infinity times 0, and those that scores divided or multiplied by leave f32."""
    with Device(ctx) as dev:
        call = lambda cap: ctx.s.op_paged_attention(ctx.handle, _record(dev, softcap=cap))  # noqa: E731
        for cap in (INF, -INF, 3e38, 2.0 ** 101, 2.0 ** -101, 1e-40, -1e-40):
            assert call(cap) == abi.ERR_INVALID_ARGUMENT, cap
        for cap in (0.0, -0.0, 2.0 ** 100, 2.0 ** -100):
            assert call(cap) == abi.OK, cap


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_scores_near_the_lowest(ctx, dtype):
    """Scores of -2.2e38, all there are: weights of 1, not none."""
    D, page = 64, 16
    q, kc, vc, table, n = problem(690 + dtype, dtype, [50, 20], 2, 2, D, page, poison=False)
    q[:], kc[:] = 0, 0
    q[:, 0::D], kc[..., 0] = -2.0 ** 60, 2.0 ** 64
    scale = 2.2e38 / 2.0 ** 124
    got, lse = attend(ctx, q, kc, vc, table, n, 2, dtype, scale=scale)
    got = got.double().view(2, 2, D)
    for r in range(2):
        for h in range(2):
            t = torch.arange(int(n[r]))
            want = vc[table[r, t // page].long(), h, t % page].double().mean(0)
            assert ((got[r, h] - want).abs() <= 2 * ROUND[dtype] * want.abs() + 2.0 ** -14).all()
            assert abs(float(lse[r, h]) + 2.2e38) < 1e32


@pytest.mark.parametrize("page,columns", [(42966, 49981), (8176, 262657)])
def test_length_just_below_31_bits(ctx, page, columns):
    """A request that ends within a tile of 2^31: one page, named by every entry of its row, so that its places count alike.

    Each lane adds up to 2^31 / 2048 / 4 terms (2048 waves, 8 of 32 tokens a lane), 2^18 roundings of 2^-24 of the sum."""
    N, D = page * columns, 8
    assert 2 ** 31 - 32 < N < 2 ** 31
    gen = torch.Generator().manual_seed(1)
    kc, vc = (0.5 * randn(gen, F16, 1, 1, page, D) for _ in range(2))
    vc = vc.abs() + 1
    q = randn(gen, F16, 1, D)
    got, lse = attend(ctx, q, kc, vc, torch.zeros(1, columns, dtype=torch.int32), torch.tensor([N], dtype=torch.int32), 1, F16)
    s = kc[0, 0].double() @ q[0].double() / D ** 0.5
    want = torch.softmax(s, 0) @ vc[0, 0].double()
    assert ((got[0].double() - want).abs() <= (2.0 ** -5 + ROUND[F16]) * want).all()
    assert abs(float(lse) - float(torch.logsumexp(s, 0) + torch.log(torch.tensor(float(columns), dtype=torch.float64)))) <= 2.0 ** -5


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
def test_nan_and_lowest_scores(ctx, dtype):
    """NaN in a key that counts makes its heads NaN and no other; a key of score -infinity has no weight."""
    q, kc, vc, table, n = problem(720 + dtype, dtype, [50, 700], 4, 2, 64, 16, poison=False)
    kc[int(table[0, 1]), 0, 3] = -INF * torch.sign(q[0, :64])  # head 0 of request 0; head 1 has infinities of both signs: NaN
    kc[int(table[1, 2]), 1, 5, 0] = float("nan")
    got, lse = attend(ctx, q, kc, vc, table, n, 4, dtype)
    got = got.double().view(2, 4, 64)
    assert torch.isnan(got[1, 2:]).all() and torch.isnan(lse[1, 2:]).all()
    kc[int(table[1, 2]), 1, 5, 0] = 0
    kc[int(table[0, 1]), 0, 3] = 0
    out, _, tol = attention_reference(q, kc, vc, table, n, 4, scale=0.125)
    keep = torch.tensor([[False, False, True, True], [True, True, False, False]])
    bound = (tol + {F32: 0, F16: 2.0 ** -21, BF16: 2.0 ** -16}[dtype])[..., None] * float(vc.double().abs().max()) + ROUND[dtype] * out.abs() + 2.0 ** -25
    assert ((got - out).abs() <= bound)[keep].all()
    t = torch.tensor([t for t in range(50) if t != 19])
    k, v = (c[table[0, t // 16].long(), 0, t % 16].double() for c in (kc, vc))
    want = torch.softmax(k @ q[0, :64].double() / 8, 0) @ v
    assert ((got[0, 0] - want).abs() <= bound[0, 0] + ROUND[dtype] * want.abs()).all()
