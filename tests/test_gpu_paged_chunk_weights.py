"""What chunk attention's weights lose in 16 bits, and its values' places.

The weights of a request that decodes, by itself or beside prompts (up to 16 rows of new
tokens and heads), enter the product with v as two values of the type: the first leaves
u of it (u = eps / 2), the second u of that.  So the bound
of prompt_util.py holds with u^2 in the place of u, and its first term weighs values
of 1 and -1 here, whose sums are often far below 1: there the result's own rounding
hides little."""
import pytest
import torch

from prompt_util import check_chunk, chunk_reference, run_chunk
from serving_util import BF16, F16, F32, ROUND, TORCH, randn
from test_gpu_paged_chunk import problem

pytestmark = pytest.mark.gpu

FEW = ([5, 1, 0, 70, 1, 33], [0, 0, 9, 130, 77, 1], 8, 2)
SHORT = ([130, 1, 0, 40] + [1] * 60, [70, 333, 5, 0] + [i * 7 for i in range(60)], 64, 4)
WIDE = ([300, 1, 2, 1, 150], [20, 500, 90, 3, 0], 64, 4)  # tiles of 256 rows; a decoding request has 16 rows
CASES = [FEW, SHORT, WIDE]


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("new,held,H,Hk", CASES)
@pytest.mark.parametrize("D,page", [(64, 16), (80, 5), (128, 16), (192, 8), (256, 16)])
def test_two_values_of_a_weight(ctx, dtype, new, held, H, Hk, D, page):
    q, kc, vc, table, starts, seq, lens = problem(D, dtype, new, held, H, Hk, D, page)
    q, kc = q / 2, kc / 2
    vc = torch.where(vc < 0, -1.0, 1.0).to(vc.dtype)
    out, lse = run_chunk(ctx, dtype, q, kc, vc, table, starts, seq, lens, H, scale=D ** -0.5)
    want, want_lse, tol, mine = ref = chunk_reference(q, kc, vc, table, starts, seq, lens, H, scale=D ** -0.5, dtype=dtype)
    check_chunk(out, lse, ref, 1.0, dtype, "one value")
    two = torch.zeros(len(out), dtype=torch.bool)
    for r, n in enumerate(new):
        if n * H // Hk <= 16:
            two[int(starts[r]):int(starts[r + 1])] = True
    assert two.any()
    off = (out.double().view(want.shape) - want).abs()[two]
    bound = (tol[two] + ROUND[dtype] ** 2)[..., None] + ROUND[dtype] * want[two].abs() + (2.0 ** -25 if dtype == F16 else 0)
    assert (off <= bound).all(), f"{int((off > bound).sum())} of {off.numel()} values off, worst {float((off / bound).max()):.3g} of the bound"


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("new,held,H,Hk", [*CASES, ([3, 1], [3000, 4500], 4, 2), ([700], [2500], 48, 2)])
@pytest.mark.parametrize("D,page", [(64, 16), (96, 3), (128, 8), (136, 16), (192, 5), (256, 16)])
@pytest.mark.parametrize("window", [0, 75])
def test_every_value_counts_once(ctx, dtype, new, held, H, Hk, D, page, window):
    """Equal scores and values that are small whole numbers by token and channel: weights and sums are exact, and a result
    is off by three roundings in 32 bits and its own."""
    q, kc, vc, table, starts, seq, lens = problem(D, dtype, new, held, H, Hk, D, page)
    q = torch.zeros_like(q)
    t = torch.arange(max(int(n) for n in lens))[:, None]
    for r, n in enumerate(lens):
        n = int(n)
        for h in range(Hk):
            v = ((t[:n] * 7 + t[:n] // 64 + torch.arange(D) * 3 + 5 * h + 11 * r) % 13 - 6).to(TORCH[dtype])
            vc[table[r].long()[t[:n, 0] // page], h, t[:n, 0] % page] = v
    table[0, 1 if table.shape[1] > 1 else 0] = -1
    out, lse = run_chunk(ctx, dtype, q, kc, vc, table, starts, seq, lens, H, scale=1.0, window=window)
    want, want_lse, _, mine = chunk_reference(q, kc, vc, table, starts, seq, lens, H, scale=1.0, window=window, dtype=dtype)
    off = (out.double().view(want.shape) - want).abs()
    bound = (ROUND[dtype] + 3 * 2.0 ** -24) * want.abs() + (2.0 ** -25 if dtype == F16 else 0)
    assert (off <= bound).all(), f"{int((off > bound).sum())} of {off.numel()} values off"
    assert torch.equal(torch.isneginf(lse), torch.isneginf(want_lse.float()))
    some = torch.isfinite(want_lse)
    assert ((lse.double() - want_lse)[some].abs() <= 4 * 2.0 ** -24 * (1 + want_lse[some].abs())).all()


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("H,Hk", [(1, 1), (64, 4)])
@pytest.mark.parametrize("infinite", [False, True])
def test_large_values_of_no_weight(ctx, dtype, H, Hk, infinite):
    """Values of 3e37 whose weights are e^-900, in other parts of the row than those that count, and in rows that are computed
    one by one: the result is that of the tokens that count, 1, with their sums' and its own roundings."""
    q, kc, vc, table, starts, seq, lens = problem(21, dtype, [2], [3000], H, Hk, 64, 16)
    q, kc = torch.zeros_like(q), torch.zeros_like(kc)
    q.view(2, H, 64)[:, :, 0] = 1.0
    line = torch.full((3008,), -1000.0)
    line[:4], line[2992:] = -900.0, 0.0
    value = torch.ones(3008)
    value[:4] = 3e37
    kc[table[0].long(), :, :, 0] = line.view(-1, 1, 16).to(kc.dtype)
    vc[table[0].long()] = value.view(-1, 1, 16, 1).to(vc.dtype)
    if infinite:
        vc[int(table[0, 60]), :, 3, 5] = float("inf")
    out, lse = run_chunk(ctx, dtype, q, kc, vc, table, starts, seq, lens, H, scale=1.0)
    out = out.double().view(2, H, 64)
    if infinite:
        assert (out[:, :, 5] == float("inf")).all()
        out[:, :, 5] = 1.0
    assert ((out - 1).abs() <= ROUND[dtype] + (64 + 16) * 2.0 ** -24).all(), float((out - 1).abs().max())
    assert ((lse.double() - torch.log(torch.tensor([[9.0], [10.0]], dtype=torch.float64))).abs() <= 16 * 2.0 ** -24).all()


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("H,Hk", [(4, 2), (64, 4)])
@pytest.mark.parametrize("scale,softcap", [(3e38, 0.0), (-3e38, 0.0), (1e10, 2.0 ** -100), (-3e38, 2.0 ** -100), (3e38, 30.0)])
def test_factors_that_pass_32_bits(ctx, dtype, H, Hk, scale, softcap):
    """Scores of 0 stay 0 where the factor by log2 e, or by the cap, passes f32: equal weights, exact sums."""
    q, kc, vc, table, starts, seq, lens = problem(22, dtype, [250, 1], [20, 300], H, Hk, 64, 16)
    q, vc = torch.zeros_like(q), (vc * 2).round()
    out, lse = run_chunk(ctx, dtype, q, kc, vc, table, starts, seq, lens, H, scale=scale, softcap=softcap)
    want, want_lse, _, _ = chunk_reference(q, kc, vc, table, starts, seq, lens, H, scale=1.0, dtype=dtype)
    off = (out.double().view(want.shape) - want).abs()
    assert (off <= (ROUND[dtype] + 3 * 2.0 ** -24) * want.abs() + (2.0 ** -25 if dtype == F16 else 0)).all()
    assert ((lse.double() - want_lse).abs() <= 4 * 2.0 ** -24 * (1 + want_lse.abs())).all()
