"""Log probabilities, entropy and top alternatives against their definitions in
64 bits (prompt_util.py has the tolerances)."""
import math

import pytest
import torch

from mlx_amd import abi
from prompt_util import logprobs_reference, run_logprobs
from serving_util import BF16, F16, F32, TORCH

pytestmark = pytest.mark.gpu


def check(ctx, dtype, logits, top, what, scale=1.0, **kw):
    T, V = logits.shape
    tokens = torch.randint(0, V, (T,), generator=torch.Generator().manual_seed(T + V), dtype=torch.int32)
    got = run_logprobs(ctx, dtype, logits, tokens, top, scale=scale, **kw)
    want, tol = logprobs_reference(logits, tokens, top, scale)
    assert torch.equal(got["top_ids"], want["top_ids"]), f"{what}: other alternatives in rows {(got['top_ids'] != want['top_ids']).any(-1).nonzero().view(-1).tolist()[:5]}"
    for k in ("lse", "logprobs", "entropy", "top_logprobs"):
        g, w = got[k].double(), want[k]
        low = torch.isneginf(w)
        assert torch.equal(torch.isneginf(g), low), f"{what}: {k}"
        off = torch.where(low, 0.0, (g - torch.where(low, 0.0, w)).abs())
        bound = tol[k] + 2.0 ** -24 * torch.where(low, 0.0, w.abs())
        assert (off <= bound).all(), f"{what}: {k} off by {float(off.max()):.3g}, {float((off / bound).max()):.3g} of the bound"


def rows(seed, dtype, T, V, spread=3.0):
    return (torch.randn(T, V, generator=torch.Generator().manual_seed(seed)) * spread).to(TORCH[dtype])


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("T,V,top", [(1, 1, 1), (1, 1, 0), (3, 2, 2), (5, 64, 64), (2, 65, 64), (7, 511, 20), (4, 513, 64), (3, 2000, 64), (2, 4095, 5),
                                     (2, 4097, 8), (9, 8191, 20), (3, 8192, 64), (2, 50021, 20), (1, 131072, 64), (5, 100003, 1), (600, 777, 8),
                                     (520, 9001, 20)])
def test_sizes(ctx, dtype, T, V, top):
    """One logit to many; rows that are cut into parts and rows that are not."""
    check(ctx, dtype, rows(T + V, dtype, T, V), top, f"{T} {V} {top}")


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("scale", [0.01, 0.7, 5.0])
def test_scale(ctx, dtype, scale):
    check(ctx, dtype, rows(1, dtype, 6, 20000), 10, f"scale {scale}", scale=scale)


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("offset,pad", [(0, 1), (1, 0), (3, 5), (8, 8)])
def test_strides(ctx, dtype, offset, pad):
    check(ctx, dtype, rows(2, dtype, 5, 9999), 10, "strides", offset=offset, pad=pad)
    check(ctx, dtype, rows(2, dtype, 700, 601), 10, "strides", offset=offset, pad=pad)


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("T", [2, 600])
def test_ties(ctx, dtype, T):
    """Equal logits: the lowest places first, whether they fit the ranked ones or not."""
    V = 20000
    flat = torch.zeros(T, V, dtype=TORCH[dtype])
    check(ctx, dtype, flat, 20, "all equal")
    few = torch.randint(0, 5, (T, V), generator=torch.Generator().manual_seed(3)).to(TORCH[dtype])
    check(ctx, dtype, few, 64, "five values")
    zeros = flat.clone()
    zeros[:, 1::2] = -0.0
    check(ctx, dtype, zeros, 9, "0 and -0")
    two = flat.clone()
    two[:, [7, 19999, 12345]] = 4.0
    check(ctx, dtype, two, 5, "three above")


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("T", [1, 3, 560])
def test_masked_rows(ctx, dtype, T):
    """-infinity and the type's lowest value in masked places: all but none, a few, fewer than the alternatives asked for."""
    V = 30000
    x = rows(4, dtype, T, V)
    for mask in (-math.inf, torch.finfo(TORCH[dtype]).min if dtype == F16 else -1e30):
        y = x.clone()
        y[:, 100:] = mask
        check(ctx, dtype, y, 20, f"{mask} behind 100")
        y[:, 3:] = mask
        check(ctx, dtype, y, 20, f"{mask} behind 3")
        y = x.clone()
        y[:, ::2] = mask
        check(ctx, dtype, y, 20, f"{mask} every other")
    check(ctx, dtype, torch.full_like(x, -math.inf), 6, "nothing left")


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("T", [1, 530])
def test_shapes_of_rows(ctx, dtype, T):
    """Rising, falling, one far above, all the large ones in one thread's places."""
    V = 40000
    line = torch.arange(V) / 2000.0
    check(ctx, dtype, line.to(TORCH[dtype]).expand(T, V).contiguous(), 30, "rising")
    check(ctx, dtype, (-line).to(TORCH[dtype]).expand(T, V).contiguous(), 30, "falling")
    x = rows(5, dtype, T, V)
    x[:, 17] = 1000.0
    check(ctx, dtype, x, 10, "one above")
    x = rows(6, dtype, T, V)
    for i in range(8):
        x[:, 4096 * i:4096 * i + 8] = 50.0 + torch.arange(8)
    check(ctx, dtype, x, 40, "in one thread")


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("T", [1, 530])
def test_rows_that_are_not_finite(ctx, dtype, T):
    V = 20000
    x = rows(7, dtype, T, V)
    x[:, 5000] = math.inf
    tokens = torch.zeros(T, dtype=torch.int32)
    got = run_logprobs(ctx, dtype, x, tokens, 4)
    assert (got["lse"] == math.inf).all() and torch.isneginf(got["logprobs"]).all() and torch.isnan(got["entropy"]).all()
    assert (got["top_ids"][:, 0] == 5000).all() and torch.isnan(got["top_logprobs"][:, 0]).all() and torch.isneginf(got["top_logprobs"][:, 1:]).all()
    assert torch.equal(got["top_ids"][:, 1:], torch.argsort(rows(7, dtype, T, V).double().index_fill_(1, torch.tensor([5000]), -math.inf), dim=-1,
                                                            descending=True, stable=True)[:, :3].to(torch.int32))
    x[:, 9000], x[:, 400] = math.nan, math.nan
    got = run_logprobs(ctx, dtype, x, tokens, 4)
    assert all(torch.isnan(got[k]).all() for k in ("lse", "logprobs", "entropy", "top_logprobs"))
    assert (got["top_ids"][:, :3] == torch.tensor([400, 9000, 5000], dtype=torch.int32)).all()


@pytest.mark.parametrize("T", [2, 600])
def test_tokens_outside(ctx, T):
    x = rows(8, F32, T, 9000)
    tokens = torch.tensor([-1, 9000])[torch.arange(T) % 2].to(torch.int32)
    got = run_logprobs(ctx, F32, x, tokens, 3)
    assert torch.isneginf(got["logprobs"]).all() and torch.isfinite(got["lse"]).all()


@pytest.mark.parametrize("T", [2, 600])
def test_outputs_that_are_not_wanted(ctx, T):
    x = rows(9, BF16, T, 9000)
    tokens = torch.zeros(T, dtype=torch.int32)
    full = run_logprobs(ctx, BF16, x, tokens, 3)
    for left in (["logprobs", "tokens"], ["entropy"], ["lse"], ["top_ids"], ["top_logprobs"], ["top_ids", "top_logprobs", "lse", "entropy"],
                 ["logprobs", "entropy", "lse", "top_ids", "top_logprobs"]):
        got = run_logprobs(ctx, BF16, x, tokens, 3, **{k: None for k in left})
        for k, v in got.items():
            if k in left:
                assert (v == 9).all(), (left, k)
            else:
                assert torch.equal(v, full[k]), (left, k)


REFUSED = [(abi.ERR_INVALID_ARGUMENT, o) for o in (
    dict(struct_size=3), dict(rows=-1), dict(vocab=0), dict(top=-1), dict(vocab=2), dict(scale=0.0), dict(scale=-1.0), dict(scale=math.inf),
    dict(scale=math.nan), dict(logits=None), dict(tokens=None), dict(row_stride=50), dict(logits_offset=-1), dict(rows=5), dict(vocab=101))] + [
    (abi.ERR_NOT_SUPPORTED, o) for o in (dict(dtype=4), dict(top=65), dict(vocab=(1 << 24) + 1))]


@pytest.mark.parametrize("code,over", REFUSED)
def test_refusals(ctx, code, over):
    over = dict(over)
    if over.get("vocab", 0) > 1000:
        over["row_stride"] = 0
    run_logprobs(ctx, F32, rows(10, F32, 4, 100), torch.zeros(4, dtype=torch.int32), 3, expect=code, **over)


def test_no_rows(ctx):
    run_logprobs(ctx, F32, rows(10, F32, 4, 100), torch.zeros(4, dtype=torch.int32), 3, expect=0, rows=0)
