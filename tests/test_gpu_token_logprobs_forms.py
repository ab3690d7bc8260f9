"""Log probabilities where rows are cut into parts, and where they are not, with
the largest logits in places that the parts and threads share unevenly
(prompt_util.py has the tolerances)."""
import math

import pytest
import torch

from prompt_util import logprobs_reference, run_logprobs
from serving_util import BF16, F16, F32, TORCH

pytestmark = pytest.mark.gpu


def check(ctx, dtype, logits, tokens, top, what, scale=1.0, **kw):
    logits = logits.to(TORCH[dtype])
    got = run_logprobs(ctx, dtype, logits, tokens, top, scale=scale, **kw)
    want, tol = logprobs_reference(logits, tokens, top, scale)
    for k in ("lse", "logprobs", "entropy", "top_logprobs"):
        d, fin = (got[k].double() - want[k]).abs(), torch.isfinite(want[k])
        bound = tol[k].expand_as(d)
        assert torch.equal(got[k][~fin].double(), want[k][~fin]), (what, k)
        assert (d[fin] <= bound[fin]).all(), f"{what}: {k} off by {float(d[fin].max()):.3g}"
    assert torch.equal(got["top_ids"], want["top_ids"]), (what, (got["top_ids"] != want["top_ids"]).nonzero()[:5])


def tokens_of(T, V, gen):
    return torch.randint(-1, V + 1, (T,), generator=gen).to(torch.int32)


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("T,V,top", [(1, 8191, 64), (1, 8192, 64), (1, 8193, 64), (1, 300001, 64), (2, 131072, 1), (2, 131071, 33), (7, 40000, 64),
                                     (130, 9000, 5), (300, 8200, 40), (1, 4097, 64), (65, 70000, 20)])
def test_parts(ctx, dtype, T, V, top):
    gen = torch.Generator().manual_seed(V + top)
    x = torch.randn(T, V, generator=gen) * 3
    check(ctx, dtype, x, tokens_of(T, V, gen), top, "random")
    check(ctx, dtype, x, tokens_of(T, V, gen), top, "offset", offset=3, pad=5, scale=0.37)


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("T,V", [(1, 200000), (3, 20011), (600, 20011)])
@pytest.mark.parametrize("top", [7, 64])
def test_where_the_largest_lie(ctx, dtype, T, V, top):
    """All in one part, in one thread, in a thread's every vector, spread over all, in the last logits, many alike."""
    gen = torch.Generator().manual_seed(V)
    E = 4 if dtype == F32 else 8
    low = torch.randn(T, V, generator=gen).to(TORCH[dtype]).float()
    far = torch.arange(100.0) / 2 + 10
    for what, at in [("one part", torch.arange(100) * 7), ("one thread", torch.arange(E)), ("one thread's vectors", torch.arange(V // (512 * E)) * 512 * E),
                     ("spread", torch.arange(100) * (V // 100)), ("last", V - 1 - torch.arange(100))]:
        x = low.clone()
        x[:, at[:100]] = far[:len(at[:100])]
        check(ctx, dtype, x, tokens_of(T, V, gen), top, what)
    x = low.clone()
    x[:, ::3] = 9.0  # more equal ones than are ranked
    check(ctx, dtype, x, tokens_of(T, V, gen), top, "equal")
    check(ctx, dtype, torch.zeros(T, V), tokens_of(T, V, gen), top, "all equal")
    x = torch.full((T, V), -math.inf)
    x[:, 5::V // 40] = low[:, 5::V // 40]
    check(ctx, dtype, x, tokens_of(T, V, gen), top, "few that are finite")
    check(ctx, dtype, torch.full((T, V), -math.inf), tokens_of(T, V, gen), top, "none")


def test_rows_and_columns_of_one(ctx):
    for T, V, top in [(1, 1, 1), (1, 2, 2), (3, 1, 0), (5, 64, 64), (1, 65, 64), (2, 511, 3), (2, 4095, 8), (2, 4096, 8)]:
        gen = torch.Generator().manual_seed(V)
        check(ctx, F32, torch.randn(T, V, generator=gen), tokens_of(T, V, gen), top, f"{T} {V} {top}")
