"""Chunk attention over a paged cache with the tiles of calls with many rows: 256
rows where the requests fill them, 128 where most requests are short
(prompt_util.py has the tolerances)."""
import math

import pytest
import torch

from prompt_util import check_chunk, chunk_reference, run_chunk
from serving_util import BF16, F16, F32
from test_gpu_paged_chunk import check, problem

pytestmark = pytest.mark.gpu

LONG = ([160, 3, 70], [90, 200, 0])                                             # few requests, each with many rows
SHORT = ([130, 1, 0, 40] + [1] * 60, [70, 333, 5, 0] + [i * 7 for i in range(60)])  # many requests of one new token


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("new,held", [LONG, SHORT])
@pytest.mark.parametrize("H,Hk,D,page", [(96, 3, 64, 16), (96, 6, 128, 16), (90, 6, 80, 24), (64, 2, 256, 32), (64, 4, 192, 8), (100, 1, 16, 5), (64, 32, 136, 1)])
def test_ragged_batch(ctx, dtype, new, held, H, Hk, D, page):
    check(ctx, dtype, problem(H + D, dtype, new, held, H, Hk, D, page, rows=3), H, f"{H} {Hk} {D} {page}")


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("new,held", [LONG, SHORT])
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("kw", [dict(window=50), dict(window=1), dict(softcap=20.0, scale=0.3), dict(scale=-0.2), dict(window=130, softcap=3.0)])
def test_masks_and_caps(ctx, dtype, new, held, D, kw):
    check(ctx, dtype, problem(D, dtype, new, held, 64, 4, D, 16), 64, str(kw), **kw)


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("new,held", [LONG, SHORT])
@pytest.mark.parametrize("D", [64, 128])
def test_pages_that_are_none(ctx, dtype, new, held, D):
    args = problem(5, dtype, new, held, 64, 4, D, 16)
    table = args[3]
    table[0, 2], table[0, 5], table[0, 9] = -1, args[1].shape[0], -5
    table[1, 0] = 1 << 30
    table[3 if len(new) > 3 else 2, :] = -1
    check(ctx, dtype, args, 64, "holes")
    check(ctx, dtype, args, 64, "holes and window", window=20)


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("new,held", [LONG, SHORT])
@pytest.mark.parametrize("D", [128, 192])
def test_infinite_values(ctx, dtype, new, held, D):
    """Infinite values and NaN of a request's own tokens, for the rows that see them alone."""
    args = problem(9, dtype, new, held, 64, 4, D, 16)
    vc, table = args[2], args[3]
    for t, h, d, x in [(held[0] + 20, 0, 3, math.inf), (held[0] + 41, 1, D - 4, -math.inf), (held[0] + 50, 1, D - 4, math.inf), (held[0] + 90, 3, 9, math.nan)]:
        vc[int(table[0, t // 16]), h, t % 16, d] = x
    check(ctx, dtype, args, 64, "infinite")


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("new,held", [([300], [2500]), ([700], [0]), ([130, 140], [1000, 3000])])
def test_long(ctx, dtype, new, held):
    """Ranges of tokens cut between blocks, and rows of the table looked up more than once."""
    check(ctx, dtype, problem(6, dtype, new, held, 48, 2, 128, 16), 48, f"{new} {held}")
    check(ctx, dtype, problem(6, dtype, new, held, 48, 2, 64, 64), 48, f"{new} {held}", window=1200)


def test_same_result_each_time(ctx):
    for new, held in (LONG, SHORT):
        args = problem(15, BF16, new, held, 64, 4, 128, 16)
        first = run_chunk(ctx, BF16, *args, 64, scale=0.1)
        for _ in range(5):
            again = run_chunk(ctx, BF16, *args, 64, scale=0.1)
            assert torch.equal(first[0].view(torch.int16), again[0].view(torch.int16)) and torch.equal(first[1], again[1])


def test_rows_of_a_batch_and_alone(ctx):
    """A chunk's rows hardly depend on the batch around it: wide tiles there, narrow ones alone."""
    new, held = [200, 1, 1], [100, 40, 0]
    q, kc, vc, table, starts, seq, lens = problem(16, F16, new, held, 64, 4, 128, 16)
    ref = chunk_reference(q, kc, vc, table, starts, seq, lens, 64, scale=0.1, dtype=F16)
    out, lse = run_chunk(ctx, F16, q, kc, vc, table, starts, seq, lens, 64, scale=0.1)
    check_chunk(out, lse, ref, float(vc.abs().max()), F16, "together")
    for r in range(3):
        a, b = int(starts[r]), int(starts[r + 1])
        out, lse = run_chunk(ctx, F16, q[a:b], kc, vc, table[r:r + 1], starts[r:r + 2] - a, seq[r:r + 1], lens[r:r + 1], 64, scale=0.1)
        check_chunk(out, lse, tuple(x[a:b] for x in ref), float(vc.abs().max()), F16, f"alone {r}")
