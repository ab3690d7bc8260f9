"""Chunk attention's forms of wide heads: 136 to 256 channels, padded and not, with
caps, windows, and pages that hold no whole runs of tokens, in the tiles of few rows
and of many (prompt_util.py has the tolerances)."""
import math

import pytest

from serving_util import BF16, F16, F32
from test_gpu_paged_chunk import check, problem

pytestmark = pytest.mark.gpu

FEW = ([5, 1, 0, 70, 1, 33], [0, 0, 9, 130, 77, 1], 8, 2)
MANY = ([160, 3, 70], [90, 200, 0], 64, 4)
CAP, WINDOW = dict(softcap=20.0, scale=0.3), dict(window=50)


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("new,held,H,Hk", [FEW, MANY])
@pytest.mark.parametrize("D", [136, 192, 200, 248, 256])
@pytest.mark.parametrize("page,kw", [(16, {}), (16, CAP), (16, WINDOW), (5, {}), (5, CAP), (5, WINDOW), (8, {**CAP, **WINDOW}), (3, {**CAP, **WINDOW})])
def test_caps_windows_and_pages(ctx, dtype, new, held, H, Hk, D, page, kw):
    check(ctx, dtype, problem(D + page, dtype, new, held, H, Hk, D, page, rows=3), H, f"{H} {Hk} {D} {page} {kw}", **kw)


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("new,held,H,Hk", [FEW, MANY])
@pytest.mark.parametrize("D,page,kw", [(64, 5, CAP), (96, 16, CAP), (96, 5, WINDOW), (128, 5, CAP), (128, 16, {**CAP, **WINDOW}), (128, 3, WINDOW)])
def test_other_widths(ctx, dtype, new, held, H, Hk, D, page, kw):
    check(ctx, dtype, problem(D + page, dtype, new, held, H, Hk, D, page), H, f"{H} {Hk} {D} {page} {kw}", **kw)


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("new,held,H,Hk", [FEW, MANY])
@pytest.mark.parametrize("D,page", [(192, 16), (248, 16), (256, 16), (256, 5)])
@pytest.mark.parametrize("kw", [{}, CAP, WINDOW])
def test_holes_and_values_that_are_not_finite(ctx, dtype, new, held, H, Hk, D, page, kw):
    args = problem(D, dtype, new, held, H, Hk, D, page)
    vc, table = args[2], args[3]
    r = 3 if len(new) > 3 else 0
    table[r, 2], table[r, 5], table[r, 9] = -1, args[1].shape[0], -5
    check(ctx, dtype, args, H, "holes", **kw)
    for t, h, d, x in [(held[r] + 20, 0, 3, math.inf), (held[r] + 41, 1, D - 4, -math.inf), (held[r] + 50, 1, D - 4, math.inf), (held[r] + 60, 0, 9, math.nan)]:
        at = int(table[r, t // page])
        if 0 <= at < vc.shape[0]:
            vc[at, h, t % page, d] = x
    check(ctx, dtype, args, H, "infinite", **kw)
