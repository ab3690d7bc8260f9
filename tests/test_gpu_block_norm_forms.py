"""The block norm's forms for many rows: the threads and vectors of a row that
each length takes, with 16-bit and f32 values, row lengths off a multiple of 8, and the
stores past the caches that outputs of 32 MB and more take, in place too."""
import pytest
import torch

from serving_util import BF16, F16, F32, norm_reference, randn
from test_gpu_block_norm import CHANNEL, FULL, NONE, ROW, check, compare, run

pytestmark = pytest.mark.gpu

# a row length for each form, the second one ragged
LENGTHS = [(512, 397), (1024, 1001), (2048, 1999), (3000, 2901), (4096, 3601), (6144, 5003), (8192, 6997), (12288, 9001), (16384, 12289)]


@pytest.mark.parametrize("lengths", LENGTHS)
@pytest.mark.parametrize("xd,rd", [(F32, F32), (F16, F16), (BF16, F32)])
def test_many_rows(ctx, lengths, xd, rd):
    check(ctx, 513, lengths[0], xd, rd, gate_mode=CHANNEL, bias=True, seed=20)
    check(ctx, 515, lengths[1], xd, rd, post=2, pre=2, gate_mode=ROW, rscale=0.5, seed=21)


@pytest.mark.parametrize("D", [512, 1024, 2048, 3000, 4096, 5003, 8192, 12000, 16384])
@pytest.mark.parametrize("xd", [F32, BF16])
def test_one_output_of_many_rows(ctx, D, xd):
    """Half the outputs: the longest rows stay below the size of the stores past the caches."""
    gen = torch.Generator().manual_seed(D)
    x, r, w = randn(gen, xd, 513, D), randn(gen, xd, 513, D), randn(gen, xd, D)
    _, o = run(ctx, x, r, 1, 1, NONE, None, 1.0, 1e-5, None, None, w, None, xd, xd, xd, want=(False, True))
    _, ro, _, off = norm_reference(x, r, 1, 1, None, 1.0, 1e-5, None, None, w, None)
    compare(o, ro, off, xd, "out")


@pytest.mark.parametrize("lengths", LENGTHS)
@pytest.mark.parametrize("xd,rd", [(F32, F32), (F16, F16), (BF16, BF16)])
def test_outputs_past_the_caches(ctx, lengths, xd, rd):
    for D, in_place in zip(lengths, (False, True)):
        size = 8 if xd == F32 else 4
        T = max(513, -(-(33 << 20) // (D * size)))
        assert T * D * size >= 32 << 20
        check(ctx, T, D, xd, rd, gate_mode=FULL if D > 4096 else NONE, in_place=in_place, seed=22)


def test_rounding_of_large_outputs(ctx):
    """The stores past the caches round as the others do: the same rows in a small call."""
    gen = torch.Generator().manual_seed(5)
    for dt in (F16, BF16):
        x, r = randn(gen, dt, 9000, 1000), randn(gen, dt, 9000, 1000)
        big = run(ctx, x, r, 1, 1, NONE, None, 1.0, 1e-5, None, None, None, None, dt, dt, dt)
        part = run(ctx, x[:600], r[:600], 1, 1, NONE, None, 1.0, 1e-5, None, None, None, None, dt, dt, dt)
        assert all(torch.equal(b[:600].view(torch.int16), p.view(torch.int16)) for b, p in zip(big, part))
