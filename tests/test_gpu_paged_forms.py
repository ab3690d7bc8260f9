"""The paged operators' forms that depend on sizes: attention's padded channels."""
import pytest

from serving_util import BF16, F16, F32
from test_gpu_paged_attention import check

pytestmark = pytest.mark.gpu

LENS = [0, 1, 15, 17, 33, 64, 130, 257]


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("D", [56, 72, 120, 136, 160, 176, 184, 200, 248])
def test_padded_channels(ctx, dtype, D):
    check(ctx, 500 + D + dtype, dtype, LENS, 6, 2, D, 16)
