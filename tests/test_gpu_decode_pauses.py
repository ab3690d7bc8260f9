"""The decoding example where some requests of a step take no token, against 64 bits
(tolerance: test_gpu_decode_step.py)."""
import os
import sys

import numpy as np
import pytest

pytestmark = pytest.mark.gpu

sys.path.insert(0, os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "examples"))


@pytest.mark.parametrize("requests,page,running", [(3, 4, {2: 1, 3: 2, 7: 0, 8: 1}), (5, 1, {0: 2, 1: 0, 5: 4}), (2, 16, {i: 1 for i in range(0, 18, 2)})])
def test_pauses_against_64_bits(ctx, requests, page, running):
    import paged_decode
    error = paged_decode.run(ctx, 18, requests, 512, 8, 2, 64, page, seed=page, running=running)
    assert error <= 12 * 2.0 ** -11, error


def test_a_pause_in_front_of_a_token(ctx):
    """Rows by token and rows by request would not be the same: refused before anything runs."""
    import paged_decode
    block = paged_decode.Block(ctx, 512, 8, 2, 64, 3, 8, 4, 4, seed=9)
    x = np.zeros((3, 512), np.float16)
    try:
        for new in ([0, 1, 1], [1, 0, 1], [2, 1, 1], [1, 1, -1], [1, 1]):
            with pytest.raises(ValueError):
                block.feed(x, new)
        for new in (None, [1, 1, 1], [1, 1, 0], [0, 0, 0]):
            block.feed(x, new)
    finally:
        block.free_all()
