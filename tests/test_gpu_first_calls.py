"""The first calls on a new context: its workspace and counters are zero before
them, whatever the memory held."""
import numpy as np
import pytest
import torch

from mlx_amd import runtime
from serving_util import F16
from test_gpu_paged_attention import attend, problem

pytestmark = pytest.mark.gpu


def test_split_work_at_once(ctx, oracle):
    x, w, s, b, _ = oracle.make_problem(64, 3584, 4096, 3, 64, F16, F16, seed=3)
    q, kc, vc, table, n = problem(410, F16, [3000, 70, 900, 1], 8, 2, 128, 16, poison=False)
    product = lambda c: runtime.run_quantized_matmul(c, x, w, s, b, 64, 3584, 4096, 64, 3, F16, F16, F16)  # noqa: E731
    want, want_out = product(ctx), attend(ctx, q, kc, vc, table, n, 8, F16)
    for i in range(4):
        junk = torch.full((64 << 20,), -1, dtype=torch.int8, device="cuda")  # what a later allocation may find
        torch.cuda.synchronize()
        del junk
        torch.cuda.empty_cache()
        with runtime.Context(0) as c:
            if i % 2:
                assert np.array_equal(product(c), want)
            out = attend(c, q, kc, vc, table, n, 8, F16)
            assert all(torch.equal(a, b) for a, b in zip(out, want_out))
            assert np.array_equal(product(c), want)
