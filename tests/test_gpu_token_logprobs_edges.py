"""Log probabilities of rows at the edges of their definition, cut into parts and
whole (prompt_util.py has the tolerances)."""
import math

import pytest
import torch

from prompt_util import run_logprobs
from serving_util import BF16, F16, F32
from test_gpu_token_logprobs import rows

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("T", [1, 530])
@pytest.mark.parametrize("V", [700, 20000])
def test_nan_in_the_first_place(ctx, dtype, T, V):
    x = rows(11, dtype, T, V)
    x[:, 0] = math.nan
    got = run_logprobs(ctx, dtype, x, torch.zeros(T, dtype=torch.int32), 5)
    rest = torch.argsort(x.double().nan_to_num(-math.inf), dim=-1, descending=True, stable=True).to(torch.int32)
    assert (got["top_ids"][:, 0] == 0).all() and torch.equal(got["top_ids"][:, 1:], rest[:, :4])
    x[:, [3, V - 1]] = math.nan
    got = run_logprobs(ctx, dtype, x, torch.zeros(T, dtype=torch.int32), 3)
    assert (got["top_ids"] == torch.tensor([0, 3, V - 1], dtype=torch.int32)).all()
    got = run_logprobs(ctx, dtype, torch.full_like(x, math.nan), torch.zeros(T, dtype=torch.int32), 64)
    assert (got["top_ids"] == torch.arange(64, dtype=torch.int32)).all()


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("T", [2, 600])
@pytest.mark.parametrize("what", [math.nan, math.inf, -math.inf])
def test_tokens_outside_of_rows_that_are_not_finite(ctx, dtype, T, what):
    """-infinity for a token outside the vocabulary, whatever the row holds; NaN for one inside it where NaN is."""
    x = rows(12, dtype, T, 9000)
    x[:, 77] = what
    tokens = torch.tensor([-1, 9000, 5, 77])[torch.arange(T) % 4].to(torch.int32)
    got = run_logprobs(ctx, dtype, x, tokens, 3)["logprobs"]
    inside = (tokens >= 0) & (tokens < 9000)
    assert torch.isneginf(got[~inside]).all()
    if math.isnan(what):
        assert torch.isnan(got[inside]).all()
    elif what > 0:
        assert torch.isneginf(got[tokens == 5]).all() and torch.isnan(got[tokens == 77]).all()
    else:
        assert torch.isfinite(got[tokens == 5]).all() and torch.isneginf(got[tokens == 77]).all()
