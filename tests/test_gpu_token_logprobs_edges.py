"""Log probabilities of rows at the edges of their definition, cut into parts and
whole (prompt_util.py has the tolerances)."""
import math

import pytest
import torch

from prompt_util import logprobs_reference, run_logprobs
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


@pytest.mark.parametrize("T,V", [(1, 700), (1, 131072), (530, 9000)])
@pytest.mark.parametrize("scale,far", [(1.0, 93032640), (0.7, 132903776), (0.7, 132903768)])
def test_logits_around_the_far_ones(ctx, T, V, scale, far):
    """Rows whose logits lie to both sides of -2^27 / (scale log2 e), where the sums change their reference: 8 is a step of f32.
    Differences to the largest logit are exact, so only the terms of prompt_util.py that do not grow with the logits remain."""
    for above in (8, 16, 32, 4000):
        x = torch.full((T, V), -float(far))
        x[:, V // 3] += above
        x[:, V // 2:V // 2 + 3] += 8
        tokens = torch.tensor([V // 3, 5, V // 2])[torch.arange(T) % 3].to(torch.int32)
        got = run_logprobs(ctx, F32, x, tokens, 5, scale=scale)
        want, _ = logprobs_reference(x, tokens, 5, scale)
        # lse and the logits have few bits left at this size in 64 bits, too: from the differences instead
        y = (x.double() - x.double().amax(-1, keepdim=True)) * float(torch.tensor(scale))
        every = y - torch.logsumexp(y, -1, keepdim=True)
        base = 2.0 ** -24 * (12 + V / 512 + 70 + math.log2(V) * 4)
        for k, w in [("logprobs", every.gather(1, tokens.long()[:, None])[:, 0]), ("top_logprobs", every.gather(1, want["top_ids"].long()))]:
            assert ((got[k].double() - w).abs() <= base + 2.0 ** -23 * w.abs()).all(), (k, above, got[k].flatten()[:5], w.flatten()[:5])
        entropy = -(torch.exp(every) * every).sum(-1)
        assert ((got["entropy"].double() - entropy).abs() <= base * (math.log2(V) + 2) + 2.0 ** -23 * entropy).all(), above
        assert torch.equal(got["top_ids"], want["top_ids"])


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("T", [1, 530])
def test_entropy_of_rows_with_one_far_above(ctx, dtype, T):
    """One logit far above all others, which its thread saw first.  The sum of exps about the largest is 1 and some 10^-5; it is
    rounded at the size of 1, to 2^-24, in up to 8 additions of a vector, 5 of a thread, 6 of a wave, 8 of the block, 6 of the
    parts and twice in its logarithm: 35 times.  The second sum is some 10^-4."""
    for turn in range(1 if T > 1 else 20):
        x = torch.zeros(T, 9000)
        x[:, 4100] = 20.0 + (torch.arange(T) + turn) * (25.0 / (T if T > 1 else 20))
        x = x.to({F32: torch.float32, F16: torch.float16, BF16: torch.bfloat16}[dtype])
        tokens = torch.zeros(T, dtype=torch.int32)
        got = run_logprobs(ctx, dtype, x, tokens, 1)
        want = logprobs_reference(x, tokens, 1, 1.0)[0]["entropy"]
        off = (got["entropy"].double() - want).abs()
        assert (off <= 35 * 2.0 ** -24 + 2.0 ** -20 * want).all(), f"{turn}: off by {float(off.max()):.3g}"


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("T", [1, 530])
def test_entropy_of_a_thread_with_one_far_above(ctx, dtype, T):
    """The same where all other threads have nothing: one addition of all is rounded, at the size of 1, and the logarithm twice."""
    type_, E = {F32: (torch.float32, 4), F16: (torch.float16, 8), BF16: (torch.bfloat16, 8)}[dtype]
    for turn in range(1 if T > 1 else 20):
        x = torch.full((T, 9000), -math.inf)
        x[:, 3 * E:4 * E] = 0.0                 # thread 3's first vector
        x[:, 512 * E + 3 * E + 1] = 25.0 + (torch.arange(T) + turn) * (16.0 / (T if T > 1 else 20))  # in its second
        x = x.to(type_)
        tokens = torch.zeros(T, dtype=torch.int32)
        got = run_logprobs(ctx, dtype, x, tokens, 1)
        want = logprobs_reference(x, tokens, 1, 1.0)[0]["entropy"]
        off = (got["entropy"].double() - want).abs()
        assert (off <= 3 * 2.0 ** -24 + 2.0 ** -20 * want).all(), f"{turn}: off by {float(off.max()):.3g}"


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("T,V", [(1, 700), (1, 20000), (530, 9000)])
def test_scales_that_pass_32_bits_by_log2_e(ctx, dtype, T, V):
    """Logits of 0, and of -infinity, are what they are by any scale: V / 2 equal ones."""
    x = rows(13, dtype, T, V) * 0
    x[:, ::2] = -math.inf
    tokens = (torch.arange(T) % 2).to(torch.int32)
    got = run_logprobs(ctx, dtype, x, tokens, 3, scale=3e38)
    want = math.log(V // 2)
    bound = 2.0 ** -24 * (12 + V / 512 + 70 + math.log2(V) * 4)
    assert ((got["lse"].double() - want).abs() <= bound).all() and ((got["entropy"].double() - want).abs() <= bound * (math.log2(V) + 2)).all()
    assert torch.isneginf(got["logprobs"][::2]).all() and ((got["logprobs"][1::2].double() + want).abs() <= bound).all()
    assert (got["top_ids"] == torch.tensor([1, 3, 5], dtype=torch.int32)).all() and ((got["top_logprobs"].double() + want).abs() <= bound).all()
