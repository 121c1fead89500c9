"""sample_token on rows with hundreds of thousands of tokens far below the largest.

Two tokens of nearly the same weight, 1 and b, and n tokens whose weights add up to t:
with u between 1 / (1 + b + t) and 1 / (1 + b) the draw is the second token only if the
tail is summed: u (1 + b + t) > 1. b is chosen for u (1 + b + t / 2) = 1, so the draw is
t / 4 from either border, 1e-9 and more of a weight, where the kernel's sums are off by
2^-34 of a weight for each of the two, 2^-34 t for the tail and, rounded once a bin and
chunk, some 2^-44: 1.2e-10 together. The logit of b, 2^-14 T at most, is within 2^-38 T of
b's logarithm in fp32, which moves the draw by 2^-39.
"""
import math

import pytest
import torch

from hackthenorth_amd.kernels.sample import sample_token
from test_gpu_sample import reference

pytestmark = pytest.mark.gpu
VOCAB = 524160  # the most that a row may have


def rows_of(below, temperature, count=8):
    """(logits, uniform) with n tokens `below` temperatures under the first."""
    tail = (VOCAB - 2) * math.exp(-below)
    u = 0.5 + (1 + torch.arange(count).double()) * 2.0 ** -19
    second = torch.log(1 / u - 1 - tail / 2)
    logits = torch.full((count, VOCAB), -below * temperature, dtype=torch.float32)
    logits[:, VOCAB // 3] = 0.0
    logits[:, 5] = (second * temperature).float()
    return logits, u.float()


@pytest.mark.parametrize("temperature", [1.0, 0.5, 4.0])
@pytest.mark.parametrize("below", [29.0, 31.0, 31.9])
def test_a_tail_within_32_temperatures_is_summed(below, temperature):
    logits, u = rows_of(below, temperature)
    got = sample_token(logits.cuda(), u.cuda(), temperature).tolist()
    assert got == [5] * len(got)
    assert got == [reference(logits[r], u[r].item(), temperature, 0, 1.0, 0.0) for r in range(len(got))]
    # As in the definition, the first token without the tail.
    logits[:, 6:VOCAB // 3] = logits[:, VOCAB // 3 + 1:] = logits[:, :5] = -float("inf")
    got = sample_token(logits.cuda(), u.cuda(), temperature).tolist()
    assert got == [VOCAB // 3] * len(got)


@pytest.mark.parametrize("temperature", [1.0, 0.5, 4.0])
@pytest.mark.parametrize("below", [32.1, 33.0])
def test_a_tail_past_32_temperatures_is_not(below, temperature):
    """The draw is the definition's without the tail, which is within its weight of it."""
    logits, u = rows_of(below, temperature)
    got = sample_token(logits.cuda(), u.cuda(), temperature).tolist()
    assert got == [VOCAB // 3] * len(got)


@pytest.mark.parametrize("settings", [dict(), dict(top_p=0.9), dict(top_k=300000), dict(top_p=1 - 2.0 ** -24)])
def test_draws_never_fall_behind_the_tail(settings):
    """Tails from 30 to 34 temperatures under the top, any u: between the definition's
    token and the one without the cut tokens, in the order of the row."""
    g = torch.Generator().manual_seed(3)
    logits = -30 - 4 * torch.rand(6, VOCAB, generator=g)
    at = torch.randint(VOCAB, (6, 9), generator=g)
    logits.scatter_(1, at, -6 * torch.rand(6, 9, generator=g))
    u = torch.tensor([0.0, 0.3, 0.77, 1 - 2.0 ** -10, 1 - 2.0 ** -22, 1 - 2.0 ** -24])
    got = sample_token(logits.cuda(), u.cuda(), **settings).tolist()
    top_k, top_p = settings.get("top_k", 0), settings.get("top_p", 1.0)
    for r in range(6):
        rank = torch.empty(VOCAB, dtype=torch.int64)
        rank[torch.argsort(logits[r], descending=True, stable=True)] = torch.arange(VOCAB)
        cut = torch.where(logits[r] > logits[r].max() - 32, logits[r], -float("inf"))
        low, high = (reference(x, u[r].item(), 1.0, top_k, top_p, 0.0) for x in (cut, logits[r]))
        assert rank[low] <= rank[got[r]] <= rank[high]
