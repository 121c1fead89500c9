"""Single tokens and verify rows keep some 16 bits of a softmax weight.

Bound, relative to sum_s p_s |v_s|, of blocks whose rows number up to 32:
  * a score of 128 products that are exact, added in fp32: 2^-16 sum|q k| / sqrt(128) in
    the exponent, and 2^-20 for the scaling, the difference and exp2; in the weight and
    in their sum, so twice;
  * a weight as two bf16, the upper half off by 2^-8 of it and the lower by 2^-8 of what
    is left: 2^-16;
  * fp32 sums: 2^-23 an addition that changes a sum: two for each slot with a V that is
    not zero, one a 64-slot tile for the weights, and 64 more across lanes, waves, chunks
    and in the rescalings;
and 2^-8 of the output for its own rounding. Weights rounded to one bf16 are off by 2^-9
where they lie in [1/2, 1): the bound tells the two apart where few slots have a V that
is not zero, and where the outputs cancel.
"""
import math

import pytest
import torch

from hackthenorth_amd.kernels.paged import paged_attention, shared_prefix_attention
from test_gpu_paged import D, Batch

# (new, lengths, heads, kv heads, prefix, every how many slots have a V that is not zero)
CASES = [([1] * 4, [2, 5, 9, 33], 32, 8, 0, 1), ([5], [40], 16, 4, 0, 1), ([2], [17], 32, 2, 0, 1),
         ([3, 1], [600, 2500], 16, 8, 0, 97), ([1], [5000], 8, 1, 0, 611), ([1, 2], [700, 612], 8, 4, 512, 67)]


def batch(new, lengths, heads, kv_heads, prefix, every):
    b = Batch(new, lengths, heads, kv_heads, 16, seed=4, prefix=prefix, poison=0.0)
    b.q = b.q / 16
    for i, length in enumerate(lengths):
        slots = torch.arange(length)[torch.arange(length) % every != every // 2]
        b.values[b.table[i].long()[slots // 16], :, slots % 16] = 0.0
    return b


def excess(b, every, got=None):
    """By how much outputs pass the bound: those given, or those of weights of one bf16
    each, which add up to their sum or to that of the unrounded ones."""
    worst = [[], []]
    for i, (n, length) in enumerate(zip(b.new, b.lens)):
        k, v = (b.slots(pool, i).repeat_interleave(b.heads // b.kv_heads, 1) for pool in (b.keys, b.values))
        rows = slice(int(b.starts[i]), int(b.starts[i]) + n)
        q = b.q[rows].double()
        scores = torch.einsum("ihd,shd->his", q, k) / math.sqrt(D)
        sizes = torch.einsum("ihd,shd->his", q.abs(), k.abs()) / math.sqrt(D)
        hidden = torch.arange(length) > length - n + torch.arange(n)[:, None]
        scores, sizes = scores.masked_fill(hidden, -math.inf), sizes.masked_fill(hidden, 0.0)
        weights = torch.exp(scores - scores.amax(-1, keepdim=True))
        total = weights.sum(-1, keepdim=True)

        def out(w, t, v):
            return torch.einsum("his,shd->ihd", w / t, v)
        want = out(weights, total, v)
        share = 2 * (2.0 ** -16 * sizes.amax(-1) + 2.0 ** -20) + 2.0 ** -16 \
            + (2 * -(-length // every) + length / 64 + 64) * 2.0 ** -23
        bound = share.t()[..., None] * out(weights, total, v.abs()) + 2.0 ** -8 * want.abs()
        one = weights.bfloat16().double()
        results = [got[rows].cpu().double()] if got is not None else \
            [out(one, t, v).bfloat16().double() for t in (total, one.sum(-1, keepdim=True))]
        for kept, result in zip(worst, results):
            kept.append(float(((result - want).abs() - bound).max()))
    return [max(kept) for kept in worst if kept]


@pytest.mark.gpu
@pytest.mark.parametrize("new,lengths,heads,kv_heads,prefix,every", CASES)
def test_weights_keep_16_bits(new, lengths, heads, kv_heads, prefix, every):
    b = batch(new, lengths, heads, kv_heads, prefix, every)
    q, keys, values, table, starts, dev_lengths = (t.cuda() for t in (b.q, b.keys, b.values, b.table,
                                                                      b.starts, b.lengths))
    got = paged_attention(q, keys, values, table, starts, dev_lengths)
    assert excess(b, every, got)[0] <= 0
    if prefix:
        got = shared_prefix_attention(q, keys, values, table[0, :prefix // 16].contiguous(),
                                      torch.tensor([prefix], device="cuda"), table, starts, dev_lengths)
        assert excess(b, every, got)[0] <= 0


@pytest.mark.parametrize("new,lengths,heads,kv_heads,prefix,every", CASES)
def test_the_bound_tells_8_bits_apart(new, lengths, heads, kv_heads, prefix, every):
    b = batch(new, lengths, heads, kv_heads, prefix, every)
    assert min(excess(b, every)) > 0
