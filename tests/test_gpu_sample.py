"""sample_token against the definition in 64 bits, one row at a time.

Tokens have to be equal. The kernel's weights are off by 2^-34 relative each, the
reference's by 2^-53, so a running sum of n tokens is off by some sqrt(n) 2^-34 of a
weight where the next border is a whole weight away: a draw falls between with a
probability of about 1e-8, less than 1e-4 over all rows here, and the inputs are
fixed by their seeds.
"""
import pytest
import torch

from hackthenorth_amd.kernels.greedy import argmax
from hackthenorth_amd.kernels.sample import sample_token

pytestmark = pytest.mark.gpu
INF, NAN = float("inf"), float("nan")


def reference(logits, u, temperature, top_k, top_p, min_p):
    """One row (any type, on the CPU) by the definition."""
    x = logits.double()
    x = torch.where(x.isnan(), -INF, x)
    order = torch.argsort(x, descending=True, stable=True)
    order = order[x[order] > -INF]
    if not len(order):
        return -1
    if not temperature > 0:
        return int(order[0])
    x = x[order]
    weight = torch.where(x == x[0], 1.0, torch.exp((x - x[0]) / temperature))
    if top_k > 0:
        weight = weight[:top_k]
    before = weight.cumsum(0) - weight
    if top_p < 1:
        weight = weight[:max(1, int((before < top_p * weight.sum()).sum()))]
    weight = weight[:max(1, int((weight >= min_p).sum()))]
    total = weight.cumsum(0)
    return int(order[min(int((total <= u * total[-1]).sum()), len(total) - 1)])


def check(logits, uniform, temperature=1.0, top_k=0, top_p=1.0, min_p=0.0):
    def row(value, r):
        return value[r].item() if isinstance(value, torch.Tensor) else value

    def cuda(value):
        return value.cuda() if isinstance(value, torch.Tensor) else value
    settings = (temperature, top_k, top_p, min_p)
    got = sample_token(logits.cuda(), uniform.cuda(), *map(cuda, settings)).cpu()
    single = torch.tensor(1.0, dtype=torch.float32)
    want = [reference(logits[r], uniform[r].item(),
                      *(row(v if isinstance(v, torch.Tensor) or i == 1 else float(single * v), r)
                        for i, v in enumerate(settings)))
            for r in range(logits.shape[0])]
    assert got.tolist() == want


def normal(seed, *shape, std=1.0):
    return std * torch.randn(*shape, generator=torch.Generator().manual_seed(seed))


def uniforms(seed, rows):
    return torch.rand(rows, generator=torch.Generator().manual_seed(1000 + seed))


SETTINGS = [dict(), dict(temperature=0.0), dict(temperature=0.7, top_k=50), dict(top_p=0.9),
            dict(min_p=0.05), dict(temperature=1.3, top_k=1000, top_p=0.95, min_p=0.01),
            dict(top_k=1), dict(top_p=1e-6), dict(temperature=0.05, top_p=0.99),
            dict(temperature=30.0, top_p=0.5), dict(min_p=1.0), dict(top_k=10 ** 9)]


@pytest.mark.parametrize("settings", SETTINGS)
@pytest.mark.parametrize("kind", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("rows,vocab,std", [(1, 151936, 2.0), (3, 50257, 5.0), (40, 1000, 1.0),
                                            (9, 97, 3.0), (5, 1, 1.0), (7, 2, 1.0), (2, 151936, 0.01),
                                            (2, 32001, 0.0), (600, 63, 1.0)])
def test_matches_the_definition(rows, vocab, std, kind, settings):
    logits = normal(rows, rows, vocab, std=std).to(kind)
    check(logits, uniforms(vocab, rows), **settings)


@pytest.mark.parametrize("kind", [torch.bfloat16, torch.float32])
def test_settings_per_row(kind):
    rows = 64
    g = torch.Generator().manual_seed(3)

    def pick(values, dtype):
        return torch.tensor(values, dtype=dtype)[torch.randint(len(values), (rows,), generator=g)]
    check(normal(8, rows, 20011, std=3.0).to(kind), uniforms(8, rows),
          pick((0.0, -1.0, 0.3, 1.0, 2.0), torch.float32), pick((0, -5, 1, 40, 5000), torch.int64),
          pick((1.0, 2.0, 0.0, 0.5, 0.95), torch.float32), pick((0.0, 0.1, 0.5, 3.0), torch.float32))


@pytest.mark.parametrize("vocab", [2, 700, 1024, 5000, 151936])
@pytest.mark.parametrize("top_p", [1.0, 0.5, 0.3])
def test_equal_logits_take_the_lowest_ids(vocab, top_p):
    """All the same: the order is the ids', and the place in it exact."""
    u = torch.tensor([0.0, 0.25, 0.5, 0.75, 1 - 2.0 ** -24, 0.123456])
    for kind in (torch.bfloat16, torch.float32):
        check(torch.full((6, vocab), -3.25, dtype=kind), u, top_p=top_p)
        check(torch.full((6, vocab), 7.0, dtype=kind), u, top_k=max(1, vocab // 3), top_p=top_p)


def test_many_tokens_on_few_values():
    """Thousands of tokens on each of a few logits, around the borders of the counts."""
    g = torch.Generator().manual_seed(1)
    logits = torch.randint(3, (12, 60000), generator=g).to(torch.float32) * 0.004
    for k in (0, 1, 1023, 1024, 1025, 20000, 45000):
        check(logits, uniforms(k, 12), top_k=k)
        check(logits.to(torch.bfloat16), uniforms(k + 1, 12), top_k=k, top_p=0.7)


@pytest.mark.parametrize("kind", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("std", [0.1, 0.3, 0.6, 1.2])
@pytest.mark.parametrize("rows,vocab", [(2, 151936), (5, 40000), (60, 20000)])
def test_flat_rows_with_thousands_of_tokens_in_a_bin(rows, vocab, std, kind):
    """A bin, 1/32 nat, of 500 to 19000 tokens: lists in the block, in memory, and rows
    that are read again."""
    logits = normal(vocab + rows, rows, vocab, std=std).to(kind)
    for i, settings in enumerate((dict(), dict(top_p=0.6), dict(temperature=1.5, top_k=vocab // 3, top_p=0.9),
                                  dict(temperature=0.8, min_p=0.4))):
        check(logits, uniforms(rows + i, rows), **settings)


@pytest.mark.parametrize("vocab,tie", [(151936, 2500), (151936, 1030), (20000, 19000), (40000, 1025)])
def test_thousands_of_equal_logits_inside_a_row(vocab, tie):
    """As coarse logits have them: `tie` tokens on one value, in the lists or past them."""
    g = torch.Generator().manual_seed(tie)
    logits = torch.randn(4, vocab, generator=g) * 2 + 20
    for r in range(4):
        logits[r, torch.randperm(vocab, generator=g)[:tie]] = 20.125 + r
    for settings in (dict(), dict(temperature=2.0), dict(top_p=0.5), dict(top_k=tie // 2, temperature=30.0)):
        check(logits, uniforms(tie, 4), **settings)
        check(logits.to(torch.bfloat16), uniforms(vocab, 4), **settings)


def test_masked_and_infinite_logits():
    logits = normal(4, 10, 3000, std=2.0)
    logits[0] = -INF
    logits[1] = NAN
    logits[2, ::2] = -INF
    logits[3, 1::2] = NAN
    logits[4, [7, 2999, 100]] = INF
    logits[5, :2999] = -INF
    logits[6, 17:] = torch.finfo(torch.float32).min
    logits[7] = torch.finfo(torch.float32).max
    logits[8, ::3], logits[8, 1::3], logits[8, 2::3] = -INF, NAN, 0.0
    logits[9, 0], logits[9, 1:] = 0.0, -0.0
    for kind in (torch.float32, torch.bfloat16):
        for seed in range(4):
            check(logits.to(kind), uniforms(seed, 10), **SETTINGS[seed])


def test_extreme_temperatures_and_uniforms():
    logits = normal(5, 8, 5000, std=4.0)
    u = torch.tensor([0.0, 1e-38, 0.5, 1 - 2.0 ** -24, 1.0, 2.0, -1.0, NAN])
    for t in (1e-30, 1e-3, 1e6, 3e38):
        got = sample_token(logits.cuda(), u.cuda(), t).cpu()
        clean = u.nan_to_num(0.0).clamp(0.0, 1 - 2.0 ** -24)
        assert got.tolist() == [reference(logits[r], clean[r].item(), float(torch.tensor(t)), 0, 1.0, 0.0)
                                for r in range(8)]


@pytest.mark.parametrize("kind", [torch.bfloat16, torch.float32])
def test_greedy_is_argmax(kind):
    logits = normal(6, 33, 4099).to(kind)
    got = sample_token(logits.cuda(), uniforms(6, 33).cuda(), 0.0)
    want = argmax(logits.cuda()) if kind is torch.bfloat16 else logits.argmax(1).cuda()
    assert torch.equal(got, want)


def test_strided_rows_shapes_and_out():
    wide = normal(7, 4, 6, 1031)
    for kind in (torch.bfloat16, torch.float32):
        logits = wide.to(kind).cuda()
        u = uniforms(7, 24).view(4, 6).cuda()
        want = sample_token(logits[..., 3:1003].contiguous(), u, 0.8, 40)
        assert want.shape == (4, 6)
        out = torch.empty(4, 6, dtype=torch.int64, device="cuda")
        assert sample_token(logits[..., 3:1003], u, 0.8, 40, out=out) is out
        assert torch.equal(out, want)
        assert torch.equal(sample_token(logits[1, 2, 3:1003], u[1, 2:3].clone(), 0.8, 40), want[1, 2])
        by_columns = logits[0, :, 3:1003].t().contiguous().t()
        assert torch.equal(sample_token(by_columns, u[0].contiguous(), 0.8, 40), want[0])


def test_batch_does_not_change_a_row():
    logits, u = normal(9, 300, 30000, std=3.0).cuda(), uniforms(9, 300).cuda()
    whole = sample_token(logits, u, 0.9, 0, 0.95)
    for r in (0, 17, 299):
        assert int(sample_token(logits[r:r + 1], u[r:r + 1], 0.9, 0, 0.95)) == int(whole[r])


def test_frequencies_follow_the_weights():
    """An even grid of uniforms meets each token as often as it weighs, to one."""
    logits = normal(10, 1, 50, std=1.5)
    n = 4096
    u = (torch.arange(n) + 0.5) / n
    got = sample_token(logits.expand(n, 50).cuda(), u.float().cuda(), 0.7).cpu()
    want = torch.softmax(logits[0].double() / float(torch.tensor(0.7)), 0) * n
    assert bool(((torch.bincount(got, minlength=50) - want).abs() <= 1 + 1e-3).all())


def test_captured_and_replayed():
    logits, u = normal(11, 5, 9000, std=2.0).cuda(), uniforms(11, 5).cuda()
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        sample_token(logits, u, 0.8, 100, 0.9)
    torch.cuda.current_stream().wait_stream(stream)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=stream):
        out = sample_token(logits, u, 0.8, 100, 0.9)
    for turn in range(4):
        logits.copy_(normal(20 + turn, 5, 9000, std=2.0))
        u.copy_(uniforms(20 + turn, 5))
        want = sample_token(logits, u, 0.8, 100, 0.9)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, want)
