"""The paged cache's append and attention and the sampling as a server runs them: a
one-layer model over packed rows, prompts in chunks beside single tokens, greedy and
sampled requests in one batch, eager and captured.

Each step's attention is checked against the 64-bit one over the pages as the step
left them (bounds as in test_gpu_paged.py: weights and their sum rounded to bf16, 2^-8
each, and the output), its tokens against the definition on the step's own logits.
"""
import math
from types import SimpleNamespace

import pytest
import torch

from hackthenorth_amd.kernels.embed import embed_gather
from hackthenorth_amd.kernels.paged import (norm_rope_paged, paged_attention,
                                            shared_prefix_attention)
from hackthenorth_amd.kernels.rows import projection_rows, residual_rows
from hackthenorth_amd.kernels.sample import sample_token
from test_gpu_sample import reference as sampled

pytestmark = pytest.mark.gpu
D, HIDDEN, HEADS, KV, VOCAB, PAGE, LIMIT = 128, 512, 8, 2, 4096, 16, 160


class Model:
    def __init__(self):
        g = torch.Generator().manual_seed(5)

        def weight(*shape):
            return (torch.randn(shape, generator=g) / math.sqrt(shape[-1])).to(torch.bfloat16).cuda()
        self.embed = (torch.randn(VOCAB, HIDDEN, generator=g)).to(torch.bfloat16).cuda()
        self.qkv = weight((HEADS + 2 * KV) * D, HIDDEN)
        self.o = weight(HIDDEN, HEADS * D)
        self.head = 3 * weight(VOCAB, HIDDEN)
        self.gain = torch.ones(HIDDEN, dtype=torch.bfloat16, device="cuda")
        self.q_norm, self.k_norm = (
            SimpleNamespace(weight=(1 + 0.1 * torch.randn(D, generator=g)).to(torch.bfloat16).cuda(),
                            variance_epsilon=1e-6) for _ in range(2))
        angle = torch.arange(LIMIT)[:, None] * 1e4 ** (-torch.arange(0, D, 2) / D)
        angle = torch.cat([angle, angle], 1)
        self.cos, self.sin = angle.cos().cuda(), angle.sin().cuda()


class Server:
    """Three requests' pages; the first `shared` slots of all are the same pages."""

    def __init__(self, requests=3, shared=0):
        each = LIMIT // PAGE
        ids = torch.randperm(requests * each, generator=torch.Generator().manual_seed(9))
        table = ids.view(requests, each).to(torch.int32)
        table[:, :shared // PAGE] = table[0, :shared // PAGE]
        self.table = table.cuda()
        self.prefix = self.table[0, :max(1, shared // PAGE)].clone()
        self.prefix_length = torch.tensor([shared], device="cuda")
        self.shared = shared
        pool = (requests * each, KV, PAGE, D)
        self.keys = torch.full(pool, float("nan"), dtype=torch.bfloat16, device="cuda")
        self.values = self.keys.clone()
        self.heat = torch.tensor([0.0, 0.8, 1.2][:requests], device="cuda")
        self.k = torch.tensor([0, 40, 0][:requests], device="cuda")
        self.p = torch.tensor([1.0, 1.0, 0.9][:requests], device="cuda")

    def layer(self, model, ids, starts, lengths):
        """(q, attention, logits) of the packed tokens."""
        x = embed_gather(ids, model.embed)
        rows = projection_rows(x, model.qkv, model.gain).view(len(ids), -1, D)
        q = norm_rope_paged(rows[:, :HEADS], rows[:, HEADS:HEADS + KV], rows[:, HEADS + KV:],
                            model.q_norm, model.k_norm, model.cos, model.sin, self.keys,
                            self.values, self.table, starts, lengths)
        if self.shared:
            a = shared_prefix_attention(q, self.keys, self.values, self.prefix, self.prefix_length,
                                        self.table, starts, lengths)
        else:
            a = paged_attention(q, self.keys, self.values, self.table, starts, lengths)
        x = residual_rows(a.view(len(ids), -1), model.o, x)
        return q, a, projection_rows(x, model.head, model.gain)

    def step(self, model, ids, starts, lengths, uniform):
        q, a, logits = self.layer(model, ids, starts, lengths)
        last = logits[(starts[1:] - 1).clamp(min=0)]
        return q, a, last, sample_token(last, uniform, self.heat, self.k, self.p)

    def check(self, q, a, starts, lengths):
        q, a = q.cpu().double(), a.cpu().double()
        for b, length in enumerate(lengths):
            rows = range(starts[b], starts[b + 1])
            slots = torch.arange(length)
            at = self.table[b].cpu().long()[slots // PAGE], slots % PAGE
            k, v = (pool.cpu()[at[0], :, at[1]].double().repeat_interleave(HEADS // KV, 1)
                    for pool in (self.keys, self.values))
            for i, r in enumerate(rows):
                n = length - len(rows) + i + 1
                p = torch.softmax(torch.einsum("hd,shd->hs", q[r], k[:n]) / math.sqrt(D), -1)
                want = torch.einsum("hs,shd->hd", p, v[:n])
                bound = torch.einsum("hs,shd->hd", p, v[:n].abs())
                assert bool(a[r].isfinite().all())
                assert float(((a[r] - want).abs() - 2.0 ** -8 * (2 * bound + want.abs()) - 1e-6).max()) <= 0


def tokens_of(server, logits, uniform):
    return [sampled(logits[r].cpu(), uniform[r].item(), float(server.heat[r]), int(server.k[r]),
                    float(server.p[r]), 0.0) for r in range(len(logits))]


@pytest.mark.parametrize("shared", [0, 32])
def test_requests_served_together(shared):
    model, server = Model(), Server(shared=shared)
    g = torch.Generator().manual_seed(11)
    lengths = [0, 0, 0]
    if shared:  # the shared prompt, once
        ids = torch.randint(VOCAB, (shared,), generator=g).cuda()
        lone = Server(shared=0)
        lone.keys, lone.values, lone.table = server.keys, server.values, server.table[:1]
        starts, length = torch.tensor([0, shared]).cuda(), torch.tensor([shared]).cuda()
        q, a, _ = lone.layer(model, ids, starts, length)
        lone.check(q, a, [0, shared], [shared])
        lengths = [shared] * 3
    # A prompt beside two others; its second chunk beside single tokens; single tokens
    # over the end of a page.
    for new in ([37, 5, 1], [41, 1, 1], [1, 1, 1], [1, 1, 1], [3, 1, 1]) + ([1, 1, 1],) * 8:
        lengths = [a + b for a, b in zip(lengths, new)]
        starts = [0, new[0], new[0] + new[1], sum(new)]
        ids = torch.randint(VOCAB, (sum(new),), generator=g).cuda()
        uniform = torch.rand(3, generator=g)
        q, a, logits, tokens = server.step(model, ids, torch.tensor(starts).cuda(),
                                           torch.tensor(lengths).cuda(), uniform.cuda())
        server.check(q, a, starts, lengths)
        assert tokens.tolist() == tokens_of(server, logits, uniform)


@pytest.mark.parametrize("shared", [0, 32])
def test_captured_decode_loop_equals_the_eager_one(shared):
    """Tokens feed the next step on the device; 40 steps cross pages."""
    steps, model = 40, Model()
    uniform = torch.rand(steps, 3, generator=torch.Generator().manual_seed(13)).cuda()
    starts = torch.arange(4).cuda()

    def fresh():
        server = Server(shared=shared)
        server.keys.zero_(), server.values.zero_()
        s = SimpleNamespace(server=server, ids=torch.tensor([1, 2, 3]).cuda(), step=torch.zeros(1, dtype=torch.int64).cuda(),
                            lengths=torch.tensor([shared, shared + 13, shared + 70]).cuda())
        return s

    def step(s):
        s.lengths += 1
        u = uniform.index_select(0, s.step).view(3)
        s.ids.copy_(s.server.step(model, s.ids, starts, s.lengths, u)[3])
        s.step += 1

    eager, replayed, want = fresh(), fresh(), []
    for _ in range(steps):
        step(eager)
        want.append(eager.ids.tolist())
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        step(replayed)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    got = [replayed.ids.tolist()]
    with torch.cuda.graph(graph, stream=stream):
        step(replayed)
    for _ in range(steps - 1):
        graph.replay()
        got.append(replayed.ids.tolist())
    assert got == want
    assert torch.equal(eager.server.keys, replayed.server.keys)
    assert torch.equal(eager.server.values, replayed.server.values)


@pytest.mark.parametrize("new,length,shared", [(1, 2000, 0), (3, 300, 0), (40, 1500, 0), (200, 2600, 0),
                                               (1, 1400, 512), (50, 1400, 1040)])
def test_infinite_value_of_a_slot_without_weight(new, length, shared):
    """The first 1024 slots' scores lie some 900 below the others', their weights below
    what 32 bits hold; an infinite V there still reaches the rows, and no other dim."""
    g = torch.Generator().manual_seed(21)
    pages, low = -(-length // PAGE), min(1024, length // 2)
    keys, values = (torch.randn(pages, KV, PAGE, D, generator=g).to(torch.bfloat16) for _ in range(2))
    keys.view(pages, KV, PAGE, D)[:low // PAGE] = -40.0
    q = torch.full((new, HEADS, D), 2.0, dtype=torch.bfloat16).cuda()
    table = torch.arange(pages, dtype=torch.int32)[None].cuda()
    starts, lengths = torch.tensor([0, new]).cuda(), torch.tensor([length]).cuda()
    keys, values = keys.cuda(), values.cuda()

    def run():
        if shared:
            return shared_prefix_attention(q, keys, values, table[0, :shared // PAGE].contiguous(),
                                           torch.tensor([shared]).cuda(), table, starts, lengths)
        return paged_attention(q, keys, values, table, starts, lengths)
    clean = run()
    for slot in (0, 37, low - PAGE - 1):
        kept = values[slot // PAGE, 0, slot % PAGE, 5].clone()
        values[slot // PAGE, 0, slot % PAGE, 5] = float("inf")
        got = run()
        values[slot // PAGE, 0, slot % PAGE, 5] = kept
        assert not bool(got[:, :HEADS // KV, 5].isfinite().any())
        other = [d for d in range(D) if d != 5]
        assert torch.equal(got[..., other], clean[..., other])
        assert torch.equal(got[:, HEADS // KV:], clean[:, HEADS // KV:])


def test_two_streams_at_once():
    """Two servers' steps, each on a stream of its own, as one after the other."""
    model = Model()
    streams, g = [torch.cuda.Stream(), torch.cuda.Stream()], torch.Generator().manual_seed(17)
    ids = [torch.randint(VOCAB, (n,), generator=g).cuda() for n in (300, 222)]
    starts = [torch.tensor(s).cuda() for s in ([0, 100, 150, 300], [0, 1, 111, 222])]
    lengths = [torch.tensor(s).cuda() for s in ([100, 50, 150], [1, 110, 111])]
    uniform = torch.rand(3, generator=g).cuda()
    want = [Server().step(model, ids[i], starts[i], lengths[i], uniform) for i in range(2)]
    servers = [[Server() for _ in range(5)] for _ in range(2)]
    got = [[], []]
    torch.cuda.synchronize()
    for n in range(5):
        for i, stream in enumerate(streams):
            with torch.cuda.stream(stream):
                got[i].append(servers[i][n].step(model, ids[i], starts[i], lengths[i], uniform))
    torch.cuda.synchronize()
    for i in range(2):
        for one in got[i]:
            assert all(torch.equal(x, y) for x, y in zip(one, want[i]))
