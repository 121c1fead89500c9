"""Paged append and attention against plain 64-bit implementations.

Bounds. An output is a bf16 value: half a step, 2^-9 relative to the next power
of two below, at most 2^-8 of the value. The append computes in fp32 (errors of a
few 2^-24 beside it), so |got - want| <= 2^-8 |want| + 2^-18 scale, where the
second term covers the fp32 sum's cancellation (two products of up to `scale`).
The attention's weights are rounded to bf16 before they multiply V, at most 2^-8
relative each (half a step of bf16), and so is their sum, so an output is off by
at most 2 * 2^-8 sum_s p_s |v_s| from that, plus 2^-8 |out| for its own rounding;
scores accumulate 128 exact products in fp32 (2^-17 sum|q k| at most, through
exp relative in the weights). Checked per element with sum_s p_s |v_s| from the
64-bit reference.
"""
import math
from types import SimpleNamespace

import pytest
import torch

from hackthenorth_amd.kernels.paged import (norm_rope_paged, paged_attention,
                                            shared_prefix_attention)

pytestmark = pytest.mark.gpu
D = 128


class Batch:
    """A ragged batch over pools whose unused slots and pages hold NaN."""

    def __init__(self, new, lengths, heads, kv_heads, page, seed=0, spare=2, prefix=0,
                 poison=float("nan")):
        g = torch.Generator().manual_seed(seed)
        self.new, self.lens = new, lengths
        self.heads, self.kv_heads, self.page, self.prefix = heads, kv_heads, page, prefix
        counts = [-(-n // page) for n in lengths]
        shared = prefix // page
        total = sum(counts) - shared * (len(counts) - 1) if prefix else sum(counts)
        ids = torch.randperm(total + spare, generator=g)
        table = torch.full((len(new), max(counts + [1]) + 1), -1)
        at = shared
        for b, count in enumerate(counts):
            table[b, :shared] = ids[:shared]
            table[b, shared:count] = ids[at:at + count - shared]
            at += count - shared
        self.table = table.to(torch.int32)
        pool = (total + spare, kv_heads, page, D)
        keys = torch.randn(pool, generator=g)
        values = torch.randn(pool, generator=g)
        used = torch.zeros(pool[0], page, dtype=torch.bool)
        for b, n in enumerate(lengths):
            slots = torch.arange(n)
            used[table[b][slots // page], slots % page] = True
        keys.transpose(1, 2)[~used] = poison
        values.transpose(1, 2)[~used] = poison
        self.keys, self.values = keys.to(torch.bfloat16), values.to(torch.bfloat16)
        self.q = (2 * torch.randn(sum(new), heads, D, generator=g)).to(torch.bfloat16)
        self.starts = torch.tensor([0] + new).cumsum(0)
        self.lengths = torch.tensor(lengths)

    def cuda(self):
        return [t.cuda() for t in (self.q, self.keys, self.values, self.table, self.starts,
                                   self.lengths)]

    def slots(self, pool, b):
        n = self.lens[b]
        s = torch.arange(n)
        return pool[self.table[b].long()[s // self.page], :, s % self.page].double()

    def reference(self, window=0, sinks=0):
        """(out, sum_s p_s |v_s|) in 64 bits."""
        out, bound = [], []
        for b, (n, length) in enumerate(zip(self.new, self.lens)):
            if not n:
                continue
            k, v = self.slots(self.keys, b), self.slots(self.values, b)
            group = self.heads // self.kv_heads
            k, v = (x.repeat_interleave(group, 1) for x in (k, v))
            q = self.q[int(self.starts[b]):int(self.starts[b]) + n].double()
            scores = torch.einsum("ihd,shd->his", q, k) / math.sqrt(D)
            position = length - n + torch.arange(n)[:, None]
            slot = torch.arange(length)
            seen = slot <= position
            if window:
                seen &= (slot > position - window) | (slot < sinks)
            p = torch.softmax(scores.masked_fill(~seen, -math.inf), -1).nan_to_num(0.0)
            out.append(torch.einsum("his,shd->ihd", p, v))
            bound.append(torch.einsum("his,shd->ihd", p, v.abs()))
        return torch.cat(out), torch.cat(bound)

    def check(self, got, window=0, sinks=0):
        want, bound = self.reference(window, sinks)
        got = got.cpu().double()
        assert bool(got.isfinite().all())
        excess = (got - want).abs() - (2 * 2.0 ** -8 * bound + 2.0 ** -8 * want.abs() + 1e-6)
        assert float(excess.max()) <= 0, float(excess.max())


# (new tokens per sequence, lengths, query heads, kv heads, page): single tokens
# from the first slot on, lengths around pages and tiles, sequences without new
# tokens, every group size up to 16 rows and past it, verify rows, prompts whose
# row tiles end inside a token's heads, and mixtures.
CASES = [
    ([1], [1], 4, 2, 16), ([1], [64], 16, 8, 16), ([1], [65], 16, 8, 64),
    ([1, 1, 1], [15, 16, 17], 32, 8, 16), ([1] * 5, [540, 1, 63, 128, 129], 16, 8, 32),
    ([1, 0, 1, 0], [700, 5, 33, 0], 32, 8, 16), ([1] * 3, [2500, 7, 900], 8, 1, 128),
    ([1] * 2, [300, 301], 3, 3, 16), ([1] * 2, [300, 3000], 20, 4, 1024),
    ([1] * 2, [999, 130], 32, 2, 16), ([5] * 3, [500, 5, 77], 32, 8, 16),
    ([4], [1000], 4, 1, 64), ([2, 8, 3], [200, 8, 1500], 16, 8, 16),
    ([130], [130], 4, 2, 16), ([77], [1077], 12, 4, 64), ([33, 1, 200, 1], [33, 800, 900, 4], 32, 8, 16),
    ([1500], [1500], 8, 2, 128), ([43, 90], [43, 300], 15, 5, 32), ([129], [4000], 2, 2, 256),
    ([1] * 300, [1 + 7 * i % 90 for i in range(300)], 4, 2, 16),
    ([1], [20000], 32, 8, 16), ([1], [9000], 2, 1, 16),
]


@pytest.mark.parametrize("new,lengths,heads,kv_heads,page", CASES)
def test_attention_matches_plain(new, lengths, heads, kv_heads, page):
    b = Batch(new, lengths, heads, kv_heads, page)
    b.check(paged_attention(*b.cuda()))


# Windows of one slot, around a page and a tile, past the context; sinks within
# the first tile, past it, and overlapping the window.
@pytest.mark.parametrize("window,sinks", [(1, 0), (1, 1), (16, 4), (64, 0), (63, 67), (100, 4),
                                          (700, 130), (5000, 4), (200, 4000)])
@pytest.mark.parametrize("new,lengths,heads,kv_heads,page",
                         [([1] * 4, [1, 70, 1000, 2777], 32, 8, 16), ([5, 5], [900, 9], 32, 8, 64),
                          ([300, 1, 150], [300, 650, 1400], 16, 8, 16), ([520], [520], 6, 2, 128)])
def test_window_and_sinks_match_plain(new, lengths, heads, kv_heads, page, window, sinks):
    b = Batch(new, lengths, heads, kv_heads, page)
    b.check(paged_attention(*b.cuda(), window=window, sinks=sinks), window, sinks)


@pytest.mark.parametrize("heads,kv_heads", [(32, 8), (2, 2)])
def test_pages_behind_the_window_are_not_used(heads, kv_heads):
    """Pages that no row sees may be gone: given to others (NaN here) or unmapped."""
    b = Batch([1, 40, 1], [2000, 1500, 40], heads, kv_heads, 16)
    window, sinks = 100, 20
    q, keys, values, table, starts, lengths = b.cuda()
    want = paged_attention(q, keys, values, table, starts, lengths, window=window, sinks=sinks)
    b.check(want, window, sinks)
    for s, (n, length) in enumerate(zip(b.new, b.lens)):
        low = length - n - window + 1
        for p in range(-(-sinks // 16), max(0, low) // 16):
            if p % 2:
                keys[table[s, p].long()] = float("nan")
                values[table[s, p].long()] = float("inf")
            else:
                table[s, p] = -1
    got = paged_attention(q, keys, values, table, starts, lengths, window=window, sinks=sinks)
    assert torch.equal(got, want)


@pytest.mark.parametrize("value", [float("inf"), float("-inf"), float("nan")])
@pytest.mark.parametrize("new,lengths,window", [([6], [70], 0), ([200], [230], 0), ([1], [300], 33),
                                                ([90], [400], 33), ([300, 5], [300, 70], 0)])
def test_nonfinite_values_reach_only_rows_that_see_them(new, lengths, window, value):
    """An infinite or NaN K or V in every slot but a few: a row that sees none of them has
    the same output as without, and one that sees an infinite V has it there."""
    b = Batch(new, lengths, 8, 4, 16)
    q, keys, values, table, starts, dev_lengths = b.cuda()
    clean = paged_attention(q, keys, values, table, starts, dev_lengths, window=window)
    position = torch.cat([n - k + torch.arange(k) for k, n in zip(new, lengths)])
    seq = torch.repeat_interleave(torch.arange(len(new)), torch.tensor(new))
    for slot in (0, 15, lengths[0] - new[0], lengths[0] - new[0] // 2, lengths[0] - 1):
        page, row = int(table[0, slot // 16]), slot % 16
        sees = (seq == 0) & (position >= slot) & ((position - slot < window) if window else True)
        for pool in (keys, values):
            kept = pool[page, 1, row, 5].clone()
            pool[page, 1, row, 5] = value
            got = paged_attention(q, keys, values, table, starts, dev_lengths, window=window).cpu()
            pool[page, 1, row, 5] = kept
            assert torch.equal(got[~sees], clean.cpu()[~sees])
            assert torch.equal(got[:, :2], clean.cpu()[:, :2])  # other kv heads
            if pool is values:
                other = [d for d in range(D) if d != 5]
                torch.testing.assert_close(got[..., other], clean.cpu()[..., other], rtol=0, atol=0)
                assert not bool(got[sees][:, 2:4, 5].isfinite().any())


def test_strides_offsets_and_untouched_rows():
    """q and out as slices of wider rows, rows before the first and behind the last sequence
    left as they were, pages and tables at odd places."""
    b = Batch([3, 40], [100, 222], 16, 8, 16, seed=3)
    q, keys, values, table, starts, lengths = b.cuda()
    want = paged_attention(q, keys, values, table, starts, lengths)
    wide = torch.randn(60, 40 * D, device="cuda").to(torch.bfloat16)
    packed = wide[:, 8 * D:].view(60, 32, D)[:, ::2]
    packed[7:50] = q
    before = torch.full((60, 20 * D), 3.0, device="cuda", dtype=torch.bfloat16)
    out = before.clone()[:, D:17 * D].view(60, 16, D)
    bigger = torch.full((4, 77), 12345, device="cuda", dtype=torch.int32)
    bigger[1:3, 5:5 + table.shape[1]] = table
    got = paged_attention(packed, keys, values, bigger[1:3, 5:], starts + 7, lengths, out=out)
    assert got is out and torch.equal(out[7:50], want)
    assert bool((out[:7] == 3).all()) and bool((out[50:] == 3).all())


def test_malformed_batches_write_nothing_or_zeros():
    b = Batch([2, 3], [50, 60], 8, 2, 16)
    q, keys, values, table, starts, lengths = b.cuda()
    want = paged_attention(q, keys, values, table, starts, lengths)
    for bad in ([0, 5, 2], [-1, 2, 5], [0, 2, 6], [5, 2, 0], [0, 2, 1 << 40]):
        out = torch.full_like(q, 7.0)
        paged_attention(q, keys, values, table, torch.tensor(bad, device="cuda"), lengths, out=out)
        assert bool((out == 7).all())
    for bad in (-1, 16 * table.shape[1] + 1, 1 << 40, -(1 << 60)):
        changed = lengths.clone()
        changed[1] = bad
        out = paged_attention(q, keys, values, table, starts, changed)
        assert torch.equal(out[:2], want[:2]) and bool((out[2:] == 0).all())
    # A row before slot 0 sees nothing; the one at slot 0 only itself.
    changed = lengths.clone()
    changed[1] = 1
    out = paged_attention(q, keys, values, table, starts, changed)
    assert torch.equal(out[:2], want[:2]) and bool((out[2:4] == 0).all())
    group = q.shape[1] // keys.shape[1]
    first = values[table[1, 0].long(), :, 0].repeat_interleave(group, 0)
    assert torch.equal(out[4], first)
    # Page ids outside the pool count as zero keys and values.
    for bad in (-1, keys.shape[0], 1 << 30, -(1 << 31)):
        t = table.clone()
        t[0, 1] = bad
        zeroed = (keys.clone(), values.clone())
        for pool in zeroed:
            pool[table[0, 1].long()] = 0
        assert torch.equal(paged_attention(q, keys, values, t, starts, lengths),
                           paged_attention(q, *zeroed, table, starts, lengths))


PREFIX_CASES = [
    ([1] * 4, [300, 301, 290, 333], 16, 8, 16, 256), ([1] * 3, [101, 130, 200], 32, 8, 64, 100),
    ([1] * 20, [600 + 13 * i for i in range(20)], 32, 8, 16, 512), ([5] * 6, [2100] * 6, 32, 8, 64, 2048),
    ([1, 1], [65, 66], 4, 2, 16, 64), ([40, 1, 60], [540, 501, 700], 12, 4, 16, 500),
    ([1, 0, 2], [5000, 4900, 4802], 8, 8, 128, 4800), ([3], [20], 4, 1, 16, 9),
    ([1] * 260, [40 + i % 30 for i in range(260)], 2, 1, 16, 32),
]


@pytest.mark.parametrize("new,lengths,heads,kv_heads,page,prefix", PREFIX_CASES)
def test_shared_prefix_matches_plain(new, lengths, heads, kv_heads, page, prefix):
    b = Batch(new, lengths, heads, kv_heads, page, prefix=prefix)
    count = -(-prefix // page)
    # A last, part page of the prefix is a page of its own, whose tail is unused.
    pages = b.table[0, :count].clone()
    if prefix % page:
        for s in range(1, len(new)):
            for pool in (b.keys, b.values):
                pool[b.table[s, count - 1], :, :prefix % page] = pool[pages[-1], :, :prefix % page]
    q, keys, values, table, starts, dev_lengths = b.cuda()
    args = (q, keys, values, pages.cuda(), torch.tensor([prefix], device="cuda"))
    b.check(shared_prefix_attention(*args, table, starts, dev_lengths))
    unused = table.clone()
    unused[:, :prefix // page] = -1
    got = shared_prefix_attention(*args, unused, starts, dev_lengths)
    b.check(got)
    # Without a prefix: the plain call.
    none = shared_prefix_attention(q, keys, values, pages.cuda(), torch.tensor([-3], device="cuda"),
                                   table, starts, dev_lengths)
    b.check(none)


@pytest.mark.parametrize("seed", range(16))
def test_drawn_batches_match_plain(seed):
    """Batches of 1 to 150 sequences with none, one, a few or many new tokens each, groups
    of 1 to 160 heads, all page sizes, windows and prefixes as they come."""
    g = torch.Generator().manual_seed(100 + seed)

    def draw(options):
        return options[int(torch.randint(len(options), (1,), generator=g))]
    heads, kv_heads = draw([(160, 1), (33, 1), (48, 4), (7, 7), (32, 8), (4, 2), (130, 2)])
    page, count = draw([16, 32, 64, 256, 1024]), draw([1, 2, 5, 64, 65, 150])
    most = 600 if count <= 5 else 60
    new = [draw([0, 1, 1, 1, 3, 9, most // 2, most]) if count <= 5 or draw([0, 1]) else 1
           for _ in range(count)]
    new[draw(range(count))] = 1
    prefix = draw([0, 0, 16, 50, 300])
    lengths = [prefix + n + draw([0, 0, 1, 40, most]) for n in new]
    b = Batch(new, lengths, heads, kv_heads, page, seed=seed, prefix=prefix // page * page)
    args = b.cuda()
    window, sinks = draw([(0, 0), (1, 0), (37, 5), (200, 64)])
    b.check(paged_attention(*args, window=window, sinks=sinks), window, sinks)
    if prefix // page:
        q, keys, values, table, starts, dev_lengths = args
        whole = prefix // page
        b.check(shared_prefix_attention(q, keys, values, table[0, :whole].contiguous(),
                                        torch.tensor([whole * page], device="cuda"), table, starts,
                                        dev_lengths))


def test_two_graphs_replayed_in_turn():
    """Calls of two captured graphs keep workspaces of their own."""
    batches = [Batch([1, 20, 3], [900, 300, 500], 16, 4, 16, seed=1), Batch([60, 1], [700, 2000], 8, 8, 64, seed=2)]
    graphs, outs, wants = [], [], []
    for b in batches:
        args = b.cuda()
        wants.append(paged_attention(*args))
        stream = torch.cuda.Stream()
        stream.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(stream):
            paged_attention(*args)
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=stream):
            outs.append(paged_attention(*args))
        graphs.append((graph, args))
    for _ in range(3):
        for graph, _ in graphs:
            graph.replay()
        torch.cuda.synchronize()
        for out, want in zip(outs, wants):
            assert torch.equal(out, want)
            out.zero_()


def test_prefix_past_a_rows_position_stays_causal():
    """Rows inside the prefix see it only up to themselves."""
    b = Batch([100, 3], [180, 150], 8, 4, 16, prefix=128)
    q, keys, values, table, starts, lengths = b.cuda()
    b.check(shared_prefix_attention(q, keys, values, table[0, :8].contiguous(),
                                    torch.tensor([128], device="cuda"), table, starts, lengths))


def tables(rows, kind, theta=1e6):
    angles = torch.arange(rows).double()[:, None] / theta ** (torch.arange(D) % 64 * 2 / D)
    return angles.cos().to(kind), angles.sin().to(kind)


@pytest.mark.parametrize("kind", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("normed", [True, False])
@pytest.mark.parametrize("new,lengths,heads,kv_heads,page",
                         [([1], [1], 4, 2, 16), ([1] * 16, [100 + 17 * i for i in range(16)], 32, 8, 16),
                          ([33, 1, 0, 70], [33, 65, 9, 200], 15, 5, 64), ([5, 5], [5, 4000], 3, 3, 1024),
                          ([1] * 300, [1 + i for i in range(300)], 2, 1, 16)])
def test_append_matches_plain(new, lengths, heads, kv_heads, page, normed, kind):
    b = Batch(new, lengths, heads, kv_heads, page, poison=1.5)
    g = torch.Generator().manual_seed(5)
    total, width = sum(new) + 3, (heads + 2 * kv_heads) * D
    packed = torch.randn(total, width + 24, generator=g).to(torch.bfloat16)
    q, k, v = (t.view(total, -1, D) for t in
               packed[:, 16:16 + width].split((heads * D, kv_heads * D, kv_heads * D), 1))
    norms = [SimpleNamespace(weight=(1 + 0.3 * torch.randn(D, generator=g)).to(torch.bfloat16),
                             variance_epsilon=1e-6) for _ in range(2)] if normed else [None, None]
    cos, sin = tables(max(lengths), kind)
    packed_cuda = packed.cuda()
    parts = [t.view(total, -1, D) for t in packed_cuda[:, 16:16 + width].split(
        (heads * D, kv_heads * D, kv_heads * D), 1)]
    cuda_norms = [n and SimpleNamespace(weight=n.weight.cuda(), variance_epsilon=1e-6) for n in norms]
    _, keys, values, table, starts, dev_lengths = b.cuda()
    out = norm_rope_paged(*parts, *cuda_norms, cos.cuda(), sin.cuda(), keys, values, table, starts + 2,
                          dev_lengths)
    rows = slice(2, 2 + sum(new))
    position = torch.cat([n - m + torch.arange(m) for m, n in zip(new, lengths)])
    seq = torch.repeat_interleave(torch.arange(len(new)), torch.tensor(new))

    def turned(x, norm):
        x = x.double()
        if norm is not None:
            x = x / (x.square().mean(-1, keepdim=True) + 1e-6).sqrt() * norm.weight.double()
        c, s = cos[position].double()[:, None], sin[position].double()[:, None]
        half = torch.cat((-x[..., 64:], x[..., :64]), -1)
        return x * c + half * s, (x * c).abs() + (half * s).abs()

    def close(got, want):
        value, scale = want
        assert bool(((got.cpu().double() - value).abs() <= 2.0 ** -8 * value.abs() + 2.0 ** -18 * scale).all())
    close(out[rows], turned(q[rows], norms[0]))
    page_of, slot = b.table.long()[seq, position // page].cuda(), (position % page).cuda()
    close(keys[page_of, :, slot], turned(k[rows], norms[1]))
    assert torch.equal(values[page_of, :, slot].cpu(), v[rows])
    # Every other slot as it was.
    for pool, before in ((keys, b.keys), (values, b.values)):
        kept = pool.cpu()
        kept[page_of.cpu(), :, slot.cpu()] = before[page_of.cpu(), :, slot.cpu()]
        assert torch.equal(kept, before)


def test_append_skips_what_has_no_place():
    """Rows of no sequence, lengths past the table or before slot 0, unmapped pages."""
    b = Batch([2, 2, 2], [20, 40, 33], 4, 2, 16, poison=0.0)
    q, keys, values, table, starts, lengths = b.cuda()
    k = torch.ones(6, 2, D, device="cuda", dtype=torch.bfloat16)
    cos, sin = (t.cuda() for t in tables(64, torch.bfloat16))
    table[1, 2] = keys.shape[0] + 5
    lengths[2] = 16 * table.shape[1] + 1
    lengths[0] = 1
    before = keys.clone()
    norm_rope_paged(q, k, k, None, None, cos, sin, keys, values, table, starts, lengths)
    page = int(table[0, 0])
    assert torch.equal(values[page, :, 0], k[1])
    keys[page, :, 0] = before[page, :, 0]
    assert torch.equal(keys, before)


@pytest.mark.parametrize("new", [[1, 1, 1, 1], [1, 37, 1, 5]])
def test_captured_decode_step_replays_with_other_lengths(new):
    """Append, attention and shared-prefix attention in one graph, replayed with other
    lengths and rows, and eager calls on another stream between the replays."""
    b = Batch(new, [300, 310, 290, 305], 8, 4, 16, prefix=256, poison=0.0)
    q, keys, values, table, starts, lengths = b.cuda()
    k = torch.randn(sum(new), 4, D, device="cuda").to(torch.bfloat16)
    cos, sin = (t.cuda() for t in tables(400, torch.bfloat16))
    pages, prefix = table[0, :16].contiguous(), torch.tensor([256], device="cuda")

    def step():
        turned = norm_rope_paged(q, k, k, None, None, cos, sin, keys, values, table, starts, lengths)
        return (turned, paged_attention(turned, keys, values, table, starts, lengths),
                paged_attention(turned, keys, values, table, starts, lengths, window=70, sinks=3),
                shared_prefix_attention(turned, keys, values, pages, prefix, table, starts, lengths))
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        step()
    torch.cuda.current_stream().wait_stream(stream)
    graphs = [torch.cuda.CUDAGraph() for _ in range(2)]
    outs = []
    for graph in graphs:
        with torch.cuda.graph(graph, stream=stream):
            outs.append(step())
    for turn in range(3):
        lengths -= turn
        q.mul_(0.9)
        want = [t.clone() for t in step()]
        for graph in graphs:
            graph.replay()
        with torch.cuda.stream(stream):
            stream.wait_stream(torch.cuda.current_stream())
            paged_attention(q, keys, values, table, starts, lengths)
        torch.cuda.synchronize()
        for out in outs:
            for got, eager in zip(out, want):
                assert torch.equal(got, eager)


@pytest.mark.parametrize("new,length", [(5, 900), (64, 2000), (200, 700)])
def test_rows_do_not_depend_on_other_rows_scores(new, length):
    """Every other token's queries 20 times as large (their maxima move far more often):
    the others' outputs stay the same, bit for bit."""
    b = Batch([new], [length], 4, 4, 16)
    b.q *= 3
    q, *rest = b.cuda()
    want = paged_attention(q, *rest)
    q[1::2] *= 20
    got = paged_attention(q, *rest)
    assert torch.equal(got[::2], want[::2])
    assert not torch.equal(got[1::2], want[1::2])


def test_calls_repeat_bit_for_bit():
    b = Batch([1, 90, 1], [3000, 900, 77], 32, 8, 16)
    args = b.cuda()
    first = paged_attention(*args)
    for _ in range(5):
        assert torch.equal(paged_attention(*args), first)


def test_long_cache_past_32_bit_offsets():
    """Pages past 2^32 bytes into the pool, and a table row far into its tensor."""
    pages = (1 << 32) // (8 * 16 * D * 2) + 40
    keys = torch.zeros(pages, 8, 16, D, device="cuda", dtype=torch.bfloat16)
    values = torch.zeros_like(keys)
    b = Batch([1, 1], [500, 77], 32, 8, 16)
    q, small_k, small_v, table, starts, lengths = b.cuda()
    shift = pages - small_k.shape[0]
    keys[shift:], values[shift:] = small_k, small_v
    moved = torch.where(table >= 0, table + shift, table)
    got = paged_attention(q, keys, values, moved, starts, lengths)
    b.check(got)
    k = torch.ones(2, 8, D, device="cuda", dtype=torch.bfloat16)
    cos, sin = (t.cuda() for t in tables(600, torch.bfloat16))
    norm_rope_paged(q, k, k, None, None, cos, sin, keys, values, moved, starts, lengths)
    assert torch.equal(values[moved[0, 499 // 16].long(), :, 499 % 16], k[0])
