"""Serving operators over a paged K/V cache, and token sampling, as cases to time and compare.

A case is one call of one operator:

  append     norm_rope_paged: QK norm and rotation of the new tokens of a ragged
             batch, their keys and values written into cache pages.
  attention  paged_attention: those tokens against the pages, causal by position,
             over the whole context or a sliding window with a few first tokens.
  prefix     shared_prefix_attention: a batch whose sequences begin with the same
             long prefix.
  sample     sample_token: temperature, top-k, top-p, min-p and one uniform number
             per row.

Head counts and vocabulary are those of hackthenorth_amd.model.SHAPES; contexts,
batches, prompts and draft widths those of the benchmark and the tests. Sequences
of one batch differ in length, as a server's do.

Values: queries and keys as QK norm leaves them (near unit variance, queries with
a gain of 2, so that a row attends to some slots more than to others), values
N(0, 1); logits a broad normal with a few dozen tokens far above it, as a trained
head gives. Pages lie in the pool in random order, and slots that no token has
reached hold what earlier requests left there.
"""
import math
from types import SimpleNamespace

import torch

own = False

DEVICE = "cuda"
D = 128
EPS = 1e-6
THETA = 1e6
VOCAB = 151936
#: (query heads, K/V heads)
HEADS = {"tiny": (4, 2), "qwen3-0.6b": (16, 8), "qwen3-4b": (32, 8), "qwen3-8b": (32, 8)}


def listed():
    return [
        # One decode step's new tokens of a server's batch: what a launch costs.
        _case("append_8b_16", "append", "qwen3-8b", 16, 2048),
        # Prompt chunks of several requests, fp32 rotation tables.
        _case("append_4b_prompts", "append", "qwen3-4b", 7, 900, chunk=601, chunks=7, page=64,
              tables="fp32"),
        # One short sequence of a small model: the smallest attention call.
        _case("attn_0.6b_1", "attention", "qwen3-0.6b", 1, 540),
        # Batched decode at ordinary lengths.
        _case("attn_8b_16", "attention", "qwen3-8b", 16, 2048),
        # Few sequences at long contexts: the split over the slots.
        _case("attn_4b_long", "attention", "qwen3-4b", 3, 30011, page=64),
        # Many sequences behind a window of 1024 slots and four first tokens.
        _case("attn_4b_window", "attention", "qwen3-4b", 32, 8200, window=1024, sinks=4),
        # A prompt's chunk beside the single tokens of running requests.
        _case("attn_8b_mixed", "attention", "qwen3-8b", 16, 4096, chunk=1000, chunks=1),
        # A long prompt as one call: the matrix cores' case.
        _case("attn_4b_prompt", "attention", "qwen3-4b", 1, 5000, chunk=5000, chunks=1, page=128),
        # 32 requests behind one long system prompt.
        _case("prefix_8b_32", "prefix", "qwen3-8b", 32, 512, prefix=8200),
        # Verify rows of eight requests behind a shared document.
        _case("prefix_4b_verify", "prefix", "qwen3-4b", 8, 201, chunk=5, chunks=8, prefix=2048,
              page=64),
        # The token of one request.
        {"name": "sample_1", "kind": "sample", "rows": 1, "vocab": VOCAB, "type": "bf16"},
        # The tokens of a large batch, every request with settings of its own.
        {"name": "sample_64", "kind": "sample", "rows": 64, "vocab": VOCAB, "type": "fp32"},
    ]


def _case(name, kind, shape, seqs, context, chunk=1, chunks=0, prefix=0, window=0, sinks=0,
          page=16, tables="bf16"):
    """`seqs` sequences of up to `context` slots after the prefix; the first
    `chunks` of them bring up to `chunk` new tokens, the others one each."""
    return {"name": name, "kind": kind, "shape": shape, "seqs": seqs, "context": context,
            "chunk": chunk, "chunks": chunks, "prefix": prefix, "window": window,
            "sinks": sinks, "page": page, "tables": tables}


def _log(rng, low, high):
    return min(high, max(low, round(math.exp(rng.uniform(math.log(low), math.log(high))))))


def draw(rng):
    kind = rng.choice(("append", "attention", "attention", "attention", "prefix", "prefix",
                       "sample"))
    if kind == "sample":
        return {"kind": kind, "rows": _log(rng, 1, 64),
                "vocab": rng.choice((_log(rng, 64, VOCAB), VOCAB - rng.randrange(300))),
                "type": rng.choice(("bf16", "fp32"))}
    case = _case("", kind, rng.choice(tuple(HEADS)), 1, 1, page=rng.choice((16, 32, 64, 128, 256)),
                 tables=rng.choice(("bf16", "fp32")))
    del case["name"]
    if kind == "append":
        case.update(seqs=_log(rng, 1, 64), context=_log(rng, 1, 4000))
        if rng.random() < 0.5:
            case.update(chunk=_log(rng, 2, 500), chunks=min(case["seqs"], _log(rng, 1, 8)))
    elif kind == "prefix":
        case.update(seqs=_log(rng, 2, 48), context=_log(rng, 1, 600), prefix=_log(rng, 64, 8200))
        if rng.random() < 0.4:
            case.update(chunk=rng.randrange(2, 9), chunks=case["seqs"])
    else:
        case.update(seqs=_log(rng, 1, 48))
        if rng.random() < 0.4:  # prompts, alone or beside single tokens
            case.update(seqs=min(case["seqs"], 12), chunk=_log(rng, 2, 1500),
                        chunks=min(case["seqs"], rng.randrange(1, 4)), context=_log(rng, 1, 3500))
        else:
            case.update(context=_log(rng, 1, 60000 // case["seqs"]))
        if rng.random() < 0.4:
            case.update(window=_log(rng, 1, 2000), sinks=rng.choice((0, 1, 4, 67)))
    return case


def _batch(case):
    """(new tokens, length) of every sequence: up to three fifths below the
    case's sizes, spread evenly; the first sequence has them whole."""
    less = [0.6 * (b * 0.618034 % 1.0) for b in range(case["seqs"])]
    new = [max(1, round(case["chunk"] * (1 - f))) if b < case["chunks"] else 1
           for b, f in enumerate(less)]
    lengths = [case["prefix"] + max(n, round(case["context"] * (1 - f)))
               for n, f in zip(new, less)]
    return new, lengths


# ---------------------------------------------------------------- inputs

def prepare(case, seed):
    g = torch.Generator(device=DEVICE).manual_seed(seed)

    def normal(*shape, std=1.0):
        return torch.randn(shape, generator=g, device=DEVICE) * std

    if case["kind"] == "sample":
        return _prepare_sample(case, g, normal)
    heads, kv_heads = HEADS[case["shape"]]
    new, lengths = _batch(case)
    page, prefix, total = case["page"], case["prefix"], sum(new)
    counts = [-(-n // page) for n in lengths]
    shared = prefix // page  # whole pages of the prefix, the same ones for every sequence
    owned = sum(counts) - shared * (len(counts) - 1)
    ids = torch.randperm(owned + 3, generator=g, device=DEVICE).to(torch.int32)
    table = torch.full((len(new), max(counts)), -1, dtype=torch.int32, device=DEVICE)
    at = shared
    for b, count in enumerate(counts):
        table[b, :shared] = ids[:shared]
        table[b, shared:count] = ids[at:at + count - shared]
        at += count - shared
    state = SimpleNamespace(
        kind=case["kind"], page=page, heads=heads, kv_heads=kv_heads, max_new=max(new),
        max_length=max(lengths), window=case["window"], sinks=case["sinks"], table=table,
        lengths=torch.tensor(lengths, device=DEVICE),
        starts=torch.tensor([0] + new, device=DEVICE).cumsum(0),
        keys=normal(owned + 3, kv_heads, page, D).to(torch.bfloat16),
        values=normal(owned + 3, kv_heads, page, D).to(torch.bfloat16))
    if case["kind"] == "append":
        packed = normal(total, (heads + 2 * kv_heads) * D).to(torch.bfloat16)
        q, k, v = packed.split((heads * D, kv_heads * D, kv_heads * D), 1)
        state.q, state.k, state.v = (t.view(total, -1, D) for t in (q, k, v))
        state.q_norm = SimpleNamespace(weight=(1 + normal(D, std=0.2)).to(torch.bfloat16),
                                       variance_epsilon=EPS)
        state.k_norm = SimpleNamespace(weight=(1 + normal(D, std=0.2)).to(torch.bfloat16),
                                       variance_epsilon=EPS)
        slots = torch.arange(max(lengths), device=DEVICE, dtype=torch.float64)
        angles = slots[:, None] / THETA ** (torch.arange(D, device=DEVICE) % (D // 2) * 2 / D)
        kind = torch.bfloat16 if case["tables"] == "bf16" else torch.float32
        state.cos, state.sin = angles.cos().to(kind), angles.sin().to(kind)
    else:
        state.q = normal(total, heads, D, std=2.0).to(torch.bfloat16)
    if case["kind"] == "prefix":
        # The prefix's last page may hold the first sequence's own slots too.
        state.prefix_pages = table[0, :-(-prefix // page)].contiguous()
        state.prefix_length = torch.tensor([prefix], device=DEVICE)
    return state


def _prepare_sample(case, g, normal):
    rows, vocab = case["rows"], case["vocab"]

    def uniform(*shape):
        return torch.rand(shape, generator=g, device=DEVICE)

    logits = normal(rows, vocab, std=2.0)
    picked = torch.randint(vocab, (rows, 40), generator=g, device=DEVICE)
    logits.scatter_add_(1, picked, 14.0 * uniform(rows, 40))
    kind = torch.bfloat16 if case["type"] == "bf16" else torch.float32

    def mixed(values, kind):  # one of the values for each row
        at = torch.randint(len(values), (rows,), generator=g, device=DEVICE)
        return torch.tensor(values, device=DEVICE, dtype=kind)[at]

    # Settings that requests bring: plain sampling, nucleus, top-k, min-p, and
    # the greedy choice.
    return SimpleNamespace(
        kind="sample", logits=logits.to(kind), uniform=uniform(rows),
        temperature=mixed((0.0, 0.6, 0.7, 0.8, 1.0, 1.3), torch.float32),
        top_k=mixed((0, 0, 20, 50, 1000), torch.int64),
        top_p=mixed((1.0, 0.95, 0.9, 0.8), torch.float32),
        min_p=mixed((0.0, 0.0, 0.05, 0.1), torch.float32))


# ---------------------------------------------------------------- one pass

def run(state):
    if own:
        return _run_own(state)
    if state.kind == "sample":
        return _sample(state)
    if state.kind == "append":
        return _append(state)
    return _attention(state)


def _run_own(s):
    if s.kind == "sample":
        from hackthenorth_amd.kernels.sample import sample_token
        return sample_token(s.logits, s.uniform, temperature=s.temperature, top_k=s.top_k,
                            top_p=s.top_p, min_p=s.min_p)
    from hackthenorth_amd.kernels import paged
    if s.kind == "append":
        q = paged.norm_rope_paged(s.q, s.k, s.v, s.q_norm, s.k_norm, s.cos, s.sin, s.keys,
                                  s.values, s.table, s.starts, s.lengths)
        return q, s.keys, s.values
    if s.kind == "prefix":
        return paged.shared_prefix_attention(s.q, s.keys, s.values, s.prefix_pages,
                                             s.prefix_length, s.table, s.starts, s.lengths)
    return paged.paged_attention(s.q, s.keys, s.values, s.table, s.starts, s.lengths,
                                 window=s.window, sinks=s.sinks)


def _rows(s):
    """(sequence, position) of every new token."""
    token = torch.arange(s.q.shape[0], device=s.q.device)
    b = torch.searchsorted(s.starts[1:], token, right=True)
    return b, s.lengths[b] - s.starts[b + 1] + token


def _rotated(x, norm, cos, sin):
    x = x.float()
    x = x * torch.rsqrt((x * x).mean(-1, keepdim=True) + norm.variance_epsilon)
    x = x * norm.weight.float()
    half = torch.cat((-x[..., D // 2:], x[..., :D // 2]), -1)
    return (x * cos[:, None].float() + half * sin[:, None].float()).to(torch.bfloat16)


def _append(s):
    b, position = _rows(s)
    cos, sin = s.cos[position], s.sin[position]
    page, slot = s.table[b, position // s.page].long(), position % s.page
    s.keys[page, :, slot] = _rotated(s.k, s.k_norm, cos, sin)
    s.values[page, :, slot] = s.v
    return _rotated(s.q, s.q_norm, cos, sin), s.keys, s.values


def _attention(s):
    """All sequences at once, padded to the longest. Where a prefix is shared its
    pages are gathered for each sequence: the table holds them."""
    groups, seqs = s.heads // s.kv_heads, s.table.shape[0]
    new = torch.arange(s.max_new, device=s.q.device)
    counts = s.starts[1:] - s.starts[:-1]
    token = (s.starts[:-1, None] + new).clamp(max=s.q.shape[0] - 1)
    q = s.q[token].float().view(seqs, s.max_new, s.kv_heads, groups, D)
    q = q.permute(0, 2, 1, 3, 4).reshape(seqs, s.kv_heads, s.max_new * groups, D)
    pages = s.table.long().clamp(min=0)

    def slots(pool):  # [sequence, K/V head, slot, dim]
        return pool[pages].float().transpose(1, 2).reshape(seqs, s.kv_heads, -1, D)
    scores = torch.matmul(q, slots(s.keys).transpose(2, 3)) / math.sqrt(D)
    position = ((s.lengths - counts)[:, None] + new)[:, :, None]
    slot = torch.arange(scores.shape[-1], device=s.q.device)
    seen = slot <= position
    if s.window:
        seen &= (slot > position - s.window) | (slot < s.sinks)
    seen = seen.repeat_interleave(groups, 1)[:, None]
    scores = scores.masked_fill(~seen, -math.inf)
    weights = torch.exp(scores - scores.amax(-1, keepdim=True))
    weights = weights / weights.sum(-1, keepdim=True)
    values = slots(s.values).masked_fill((slot >= s.lengths[:, None])[:, None, :, None], 0.0)
    out = torch.matmul(weights, values).view(seqs, s.kv_heads, s.max_new, groups, D)
    out = out.permute(0, 2, 1, 3, 4).reshape(seqs, s.max_new, s.heads, D)
    return out[new < counts[:, None]].to(torch.bfloat16)


def _sample(s):
    """The tokens in order of falling logit, the lowest id first among equals;
    every truncation keeps a leading part of that order."""
    vocab = s.logits.shape[1]
    logits, ids = torch.sort(s.logits, dim=1, descending=True, stable=True)
    logits = logits.double()
    greedy = s.temperature <= 0
    heat = torch.where(greedy, 1.0, s.temperature.double())[:, None]
    mass = torch.exp((logits - logits[:, :1]) / heat)
    rank = torch.arange(vocab, device=logits.device)
    first = torch.where(s.top_k > 0, s.top_k, vocab)
    mass = mass * (rank < torch.where(greedy, 1, first)[:, None])
    before = mass.cumsum(1) - mass
    mass = mass * (before < s.top_p.double()[:, None] * mass.sum(1, keepdim=True))
    mass = mass * (mass >= s.min_p.double()[:, None])  # the largest mass is 1
    reached = mass.cumsum(1)
    target = s.uniform.double()[:, None] * reached[:, -1:]
    at = (reached <= target).sum(1, keepdim=True).clamp(max=vocab - 1)
    return ids.gather(1, at)[:, 0]


# ---------------------------------------------------------------- costs

def work(case):
    if case["kind"] == "sample":
        size = 2 if case["type"] == "bf16" else 4
        # A difference, a scaling, an exponential and two sums for each logit.
        return {"bytes": case["rows"] * (case["vocab"] * size + 4 * 5 + 8 + 8),
                "flops": 5 * case["rows"] * case["vocab"]}
    heads, kv_heads = HEADS[case["shape"]]
    new, lengths = _batch(case)
    rows = sum(new)
    if case["kind"] == "append":
        size = 2 if case["tables"] == "bf16" else 4
        data = rows * D * (2 * (2 * heads + 4 * kv_heads) + 2 * size)
        return {"bytes": data, "flops": rows * D * (heads + kv_heads) * 8}
    window, sinks, prefix = case["window"], case["sinks"], case["prefix"]

    def seen(position):
        if not window:
            return position + 1
        start = max(0, position + 1 - window)
        return position + 1 - start + min(start, sinks)
    # Slots that some row of the sequence sees, and the pairs of a row and a slot.
    touched = [length - prefix if not window else
               min(length, seen(length - n) + n - 1) for n, length in zip(new, lengths)]
    pairs = sum(seen(length - 1 - i) for n, length in zip(new, lengths) for i in range(n))
    return {"bytes": 2 * D * (2 * kv_heads * (sum(touched) + prefix) + 2 * rows * heads),
            "flops": 4 * D * heads * pairs}


# ---------------------------------------------------------------- 64 bits

def exact(case, seed):
    """The definitions, one sequence or row after the other, in 64 bits."""
    s = prepare(case, seed)

    def sample(i):
        x = s.logits[i].double()
        order = torch.argsort(x, descending=True, stable=True)
        if s.temperature[i] <= 0:
            return order[0]
        if s.top_k[i] > 0:
            order = order[:int(s.top_k[i])]
        p = torch.softmax(x[order] / s.temperature[i].double(), 0)
        kept = int((p.cumsum(0) - p < s.top_p[i].double()).sum())
        p = p[:kept]
        p = p[p >= s.min_p[i].double() * p[0]]
        share = p.cumsum(0) / p.sum()
        return order[min(int((share <= s.uniform[i].double()).sum()), p.numel() - 1)]

    if s.kind == "sample":
        return torch.stack([sample(i) for i in range(s.logits.shape[0])])

    def slots(pool, b, length):  # [K/V head, slot, dim] of a sequence
        count = -(-length // s.page)
        held = pool[s.table[b, :count].long()].double()
        return held.permute(1, 0, 2, 3).reshape(s.kv_heads, -1, D)[:, :length]

    def turned(x, norm, positions):
        x = x.double()
        x = x / (x.square().mean(-1, keepdim=True) + norm.variance_epsilon).sqrt()
        x = x * norm.weight.double()
        cos = s.cos[positions].double()[:, None, :D // 2]
        sin = s.sin[positions].double()[:, None, :D // 2]
        a, b = x[..., :D // 2], x[..., D // 2:]
        return torch.cat((a * cos - b * sin, b * cos + a * sin), -1)

    if s.kind == "append":
        queries, keys, values = [], s.keys.double(), s.values.double()
    out = []
    for b in range(s.lengths.numel()):
        start, end, length = int(s.starts[b]), int(s.starts[b + 1]), int(s.lengths[b])
        positions = torch.arange(length - (end - start), length, device=DEVICE)
        if s.kind == "append":
            where = s.table[b].long()[positions // s.page]
            keys[where, :, positions % s.page] = turned(s.k[start:end], s.k_norm, positions)
            values[where, :, positions % s.page] = s.v[start:end].double()
            queries.append(turned(s.q[start:end], s.q_norm, positions))
            continue
        k, v = slots(s.keys, b, length), slots(s.values, b, length)
        slot = torch.arange(length, device=DEVICE)
        ahead = positions[:, None] - slot
        visible = ahead >= 0
        if s.window:
            visible = visible & ((ahead < s.window) | (slot < s.sinks))
        rows = []
        for h in range(s.heads):
            kv = h * s.kv_heads // s.heads
            scores = s.q[start:end, h].double() @ k[kv].T / math.sqrt(D)
            scores = torch.where(visible, scores, -math.inf)
            rows.append(torch.softmax(scores, -1) @ v[kv])
        out.append(torch.stack(rows, 1))
    if s.kind == "append":
        return torch.cat(queries), keys, values
    return torch.cat(out)
