"""Paged K/V cache: append and attention for ragged batches (no reference counterpart;
the reference keeps one contiguous cache per sequence, dryft/engine/decode.py:25-46).

Pools key_pages and value_pages are contiguous bf16 [pages, Hkv, page_size, 128]
(page_size a power of two, 16 to 1024). Slot s of sequence b is row
s % page_size of page page_table[b, s // page_size] (int32 [B, P], on device).

A batch packs its new tokens: sequence b's are rows query_starts[b] ..
query_starts[b + 1] - 1 (int64 [B + 1]), and lengths[b] (int64 [B]) is its length
with them, so its last row sits at position lengths[b] - 1. One token each is
query_starts = arange(B + 1); prompts, chunks of prompts, verify rows and single
tokens may share a batch. Everything is read on the device: captured calls
replay with other lengths, tables and starts.

query_starts must not fall and must lie within [0, T], else the attention writes
nothing. A sequence whose length is negative or past its table's slots sees
nothing and stores nothing. Page ids outside the pool read as zeros and are not
written, and entries of slots that no row sees are never used. Rows of no
sequence (behind the last one in a padded batch) are left as they were.
"""
import contextlib

import torch

from .. import _lib


def _on(device):
    """The device of the tensors as the current one, for the launch."""
    if device.index is None or device.index == torch.cuda.current_device():
        return contextlib.nullcontext()
    return torch.cuda.device(device)


def _check_pools(key_pages, value_pages, kv_heads):
    if key_pages.shape != value_pages.shape or key_pages.dim() != 4 \
            or key_pages.shape[0] < 1 or key_pages.shape[1] != kv_heads \
            or key_pages.shape[3] != _lib.HEAD_DIM or not key_pages.is_contiguous() \
            or not value_pages.is_contiguous() or key_pages.dtype != torch.bfloat16 \
            or value_pages.dtype != torch.bfloat16:
        raise ValueError("page pools must be contiguous bf16 [pages, Hkv, page_size, 128]")
    page = key_pages.shape[2]
    if page < 16 or page > 1024 or page & (page - 1):
        raise ValueError("page_size must be a power of two from 16 to 1024")


def _check_batch(page_table, query_starts, lengths):
    if page_table.dim() != 2 or page_table.dtype != torch.int32 or 0 in page_table.shape \
            or page_table.stride(1) != 1:
        raise ValueError("page_table must be int32 [B, P] with unit column stride")
    batch = page_table.shape[0]
    if query_starts.dtype != torch.int64 or query_starts.shape != (batch + 1,) \
            or not query_starts.is_contiguous():
        raise ValueError("query_starts must be contiguous int64 with one entry per sequence and one more")
    if lengths.dtype != torch.int64 or lengths.shape != (batch,) or not lengths.is_contiguous():
        raise ValueError("lengths must be contiguous int64 with one entry per sequence")


def _check_device(first, *others):
    _lib.require_gpu(first, *others)
    if any(t is not None and t.device != first.device for t in others):
        raise ValueError("all tensors must be on one device")


def _rows(t, name):
    if t.dim() != 3 or t.dtype != torch.bfloat16 or t.shape[2] != _lib.HEAD_DIM \
            or t.stride(2) != 1:
        raise ValueError(f"{name} must be bf16 [T, heads, 128] with unit dim stride")


def norm_rope_paged(q, k, v, q_norm, k_norm, cos, sin, key_pages, value_pages, page_table,
                    query_starts, lengths):
    """QK-norm and RoPE of the new tokens; k and v into their pages. Returns q [T, Hq, 128].

    q, k and v are [T, heads, 128] views with packed heads (slices of the packed
    projection). cos/sin are [positions, 128] tables, bf16 or fp32, whose row p
    turns position p (zeros past the last). q_norm/k_norm are RMSNorms over the
    head; None leaves both unnormalised. Norm and rotation run in fp32 and round
    once, where norm_rope_cache keeps the reference's rounding after every step.
    """
    for t, name in ((q, "q"), (k, "k"), (v, "v")):
        _rows(t, name)
        if t.shape[1] > 1 and t.stride(1) != _lib.HEAD_DIM:
            raise ValueError(f"{name} must have packed heads")
    tokens, heads, _ = q.shape
    if k.shape[0] != tokens or v.shape != k.shape:
        raise ValueError("q, k and v must share the tokens, k and v the heads")
    if 0 in q.shape or 0 in k.shape:
        raise ValueError("q and k need tokens and heads")
    if (q_norm is None) != (k_norm is None):
        raise ValueError("q and k are both normalised or neither")
    gains = (None, None) if q_norm is None else (q_norm.weight, k_norm.weight)
    for g in gains:
        if g is not None and (g.dtype != torch.bfloat16 or g.shape != (_lib.HEAD_DIM,)
                              or not g.is_contiguous()):
            raise ValueError("norm gains must be contiguous bf16 [128]")
    if cos.shape != sin.shape or cos.dim() != 2 or cos.shape[1] != _lib.HEAD_DIM \
            or cos.shape[0] < 1 or cos.dtype != sin.dtype \
            or cos.dtype not in (torch.bfloat16, torch.float32) or cos.stride(1) != 1 \
            or cos.stride() != sin.stride():
        raise ValueError("cos/sin must be matching [positions, 128] tables, bf16 or fp32")
    _check_pools(key_pages, value_pages, k.shape[1])
    _check_batch(page_table, query_starts, lengths)
    _check_device(q, k, v, *gains, cos, sin, key_pages, value_pages, page_table, query_starts,
                  lengths)
    out = torch.empty((tokens, heads, _lib.HEAD_DIM), dtype=q.dtype, device=q.device)
    eps = (0.0, 0.0) if q_norm is None else (float(q_norm.variance_epsilon),
                                             float(k_norm.variance_epsilon))
    with _on(q.device):
        _lib.call("htn_norm_rope_paged", _lib.ptr(q), q.stride(0), _lib.ptr(k), k.stride(0),
                  _lib.ptr(v), v.stride(0), _lib.ptr(gains[0]), _lib.ptr(gains[1]), *eps,
                  _lib.ptr(cos), _lib.ptr(sin), cos.stride(0), cos.shape[0],
                  int(cos.dtype == torch.float32), _lib.ptr(key_pages), _lib.ptr(value_pages),
                  key_pages.shape[0], key_pages.shape[2], _lib.ptr(page_table),
                  page_table.stride(0), page_table.shape[1], _lib.ptr(query_starts),
                  _lib.ptr(lengths), page_table.shape[0], tokens, heads, k.shape[1],
                  _lib.ptr(out), _lib.stream(q.device))
    return out


def _attention_args(q, key_pages, value_pages, page_table, query_starts, lengths, out):
    _rows(q, "q")
    if 0 in q.shape:
        raise ValueError("q needs tokens and heads")
    tokens, heads, _ = q.shape
    if key_pages.dim() != 4 or key_pages.shape[1] < 1 or heads % key_pages.shape[1]:
        raise ValueError("query heads must be a multiple of kv heads")
    _check_pools(key_pages, value_pages, key_pages.shape[1])
    _check_batch(page_table, query_starts, lengths)
    if out is None:
        out = torch.empty((tokens, heads, _lib.HEAD_DIM), dtype=q.dtype, device=q.device)
    elif out.shape != q.shape or out.dtype != q.dtype or out.stride(2) != 1:
        raise ValueError("out must be a bf16 view shaped like q with unit dim stride")
    return out


def _attend(name, q, key_pages, value_pages, prefix, page_table, query_starts, lengths, mask, out):
    tokens, heads, _ = q.shape
    batch, kv_heads = page_table.shape[0], key_pages.shape[1]
    nbytes = _lib.load().htn_paged_attention_scratch_bytes(tokens, batch, heads, kv_heads,
                                                           int(bool(prefix)))
    scratch = torch.empty(max(nbytes, 16), dtype=torch.uint8, device=q.device)
    with _on(q.device):
        _lib.call(name, _lib.ptr(q), q.stride(0), q.stride(1), _lib.ptr(key_pages),
                  _lib.ptr(value_pages), key_pages.shape[0], key_pages.shape[2], *prefix,
                  _lib.ptr(page_table), page_table.stride(0), page_table.shape[1],
                  _lib.ptr(query_starts), _lib.ptr(lengths), *mask, _lib.ptr(out), out.stride(0),
                  out.stride(1), batch, tokens, heads, kv_heads, _lib.ptr(scratch), nbytes,
                  _lib.stream(q.device))
    return out


def paged_attention(q, key_pages, value_pages, page_table, query_starts, lengths, *, window=0,
                    sinks=0, out=None):
    """softmax(q k^T / sqrt(128)) v of every new token over the slots up to its own.

    q is [T, Hq, 128] (any token and head strides that are multiples of 8), the
    new tokens' keys and values already in their pages (norm_rope_paged). With
    `window` a row at position p sees the last `window` slots, p - window + 1 to
    p, and the first `sinks` slots of the sequence, however far back. Rows that
    see nothing get zeros. `out`, when given, is a bf16 view shaped like q.
    """
    if window < 0 or sinks < 0:
        raise ValueError("window and sinks must not be negative")
    if sinks and not window:
        raise ValueError("sinks go with a window")
    out = _attention_args(q, key_pages, value_pages, page_table, query_starts, lengths, out)
    _check_device(q, key_pages, value_pages, page_table, query_starts, lengths, out)
    return _attend("htn_paged_attention", q, key_pages, value_pages, (), page_table, query_starts,
                   lengths, (int(window), int(sinks)), out)


def shared_prefix_attention(q, key_pages, value_pages, prefix_pages, prefix_length, page_table,
                            query_starts, lengths, *, out=None):
    """paged_attention of sequences that begin with the same prefix, whose keys and
    values are read once for all rows.

    Slots below prefix_length (int64 [1], on device) are those of prefix_pages
    (int32 [P], on device) for every sequence; the others go by page_table as
    ever, whose entries of whole pages below the prefix's end are not used.
    lengths counts the prefix. A prefix_length outside the slots of prefix_pages
    is taken as the nearest one within.
    """
    if prefix_pages.dim() != 1 or prefix_pages.dtype != torch.int32 or prefix_pages.numel() < 1 \
            or not prefix_pages.is_contiguous():
        raise ValueError("prefix_pages must be contiguous int32 [P]")
    if prefix_length.dtype != torch.int64 or prefix_length.numel() != 1:
        raise ValueError("prefix_length must be one int64")
    out = _attention_args(q, key_pages, value_pages, page_table, query_starts, lengths, out)
    _check_device(q, key_pages, value_pages, prefix_pages, prefix_length, page_table,
                  query_starts, lengths, out)
    prefix = (_lib.ptr(prefix_pages), prefix_pages.numel(), _lib.ptr(prefix_length))
    return _attend("htn_shared_prefix_attention", q, key_pages, value_pages, prefix, page_table,
                   query_starts, lengths, (), out)
