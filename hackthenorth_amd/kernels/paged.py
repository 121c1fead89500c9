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
sequence (behind the last one in a padded batch) are left as they were in `out`;
without `out` they, and all rows of a batch whose starts are refused, hold
whatever the new tensor's memory held.
"""
import functools

import torch

from .. import _lib

_BF16, _I32, _I64 = torch.bfloat16, torch.int32, torch.int64
_PACKED = torch.contiguous_format
_PAGES = tuple(16 << i for i in range(7))


def _place(first, *others):
    """The index of the GPU that all the tensors are on (None ones aside)."""
    index = first.get_device()
    if index < 0:
        _lib.require_gpu(first)
    for t in others:
        if t is not None and t.get_device() != index:
            _lib.require_gpu(t)
            raise ValueError("all tensors must be on one device")
    return index


def _launch(name, index, *args):
    """The library call on the current stream of GPU `index`, current for the launch."""
    if index == torch.cuda.current_device():
        _lib.call(name, *args, torch._C._cuda_getCurrentRawStream(index))
    else:
        with torch.cuda.device(index):
            _lib.call(name, *args, torch._C._cuda_getCurrentRawStream(index))


def _check_pools(key_pages, value_pages):
    """(pages, kv heads, page size)"""
    shape = key_pages.shape
    if len(shape) != 4 or value_pages.shape != shape or shape[3] != _lib.HEAD_DIM or 0 in shape \
            or key_pages.dtype is not _BF16 or value_pages.dtype is not _BF16 \
            or not key_pages.is_contiguous() or not value_pages.is_contiguous():
        raise ValueError("page pools must be contiguous bf16 [pages, Hkv, page_size, 128]")
    if shape[2] not in _PAGES:
        raise ValueError("page_size must be a power of two from 16 to 1024")
    return shape[:3]


def _check_batch(page_table, query_starts, lengths):
    """(batch, row stride of the table, its pages)"""
    shape, strides = page_table.shape, page_table.stride()
    if len(shape) != 2 or page_table.dtype is not _I32 or 0 in shape or strides[1] != 1:
        raise ValueError("page_table must be int32 [B, P] with unit column stride")
    batch = shape[0]
    if query_starts.dtype is not _I64 or query_starts.shape != (batch + 1,) \
            or not query_starts.is_contiguous():
        raise ValueError("query_starts must be contiguous int64 with one entry per sequence and one more")
    if lengths.dtype is not _I64 or lengths.shape != (batch,) or not lengths.is_contiguous():
        raise ValueError("lengths must be contiguous int64 with one entry per sequence")
    return batch, strides[0], shape[1]


def _rows(t, name):
    """Shape and strides of packed rows."""
    shape, strides = t.shape, t.stride()
    if len(shape) != 3 or t.dtype is not _BF16 or shape[2] != _lib.HEAD_DIM or strides[2] != 1:
        raise ValueError(f"{name} must be bf16 [T, heads, 128] with unit dim stride")
    return shape, strides


@functools.lru_cache(maxsize=256)
def _scratch_bytes(tokens, batch, heads, kv_heads, shared):
    return max(16, _lib.load().htn_paged_attention_scratch_bytes(tokens, batch, heads, kv_heads,
                                                                 shared))


def norm_rope_paged(q, k, v, q_norm, k_norm, cos, sin, key_pages, value_pages, page_table,
                    query_starts, lengths, out=None):
    """QK-norm and RoPE of the new tokens; k and v into their pages. Returns q [T, Hq, 128].

    q, k and v are [T, heads, 128] views with packed heads (slices of the packed
    projection). cos/sin are [positions, 128] tables, bf16 or fp32, whose row p
    turns position p (zeros past the last). q_norm/k_norm are RMSNorms over the
    head; None leaves both unnormalised. Norm and rotation run in fp32 and round
    once, where norm_rope_cache keeps the reference's rounding after every step.
    `out`, when given, receives q: contiguous bf16 [T, Hq, 128], apart from the
    inputs' memory.
    """
    (shape, q_st), (k_shape, k_st), (v_shape, v_st) = _rows(q, "q"), _rows(k, "k"), _rows(v, "v")
    tokens, heads, dim = shape
    kv_heads = k_shape[1]
    for name, count, strides in (("q", heads, q_st), ("k", kv_heads, k_st), ("v", v_shape[1], v_st)):
        if strides[1] != dim and count > 1:
            raise ValueError(f"{name} must have packed heads")
    if k_shape[0] != tokens or v_shape != k_shape:
        raise ValueError("q, k and v must share the tokens, k and v the heads")
    if 0 in shape or kv_heads == 0:
        raise ValueError("q and k need tokens and heads")
    if q_norm is None and k_norm is None:
        q_gain, k_gain, q_eps, k_eps = None, None, 0.0, 0.0
    elif q_norm is None or k_norm is None:
        raise ValueError("q and k are both normalised or neither")
    else:
        q_gain, k_gain = q_norm.weight, k_norm.weight
        q_eps, k_eps = float(q_norm.variance_epsilon), float(k_norm.variance_epsilon)
        for g in (q_gain, k_gain):
            if g.dtype is not _BF16 or g.shape != (dim,) or not g.is_contiguous():
                raise ValueError("norm gains must be contiguous bf16 [128]")
    table_shape, table_st, kind = cos.shape, cos.stride(), cos.dtype
    if len(table_shape) != 2 or sin.shape != table_shape or table_shape[1] != dim \
            or table_shape[0] < 1 or sin.dtype is not kind or kind not in (_BF16, torch.float32) \
            or table_st[1] != 1 or sin.stride() != table_st:
        raise ValueError("cos/sin must be matching [positions, 128] tables, bf16 or fp32")
    pages, pool_heads, page = _check_pools(key_pages, value_pages)
    if pool_heads != kv_heads:
        raise ValueError("page pools must have k's heads")
    batch, row_st, row_pages = _check_batch(page_table, query_starts, lengths)
    if out is not None and (out.shape != shape or out.dtype is not _BF16 or not out.is_contiguous()):
        raise ValueError("out must be contiguous bf16 shaped like q")
    index = _place(q, k, v, q_gain, k_gain, cos, sin, key_pages, value_pages, page_table,
                   query_starts, lengths, out)
    if out is None:
        out = torch.empty_like(q, memory_format=_PACKED)
    _launch("htn_norm_rope_paged", index, q.data_ptr(), q_st[0], k.data_ptr(), k_st[0],
            v.data_ptr(), v_st[0], _lib.ptr(q_gain), _lib.ptr(k_gain), q_eps, k_eps,
            cos.data_ptr(), sin.data_ptr(), table_st[0], table_shape[0], kind is torch.float32,
            key_pages.data_ptr(), value_pages.data_ptr(), pages, page, page_table.data_ptr(),
            row_st, row_pages, query_starts.data_ptr(), lengths.data_ptr(), batch, tokens, heads,
            kv_heads, out.data_ptr())
    return out


def _attend(name, q, key_pages, value_pages, prefix, page_table, query_starts, lengths, mask, out):
    shape, strides = _rows(q, "q")
    if 0 in shape:
        raise ValueError("q needs tokens and heads")
    tokens, heads, _ = shape
    pages, kv_heads, page = _check_pools(key_pages, value_pages)
    if heads % kv_heads:
        raise ValueError("query heads must be a multiple of kv heads")
    batch, row_st, row_pages = _check_batch(page_table, query_starts, lengths)
    if out is not None and (out.shape != shape or out.dtype is not _BF16 or out.stride(2) != 1):
        raise ValueError("out must be a bf16 view shaped like q with unit dim stride")
    index = _place(q, key_pages, value_pages, page_table, query_starts, lengths, out, *prefix)
    if out is None:
        out = torch.empty_like(q, memory_format=_PACKED)
        out_t, out_h = heads * _lib.HEAD_DIM, _lib.HEAD_DIM
    else:
        out_t, out_h, _ = out.stride()
    nbytes = _scratch_bytes(tokens, batch, heads, kv_heads, bool(prefix))
    scratch = torch.empty(nbytes, dtype=torch.uint8, device=q.device)
    before = (prefix[0].data_ptr(), prefix[0].numel(), prefix[1].data_ptr()) if prefix else ()
    _launch(name, index, q.data_ptr(), strides[0], strides[1], key_pages.data_ptr(),
            value_pages.data_ptr(), pages, page, *before, page_table.data_ptr(), row_st, row_pages,
            query_starts.data_ptr(), lengths.data_ptr(), *mask, out.data_ptr(), out_t, out_h,
            batch, tokens, heads, kv_heads, scratch.data_ptr(), nbytes)
    return out


def paged_attention(q, key_pages, value_pages, page_table, query_starts, lengths, *, window=0,
                    sinks=0, out=None):
    """softmax(q k^T / sqrt(128)) v of every new token over the slots up to its own.

    q is [T, Hq, 128] (any token and head strides that are multiples of 8), the
    new tokens' keys and values already in their pages (norm_rope_paged). With
    `window` a row at position p sees the last `window` slots, p - window + 1 to
    p, and the first `sinks` slots of the sequence, however far back. Rows that
    see nothing get zeros; a NaN in a query or in a visible key gives NaN. `out`,
    when given, is a bf16 view shaped like q.
    """
    if window < 0 or sinks < 0:
        raise ValueError("window and sinks must not be negative")
    if sinks and not window:
        raise ValueError("sinks go with a window")
    return _attend("htn_paged_attention", q, key_pages, value_pages, (), page_table, query_starts,
                   lengths, (int(window), int(sinks)), out)


def shared_prefix_attention(q, key_pages, value_pages, prefix_pages, prefix_length, page_table,
                            query_starts, lengths, *, out=None):
    """paged_attention of sequences that begin with the same prefix, whose keys and
    values are read once for all rows.

    For single tokens and a few rows a sequence, which K/V reads bound. Every row's
    two parts, prefix and own, are written and merged, 520 bytes a part and head, so
    prompts are faster by paged_attention (8 chunks of up to 512 tokens behind 2048
    slots, 32 heads: 173 us, here 272).

    The whole pages below prefix_length (int64 [1], on device) are those of
    prefix_pages (int32 [P], on device) for every sequence, and page_table's
    entries of them are not used. The other slots go by page_table as ever, the
    prefix's last ones among them where it ends inside a page: each sequence has
    them in the page that holds its own next ones. lengths counts the prefix. A
    prefix_length outside the slots of prefix_pages is taken as the nearest one
    within.
    """
    if prefix_pages.dim() != 1 or prefix_pages.dtype != torch.int32 or prefix_pages.numel() < 1 \
            or not prefix_pages.is_contiguous():
        raise ValueError("prefix_pages must be contiguous int32 [P]")
    if prefix_length.dtype != torch.int64 or prefix_length.numel() != 1:
        raise ValueError("prefix_length must be one int64")
    return _attend("htn_shared_prefix_attention", q, key_pages, value_pages,
                   (prefix_pages, prefix_length), page_table, query_starts, lengths, (), out)
