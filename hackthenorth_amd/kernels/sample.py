"""Token sampling (no reference counterpart; dryft/engine/kernels/greedy.py:45 selects
greedily).

A row's tokens are taken in order of falling logit, the lowest id first among
equals, with weights exp(logit / temperature). Of them are kept, in turn: the first
top_k; the shortest leading part that holds top_p of the weight so far; those that
weigh at least min_p times the largest. The answer is the first token whose
cumulative weight passes `uniform` times the weight kept. Random numbers come from
the caller, so a draw can be repeated, and weights are summed as 64-bit integers, so
a row's token does not depend on the batch it is drawn in. They are exact to 2^-34 of a
token's weight, but tokens 32 temperatures and more below the largest logit weigh
nothing: all of them together at most vocab e^-32 of the largest weight (7e-9 at 524160,
the most a row may have).
"""
import functools

import torch

from .. import _lib
from .paged import _launch, _place


def _setting(value, name, rows, dtype, low):
    """(tensor or None, scalar) of a setting given for all rows or per row."""
    if isinstance(value, torch.Tensor):
        if value.dtype != dtype or value.shape != (rows,) or not value.is_contiguous():
            raise ValueError(f"{name} must be a number or contiguous {dtype} with one value per row")
        return value, 0
    if not value >= low:  # NaN too
        raise ValueError(f"{name} must be at least {low}")
    return None, value


@functools.lru_cache(maxsize=256)
def _scratch_bytes(rows, vocab):
    return max(16, _lib.load().htn_sample_scratch_bytes(rows, vocab))


def sample_token(logits, uniform, temperature=1.0, top_k=0, top_p=1.0, min_p=0.0, out=None):
    """One token per row of logits [..., V] (bf16 or fp32): int64 [...].

    `uniform` is fp32 in [0, 1), one per row. temperature, top_k, top_p and min_p are
    numbers, or device tensors with one value per row (fp32; top_k int64).
    temperature 0 is the greedy choice; top_k 0, top_p 1 and min_p 0 keep every
    token. Logits of -inf and NaN are masked, tokens of +inf share all the weight;
    a row with nothing left gives -1. `out`, when given, receives the tokens.
    """
    shape = logits.shape
    if len(shape) < 1 or logits.dtype not in (torch.bfloat16, torch.float32) or 0 in shape:
        raise ValueError("sample_token expects bf16 or fp32 logits [..., V]")
    vocab = shape[-1]
    flat = logits if len(shape) == 2 else logits.reshape(-1, vocab)
    rows, strides = flat.shape[0], flat.stride()
    if strides[1] != 1 or (rows > 1 and strides[0] < vocab):
        flat = flat.contiguous()
        strides = (vocab, 1)
    if uniform.dtype != torch.float32 or uniform.numel() != rows or not uniform.is_contiguous():
        raise ValueError("uniform must be contiguous float32 with one value per row")
    heat, heat_all = _setting(temperature, "temperature", rows, torch.float32, 0.0)
    k, k_all = _setting(top_k, "top_k", rows, torch.int64, 0)
    p, p_all = _setting(top_p, "top_p", rows, torch.float32, 0.0)
    m, m_all = _setting(min_p, "min_p", rows, torch.float32, 0.0)
    if out is None:
        out = torch.empty(rows, dtype=torch.int64, device=logits.device)
        if len(shape) != 2:
            out = out.view(shape[:-1])
    elif out.dtype != torch.int64 or out.shape != shape[:-1] or not out.is_contiguous():
        raise ValueError("out must be contiguous int64 with one entry per row")
    index = _place(flat, uniform, heat, k, p, m, out)
    nbytes = _scratch_bytes(rows, vocab)
    scratch = torch.empty(nbytes, dtype=torch.uint8, device=flat.device)
    _launch("htn_sample", index, flat.data_ptr(), strides[0], flat.dtype is torch.float32, rows,
            vocab, uniform.data_ptr(), _lib.ptr(heat), heat_all, _lib.ptr(k), min(int(k_all), vocab),
            _lib.ptr(p), p_all, _lib.ptr(m), m_all, out.data_ptr(), scratch.data_ptr(), nbytes)
    return out
