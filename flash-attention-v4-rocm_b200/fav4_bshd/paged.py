"""Serving from a paged key/value cache: append, attend, and attend behind a shared prefix.

The cache is two BF16 tensors ``[pages, page_size, H_kv, 128]`` (page_size a multiple of 16; any strides
with contiguous elements). Key s of sequence b lives in slot ``s % page_size`` of page
``page_table[b, s // page_size]``. Queries are packed rows: sequence b owns rows ``cu_q[b]..cu_q[b+1]``,
and they are its newest keys, so ``seq_lens[b]`` counts them already::

    q = paged.append(q, k, v, k_cache, v_cache, page_table, seq_lens, cu_q, cos, sin)
    o = paged.attention(q, k_cache, v_cache, page_table, seq_lens, cu_q, max_sq)

``page_table``, ``seq_lens`` and ``cu_q`` are device int32 and read on the device only, so a step can be
captured in a CUDA graph and replayed with other lengths. These are serving operators: they have no
gradient. ``torch.ops.fav4.paged_append`` / ``paged_forward`` / ``shared_prefix_forward``
(fav4_bshd.ops) are the same calls as PyTorch operators.
"""
from __future__ import annotations

import torch

from . import HEAD_DIM, Runner

_RUNNER: Runner | None = None


def _runner() -> Runner:
    global _RUNNER
    if _RUNNER is None:
        _RUNNER = Runner()
    return _RUNNER


def append(q, k, v, k_cache, v_cache, page_table, seq_lens, cu_q, cos=None, sin=None, *, interleaved=False,
           offsets=None, out=None):
    """Writes k and v of the new tokens into their slots and returns q, with q and k rotated by the rows of cos / sin
    (FP32 ``[positions, rotary/2]``) at their positions; ``cos=None`` appends without rotation. ``offsets`` (int32
    ``[B]``) shifts a sequence's rotation positions, for keys behind a shared prefix."""
    if out is None:
        out = torch.empty(q.shape, dtype=q.dtype, device=q.device)
    if q.device.index == torch.cuda.current_device():
        _runner().paged_append(q, k, v, out, k_cache, v_cache, page_table, seq_lens, cu_q, cos, sin, interleaved,
                               offsets)
    else:
        with torch.cuda.device(q.device):
            _runner().paged_append(q, k, v, out, k_cache, v_cache, page_table, seq_lens, cu_q, cos, sin, interleaved,
                                   offsets)
    return out


def _attend(q, k_cache, v_cache, page_table, seq_lens, cu_q, max_sq, causal, scale, out, return_lse, prefix_pages,
            prefix_len):
    if out is None:
        out = torch.empty(q.shape, dtype=q.dtype, device=q.device)
    lse = torch.empty((q.shape[1], q.shape[0]), dtype=torch.float32, device=q.device) if return_lse else None
    if q.device.index == torch.cuda.current_device():
        _runner().call_paged(q, out, lse, k_cache, v_cache, page_table, seq_lens, cu_q, max_sq, causal, scale,
                             prefix_pages, prefix_len)
    else:
        with torch.cuda.device(q.device):
            _runner().call_paged(q, out, lse, k_cache, v_cache, page_table, seq_lens, cu_q, max_sq, causal, scale,
                                 prefix_pages, prefix_len)
    return (out, lse) if return_lse else out


def attention(q, k_cache, v_cache, page_table, seq_lens, cu_q, max_sq: int, *, causal=True, scale=None, out=None,
              return_lse=False):
    """O ``[T, H, 128]``, or (O, LSE ``[H, T]``), of packed queries over the pages. ``max_sq`` bounds the new tokens of
    a sequence. Causal is bottom-right: row i of sq sees keys up to ``seq_lens[b] - sq + i``."""
    return _attend(q, k_cache, v_cache, page_table, seq_lens, cu_q, max_sq, causal, scale, out, return_lse, None, None)


def shared_prefix_attention(q, k_cache, v_cache, prefix_pages, prefix_len, page_table, seq_lens, cu_q, max_sq: int, *,
                            causal=True, scale=None, out=None, return_lse=False):
    """``attention`` where ``prefix_len`` (device int32 ``[1]``) keys at ``prefix_pages`` (device int32 ``[n]``) stand
    before every sequence's own keys and are read once for the whole batch; ``seq_lens`` and ``page_table`` are the
    sequences' own."""
    return _attend(q, k_cache, v_cache, page_table, seq_lens, cu_q, max_sq, causal, scale, out, return_lse,
                   prefix_pages, prefix_len)


__all__ = ["HEAD_DIM", "append", "attention", "shared_prefix_attention"]
