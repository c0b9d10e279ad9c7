"""Serving from a paged key/value cache: append, attend, and attend behind a shared prefix.

The cache is two BF16 tensors ``[pages, page_size, H_kv, 128]`` (page_size a multiple of 16; any strides
with contiguous elements). Key s of sequence b lives in slot ``s % page_size`` of page
``page_table[b, s // page_size]``. Queries are packed rows: sequence b owns rows ``cu_q[b]..cu_q[b+1]``,
and they are its newest keys, so ``seq_lens[b]`` counts them already::

    q = paged.append(q, k, v, k_cache, v_cache, page_table, seq_lens, cu_q, cos, sin)
    o = paged.attention(q, k_cache, v_cache, page_table, seq_lens, cu_q, max_sq)

``page_table``, ``seq_lens`` and ``cu_q`` are device int32 and read on the device only, so a step can be
captured in a CUDA graph and replayed with other lengths. Every call runs on the current stream with a
workspace of that stream's own (a captured call: of the graph's). These are serving operators: they have no
gradient and refuse inputs that want one. ``torch.ops.fav4.paged_append`` / ``paged_forward`` / ``shared_prefix_forward``
(fav4_bshd.ops) are the same calls as PyTorch operators.
"""
from __future__ import annotations

import importlib.machinery
import importlib.util

from . import BUILD_DIR, HEAD_DIM

BINDING_PATH = BUILD_DIR / "fav4_paged_torch.so"
_BINDING = None


def load_binding():
    """Load (once) the native module that checks the arguments and calls the library (csrc/paged_torch.cpp)."""
    global _BINDING
    if _BINDING is None:
        if not BINDING_PATH.exists():
            raise RuntimeError(f"{BINDING_PATH} is missing: build it with `python -m fav4_bshd.build` "
                               f"(or __graft_entry__.build()); there is no CPU fallback")
        import torch  # noqa: F401  (its libraries come first)
        loader = importlib.machinery.ExtensionFileLoader("fav4_paged_torch", str(BINDING_PATH))
        spec = importlib.util.spec_from_loader("fav4_paged_torch", loader)
        module = importlib.util.module_from_spec(spec)
        loader.exec_module(module)
        _BINDING = module
    return _BINDING


def append(q, k, v, k_cache, v_cache, page_table, seq_lens, cu_q, cos=None, sin=None, *, interleaved=False,
           offsets=None, out=None):
    """Writes k and v of the new tokens into their slots and returns q, with q and k rotated by the rows of cos / sin
    (FP32 ``[positions, rotary/2]``) at their positions; ``cos=None`` appends without rotation. q ``[T, H, 128]``, k and
    v ``[T, H_kv, 128]`` may be strided (slices of one projection). ``offsets`` (int32 ``[B]``) shifts a sequence's
    rotation positions, for keys behind a shared prefix. ``out`` may be q's own memory when q is contiguous, and
    must not overlap anything else."""
    return load_binding().append(q, k, v, k_cache, v_cache, page_table, seq_lens, cu_q, cos, sin, interleaved, offsets, out)


def attention(q, k_cache, v_cache, page_table, seq_lens, cu_q, max_sq: int, *, causal=True, scale=None, out=None,
              return_lse=False):
    """O ``[T, H, 128]``, or (O, LSE ``[H, T]``), of packed queries over the pages. ``max_sq`` bounds the new tokens of
    a sequence. Causal is bottom-right: row i of sq sees keys up to ``seq_lens[b] - sq + i``; rows without a key get
    O = 0 and LSE = -inf. ``out`` must not overlap q or the caches. Rows of no sequence, and a sequence's rows past ``max_sq``, are
    not written."""
    return load_binding().attend(q, k_cache, v_cache, page_table, seq_lens, cu_q, max_sq, causal, scale, out, return_lse,
                             None, None)


def shared_prefix_attention(q, k_cache, v_cache, prefix_pages, prefix_len, page_table, seq_lens, cu_q, max_sq: int, *,
                            causal=True, scale=None, out=None, return_lse=False):
    """``attention`` where ``prefix_len`` (device int32 ``[1]``) keys at ``prefix_pages`` (device int32 ``[n]``) stand
    before every sequence's own keys and are read once for the whole batch; ``seq_lens`` and ``page_table`` are the
    sequences' own."""
    return load_binding().attend(q, k_cache, v_cache, page_table, seq_lens, cu_q, max_sq, causal, scale, out, return_lse,
                             prefix_pages, prefix_len)


__all__ = ["HEAD_DIM", "BINDING_PATH", "load_binding", "append", "attention", "shared_prefix_attention"]
