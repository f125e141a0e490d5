"""Attention over the paged cache with a sliding window and a few first tokens that stay visible (sinks).

The reference's paged kernel has the window alone (python/dlBLAS/dlblas/kernels/paged_attention.py:421-424, 447)."""
from __future__ import annotations

import torch
from torch import Tensor

from .. import _lib


def _is64(t: Tensor, name: str) -> int:
    assert t.dtype in (torch.int32, torch.int64), f"{name} must be int32 or int64, got {t.dtype}"
    return int(t.dtype == torch.int64)


def check_paged(q: Tensor, k: Tensor, v: Tensor, o: Tensor):
    """What the paged operators of this module and of shared_prefix_attention take; returns q with rows that the copy
    engine can fetch."""
    assert q.dim() == 3 and k.dim() == 4 and v.dim() == 4, "q is [tokens, Hq, D], the caches [pages, page_size, Hkv, D]"
    assert q.dtype in (torch.float16, torch.bfloat16) and k.dtype == v.dtype == o.dtype == q.dtype, \
        "q, the caches and o must be fp16 or bf16, all the same"
    assert k.size(3) == q.size(2) and v.shape[:3] == k.shape[:3], "the caches do not fit q or each other"
    assert o.dim() == 3 and o.shape[:2] == q.shape[:2] and o.size(2) == v.size(3), "o must be [tokens, Hq, Dv]"
    assert q.size(1) % k.size(2) == 0 and q.size(1) <= 128 * k.size(2), "Hq: a multiple of Hkv, at most 128 to one"
    assert k.stride(3) == 1 and v.stride(3) == 1 and o.stride(2) == 1, "the last dimension must be contiguous"
    if q.stride(2) != 1 or q.stride(0) % 8 or q.stride(1) % 8 or q.data_ptr() % 16:
        q = q.clone(memory_format=torch.contiguous_format)
    return q


def sink_attention_fwd(
    q: Tensor,
    k: Tensor,
    v: Tensor,
    o: Tensor,
    block_offsets: Tensor,
    q_start_loc: Tensor,
    q_seqlens: Tensor,
    kv_seqlens: Tensor,
    max_seqlen: int,
    window_size: int,
    num_sinks: int,
    sm_scale: float = None,
    logit_softcapping: float = None,
):
    """Attention over the paged cache where a query at position p sees its own token, the `window_size` tokens before it
    and the first `num_sinks` tokens of its sequence.

    Arguments as in `paged_attention_fwd`: `q` [total_q, Hq, D] packed by `q_start_loc` / `q_seqlens`, caches `k` / `v`
    [num_pages, page_size, Hkv, D], which already hold the new tokens, `o` [total_q, Hq, Dv] written in place,
    `block_offsets` [batch, max_pages], `kv_seqlens` [batch] tokens in the cache, the new ones included; index tensors
    int32 or int64.  `max_seqlen` is the largest of `q_seqlens`: 1 takes the form for single tokens (sequences with
    none are left out), anything larger the one for chunks of prompts or several drafted tokens, any mixture of
    lengths.  Rows of `q` and `o` that belong to no sequence are left as they are; a query that sees no key gets zeros.

    Only pages with a token that some query of a tile of 128 rows sees are looked at: entries of `block_offsets` for
    tokens behind the window may be stale.  A page outside the cache where a visible token should be is an error
    (`check_device_status()` raises), and its sequence's output is undefined.  fp16/bf16, head sizes multiples of 8 up
    to 128, page size a power of two >= 16, at most 128 query heads to a key head, `o` and the caches 16-byte aligned
    in their rows.
    """
    dev = _lib.require_cuda(q, k, v, o, block_offsets, q_start_loc, q_seqlens, kv_seqlens)
    q = check_paged(q, k, v, o)
    batch = q_seqlens.numel()
    assert block_offsets.dim() == 2 and block_offsets.size(0) >= batch and block_offsets.size(1) >= 1, \
        "block_offsets: one row per sequence"
    assert q_start_loc.numel() >= batch and kv_seqlens.numel() >= batch, "q_start_loc and kv_seqlens: one per sequence"
    assert window_size >= 0 and num_sinks >= 0 and max_seqlen >= 0, "window_size, num_sinks and max_seqlen must not be negative"
    if block_offsets.stride(1) != 1:
        block_offsets = block_offsets.contiguous()
    q_start_loc, q_seqlens, kv_seqlens = q_start_loc.contiguous(), q_seqlens.contiguous(), kv_seqlens.contiguous()
    tokens, hq, dk = q.shape
    pages, page, hkv, dv = v.shape
    if sm_scale is None:
        sm_scale = dk ** -0.5
    status = _lib.status_word(dev)
    (qs0, qs1, _), (os0, os1, _), (ks0, ks1, ks2, _), (vs0, vs1, vs2, _) = q.stride(), o.stride(), k.stride(), v.stride()
    lib = _lib.load()
    with _lib.on_device(dev):
        rc = lib.dlb_sink_attention(
            q.data_ptr(), k.data_ptr(), v.data_ptr(), o.data_ptr(), block_offsets.data_ptr(), q_start_loc.data_ptr(),
            q_seqlens.data_ptr(), kv_seqlens.data_ptr(), batch, tokens, int(max_seqlen), hq, hkv, dk, dv, page, pages,
            block_offsets.size(1), qs0, qs1, os0, os1, ks0, ks1, ks2, vs0, vs1, vs2, block_offsets.stride(0),
            _is64(block_offsets, "block_offsets"), _is64(q_start_loc, "q_start_loc"), _is64(q_seqlens, "q_seqlens"),
            _is64(kv_seqlens, "kv_seqlens"), int(window_size), int(num_sinks), float(sm_scale),
            float(logit_softcapping or -1.0), _lib.dtype_code(q), status.data_ptr(), _lib.stream_ptr(dev))
    _lib.check(rc, "sink_attention_fwd")
    return o
