"""Decode attention for sequences that share a long prefix, whose keys and values are read once for all of them.

No counterpart in the reference, whose decode reads every sequence's whole context
(python/dlBLAS/dlblas/kernels/paged_attention.py:492-671)."""
from __future__ import annotations

from functools import lru_cache

import torch
from torch import Tensor

from .. import _lib
from .sink_attention import _is64, check_paged

_SLOTS = 148 * 2      # CTAs that are resident at a time


@lru_cache(maxsize=256)
def _pick_prefix_chunk(tiles: int, blocks: int) -> int:
    """Tokens per split of the prefix: `tiles` (row tile, kv head) pairs, `blocks` blocks of 64 keys.  A CTA costs about six
    blocks of set-up, output and joining, one of a pair on an SM about three halves of one alone; the split with
    the shortest sum over the waves is taken."""
    best, chunk = None, blocks
    for splits in range(1, min(blocks, 128) + 1):
        per = -(-blocks // splits)
        ctas = tiles * -(-blocks // per)
        cost = -(-ctas // _SLOTS) * (per + 6) * (2 if ctas <= _SLOTS // 2 else 3)
        if best is None or cost < best:
            best, chunk = cost, per
    return chunk * 64


def shared_prefix_attention_fwd(
    q: Tensor,
    k: Tensor,
    v: Tensor,
    o: Tensor,
    prefix_offsets: Tensor,
    prefix_seqlens: Tensor,
    group_start: Tensor,
    block_offsets: Tensor,
    kv_seqlens: Tensor,
    sm_scale: float = None,
    logit_softcapping: float = None,
):
    """Decode attention of a batch in groups that share a prefix: token b sees the prefix of its group and then its own
    tokens, one softmax over both.

    `q` [batch, Hq, D] holds one token per sequence, `k` / `v` are the paged caches [num_pages, page_size, Hkv, D],
    `o` [batch, Hq, Dv] is written in place.  Group g is the sequences group_start[g] .. group_start[g + 1] - 1
    (`group_start` [groups + 1], ascending); its prefix is the first prefix_seqlens[g] tokens on the pages
    prefix_offsets[g] ([groups, pages], `prefix_seqlens` [groups]).  The sequence's own tokens, the new one included,
    are the first kv_seqlens[b] on the pages block_offsets[b] ([batch, pages], `kv_seqlens` [batch]): they start on a
    page of their own, wherever the prefix ends.  Index tensors are int32 or int64.  A sequence in no group has no
    prefix, lengths may be zero, and a query without any key gets zeros.

    The prefix is cut into splits that all sequences of a group go through together as the rows of matrix products; the
    partial results wait in a workspace and join the sequences' own tokens in the second of two launches.  A page
    outside the cache where a token should be is an error (`check_device_status()` raises).  Types, head sizes, pages
    and alignment as in `sink_attention_fwd`.
    """
    dev = _lib.require_cuda(q, k, v, o, prefix_offsets, prefix_seqlens, group_start, block_offsets, kv_seqlens)
    q = check_paged(q, k, v, o)
    batch, hq, dk = q.shape
    pages, page, hkv, dv = v.shape
    groups = prefix_seqlens.numel()
    assert groups >= 1 and group_start.numel() == groups + 1, "group_start: one more entry than prefixes"
    assert prefix_offsets.dim() == 2 and prefix_offsets.size(0) >= groups and prefix_offsets.size(1) >= 1, \
        "prefix_offsets: one row per prefix"
    assert block_offsets.dim() == 2 and block_offsets.size(0) >= batch and block_offsets.size(1) >= 1, \
        "block_offsets: one row per sequence"
    assert kv_seqlens.numel() >= batch, "kv_seqlens: one per sequence"
    if prefix_offsets.stride(1) != 1:
        prefix_offsets = prefix_offsets.contiguous()
    if block_offsets.stride(1) != 1:
        block_offsets = block_offsets.contiguous()
    prefix_seqlens, group_start, kv_seqlens = prefix_seqlens.contiguous(), group_start.contiguous(), kv_seqlens.contiguous()
    if sm_scale is None:
        sm_scale = dk ** -0.5
    prefix_pages = prefix_offsets.size(1)
    rows = 128 // (hq // hkv)             # tokens to a row tile
    chunk = _pick_prefix_chunk((batch // rows + min(groups, batch)) * hkv, -(-prefix_pages * page // 64))
    splits = -(-prefix_pages * page // chunk)
    lib = _lib.load()
    floats = lib.dlb_shared_prefix_workspace_floats(batch, hq, max(dk, dv), splits)
    partial = torch.empty(floats, dtype=torch.float32, device=dev)
    status = _lib.status_word(dev)
    (qs0, qs1, _), (os0, os1, _), (ks0, ks1, ks2, _), (vs0, vs1, vs2, _) = q.stride(), o.stride(), k.stride(), v.stride()
    with _lib.on_device(dev):
        rc = lib.dlb_shared_prefix_attention(
            q.data_ptr(), k.data_ptr(), v.data_ptr(), o.data_ptr(), prefix_offsets.data_ptr(),
            prefix_seqlens.data_ptr(), group_start.data_ptr(), block_offsets.data_ptr(), kv_seqlens.data_ptr(),
            partial.data_ptr(), batch, groups, hq, hkv, dk, dv, page, pages, prefix_pages, block_offsets.size(1),
            qs0, qs1, os0, os1, ks0, ks1, ks2, vs0, vs1, vs2, prefix_offsets.stride(0), block_offsets.stride(0),
            _is64(prefix_offsets, "prefix_offsets"), _is64(prefix_seqlens, "prefix_seqlens"),
            _is64(group_start, "group_start"), _is64(block_offsets, "block_offsets"), _is64(kv_seqlens, "kv_seqlens"),
            chunk, float(sm_scale), float(logit_softcapping or -1.0), _lib.dtype_code(q), status.data_ptr(),
            _lib.stream_ptr(dev))
    _lib.check(rc, "shared_prefix_attention_fwd")
    return o
