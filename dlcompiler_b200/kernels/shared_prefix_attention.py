"""Decode attention for sequences that share a long prefix, whose keys and values are read once for all of them.

No counterpart in the reference, whose decode reads every sequence's whole context
(python/dlBLAS/dlblas/kernels/paged_attention.py:492-671)."""
from __future__ import annotations

from functools import lru_cache

import torch
from torch import Tensor

from .. import _lib
from .sink_attention import check_paged, is64, rows_of_table

# CTAs that run at a time, by the size of their clusters: a cluster stays inside a GPC, so that larger ones leave slots empty
_SLOTS = {1: 296, 2: 296, 4: 280, 8: 256}


@lru_cache(maxsize=256)
def _pick_prefix_split(tiles: int, blocks: int):
    """(tokens per split, CTAs per split) for `tiles` (row tile, kv head) pairs and `blocks` blocks of 64 keys.  In microseconds a
    CTA takes about 0.7 for a block and 4 for the rest, a partial result 0.02 per pair (128 rows written and read again)
    and 0.3 for its place in the join; the CTAs of a cluster join theirs among themselves in 1.  The shortest sum is taken."""
    best, pick = None, (blocks, 1)
    for cluster in (1, 2, 4, 8):
        for splits in range(1, min(blocks, 64) + 1):
            per = -(-blocks // splits)
            splits = -(-blocks // per)
            mine = -(-per // cluster)
            cost = -(-tiles * splits * cluster // _SLOTS[cluster]) * (mine * 0.7 + 4 + (cluster > 1)) + splits * (0.02 * tiles + 0.3)
            if best is None or cost < best:
                best, pick = cost, (per, cluster)
    return pick[0] * 64, pick[1]


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
    q, (batch, hq, hkv, dk, dv, page, pages), strides = check_paged(q, k, v, o)
    groups = prefix_seqlens.numel()
    assert groups >= 1 and group_start.numel() == groups + 1, "group_start: one more entry than prefixes"
    prefix_offsets, prefix_pages, pt_stride = rows_of_table(prefix_offsets, groups, "prefix_offsets")
    block_offsets, columns, bt_stride = rows_of_table(block_offsets, batch, "block_offsets")
    assert kv_seqlens.numel() >= batch, "kv_seqlens: one per sequence"
    prefix_seqlens, group_start, kv_seqlens = prefix_seqlens.contiguous(), group_start.contiguous(), kv_seqlens.contiguous()
    wide = (is64(prefix_offsets, "prefix_offsets"), is64(prefix_seqlens, "prefix_seqlens"), is64(group_start, "group_start"),
            is64(block_offsets, "block_offsets"), is64(kv_seqlens, "kv_seqlens"))
    most = prefix_pages * page
    heads = hq // hkv
    tokens = (64 if -(-batch // groups) * heads <= 64 else 128) // heads              # to a row tile
    chunk, cluster = _pick_prefix_split((batch // tokens + min(groups, batch)) * hkv, -(-most // 64))
    lib = _lib.load()
    with _lib.on_device(dev):
        floats = lib.dlb_shared_prefix_workspace_floats(batch, hq, max(dk, dv), -(-most // chunk))
        partial = torch.empty(floats, dtype=torch.float32, device=dev)
        rc = lib.dlb_shared_prefix_attention(
            q.data_ptr(), k.data_ptr(), v.data_ptr(), o.data_ptr(), prefix_offsets.data_ptr(),
            prefix_seqlens.data_ptr(), group_start.data_ptr(), block_offsets.data_ptr(), kv_seqlens.data_ptr(),
            partial.data_ptr(), batch, groups, hq, hkv, dk, dv, page, pages, prefix_pages, columns, *strides, pt_stride,
            bt_stride, *wide, chunk, cluster, dk ** -0.5 if sm_scale is None else sm_scale, logit_softcapping or -1.0,
            _lib.dtype_code(q), _lib.status_word(dev).data_ptr(), _lib.stream_ptr(dev))
    _lib.check(rc, "shared_prefix_attention_fwd")
    return o
