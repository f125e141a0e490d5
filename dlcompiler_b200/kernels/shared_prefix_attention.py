"""Decode attention for sequences that share a long prefix, whose keys and values are read once for all of them.

No counterpart in the reference, whose decode reads every sequence's whole context
(python/dlBLAS/dlblas/kernels/paged_attention.py:492-671)."""
from __future__ import annotations

from functools import lru_cache

import torch
from torch import Tensor

from .. import _lib
from .sink_attention import check_paged, is64, rows_of_table


@lru_cache(maxsize=256)
def _pick_prefix_split(tiles: int, groups: int, hkv: int, blocks: int):
    """(tokens per split, CTAs per split) for `tiles` (row tile, kv head) pairs of `groups` prefixes of up to `blocks` blocks of
    64 keys, by the shortest sum, in microseconds: a block takes a CTA 1.0, beside another on its SM 1.1, or what memory needs
    for it (32 KiB at 5.8 TB/s); every wave of CTAs 4, in clusters 10 more behind the first one; a partial result 0.02 a pair
    (written and read again) and 0.3 for its place in the join, joining a cluster 1.5; and past 224 CTAs (200 in clusters of
    four) no SM has room for the launch that follows, which otherwise goes through the sequences' own tokens meanwhile: 10.
    (8 pairs, 1876 blocks, with 128 / 192 / 224 / 288 / 384 CTAs: 129 / 113 / 114 / 136 / 124; 16 pairs, 512 blocks: 106 / 87 /
    90 / 115 / 100.  256 pairs, 313 blocks, whole / in 4 splits / in 3 splits of clusters of four: 417 / 445 / 512.)  Clusters
    of two where prefixes differ in length, which splits share out more evenly."""
    memory = groups * hkv * blocks * 32768 / 5.8e6
    best, pick = None, (blocks, 1)
    for cluster in (1, 2, 4) if groups == 1 else (1, 2):
        for splits in range(1, min(blocks, 64) + 1):
            per = -(-blocks // splits)
            splits = -(-blocks // per)
            ctas = tiles * splits * cluster
            waves = -(-ctas // 280)
            work = waves * (-(-per // cluster) * (1.0 if ctas <= 148 else 1.1) + 4) + 10 * (waves - 1) * (cluster > 1)
            cost = max(work, memory + 4) + 1.5 * (cluster > 1) + splits * (0.02 * tiles + 0.3) \
                + 10 * (ctas > (224 if cluster < 4 else 200))
            if best is None or cost < best:
                best, pick = cost, (per, cluster)
    return pick[0] * 64, pick[1]


@lru_cache(maxsize=256)
def _workspace_floats(*sizes):
    return _lib.load().dlb_shared_prefix_workspace_floats(*sizes)


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
    partial results wait in a workspace and join the sequences' own tokens in the second of two launches.  Lengths stay on the
    device, so splits, workspace and the CTAs for the own tokens (at most 8 to a sequence and key head) are planned from the widths
    of the two tables: pass them about as wide as the longest entry needs (8 sequences behind 4000 tokens: 20 us, with a prefix
    table of 131072 tokens 27).  A page
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
    heads, members = hq // hkv, -(-batch // groups)
    tokens = (64 if members * heads <= 64 else 128) // heads                # to a row tile, as the launch has it
    chunk, cluster = _pick_prefix_split(min(groups, batch) * -(-members // tokens) * hkv, groups, hkv, -(-most // 64))
    lib = _lib.load()
    with _lib.on_device(dev):
        partial = torch.empty(_workspace_floats(batch, hq, max(dk, dv), -(-most // chunk)), dtype=torch.float32, device=dev)
        rc = lib.dlb_shared_prefix_attention(
            q.data_ptr(), k.data_ptr(), v.data_ptr(), o.data_ptr(), prefix_offsets.data_ptr(),
            prefix_seqlens.data_ptr(), group_start.data_ptr(), block_offsets.data_ptr(), kv_seqlens.data_ptr(),
            partial.data_ptr(), batch, groups, hq, hkv, dk, dv, page, pages, prefix_pages, columns, *strides, pt_stride,
            bt_stride, *wide, chunk, cluster, dk ** -0.5 if sm_scale is None else sm_scale, logit_softcapping or -1.0,
            _lib.dtype_code(q), _lib.status_word(dev).data_ptr(), _lib.stream_ptr(dev))
    _lib.check(rc, "shared_prefix_attention_fwd")
    return o
