"""Attention over the paged cache with a sliding window and a few first tokens that stay visible (sinks).

The reference's paged kernel has the window alone (python/dlBLAS/dlblas/kernels/paged_attention.py:421-424, 447)."""
from __future__ import annotations

import torch
from torch import Tensor

from .. import _lib


_IS64 = {torch.int32: 0, torch.int64: 1}


def is64(t: Tensor, name: str) -> int:
    code = _IS64.get(t.dtype)
    assert code is not None, f"{name} must be int32 or int64, got {t.dtype}"
    return code


def rows_of_table(table: Tensor, rows: int, name: str):
    """A block table (copied where its rows are not contiguous), its columns and the stride of its rows."""
    assert table.dim() == 2, f"{name} has two dimensions"
    have, columns = table.shape
    assert have >= rows and columns >= 1, f"{name}: one row of pages for each of {rows}, got {tuple(table.shape)}"
    stride, step = table.stride()
    if step != 1:
        table = table.contiguous()
        stride = columns
    return table, columns, stride


def check_paged(q: Tensor, k: Tensor, v: Tensor, o: Tensor):
    """What the paged operators of this module and of shared_prefix_attention take.  Returns q with rows that the copy engine
    can fetch, the sizes (tokens, Hq, Hkv, D, Dv, page size, pages) and the strides of q, o, k and v in the order of the
    C entries."""
    assert q.dim() == 3 and k.dim() == 4 and v.dim() == 4 and o.dim() == 3, \
        "q and o are [tokens, Hq, D], the caches [pages, page_size, Hkv, D]"
    dtype = q.dtype
    assert (dtype is torch.bfloat16 or dtype is torch.float16) and k.dtype is dtype and v.dtype is dtype and o.dtype is dtype, \
        "q, the caches and o must be fp16 or bf16, all the same"
    (tokens, hq, dk), (pages, page, hkv, dim_k), (*like, dv) = q.shape, k.shape, v.shape
    assert dim_k == dk and like == [pages, page, hkv], "the caches do not fit q or each other"
    assert o.shape == (tokens, hq, dv), "o must be [tokens, Hq, Dv]"
    assert hkv > 0 and hq % hkv == 0 and hq <= 128 * hkv, "Hq: a multiple of Hkv, at most 128 to one"
    (q_st, q_sh, q_last), (o_st, o_sh, o_last) = q.stride(), o.stride()
    (*k_strides, k_last), (*v_strides, v_last) = k.stride(), v.stride()
    assert k_last == 1 and v_last == 1 and o_last == 1, "the last dimension must be contiguous"
    if q_last != 1 or q_st % 8 or q_sh % 8 or not (q_st and q_sh) or q.data_ptr() % 16:
        q = q.clone(memory_format=torch.contiguous_format)
        q_st, q_sh = hq * dk, dk
    return q, (tokens, hq, hkv, dk, dv, page, pages), (q_st, q_sh, o_st, o_sh, *k_strides, *v_strides)


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
    int32 or int64.  Other than there, `window_size` has no value for no window (None and -1 are refused, one as long as the
    longest context hides nothing), and 0 leaves the query's own token and the sinks.  `max_seqlen` is the largest of `q_seqlens`: 1 takes the form for single tokens (sequences with
    none are left out, of longer ones only the first token is computed), anything larger the one for chunks of prompts or
    several drafted tokens, any mixture of lengths.  Rows of `q` and `o` that belong to no sequence are left as they are; a
    query that sees no key gets zeros.  Where `kv_seqlens` is past what a row of `block_offsets` has room for, queries keep their
    positions and the tokens past the table are not there.

    The form for single tokens is one launch without a workspace, in which at most 8 CTAs share the keys of a sequence and key
    head: made for windows of some thousand keys, or batches that fill the GPU.  A few sequences behind a window of 100000 keys
    and more are better served by `paged_attention_fwd` where there are no sinks to keep (one sequence, one key head, 131072 keys:
    178 us here, 123 there).

    Only pages with a token that some query of a tile of 128 rows sees are looked at: entries of `block_offsets` for
    tokens behind the window may be stale.  A page outside the cache where a visible token should be is an error
    (`check_device_status()` raises), and its sequence's output is undefined.  fp16/bf16, head sizes multiples of 8 up
    to 128, page size a power of two >= 16, at most 128 query heads to a key head, `o` and the caches 16-byte aligned
    in their rows, `sm_scale` positive.  An infinity or NaN in a visible token's values reaches every query of the sequence
    that shares a tile with one that sees it (its weight there is 0, and 0 x inf is no number).
    """
    dev = _lib.require_cuda(q, k, v, o, block_offsets, q_start_loc, q_seqlens, kv_seqlens)
    q, (tokens, hq, hkv, dk, dv, page, pages), strides = check_paged(q, k, v, o)
    batch = q_seqlens.numel()
    block_offsets, columns, bt_stride = rows_of_table(block_offsets, batch, "block_offsets")
    assert q_start_loc.numel() >= batch and kv_seqlens.numel() >= batch, "q_start_loc and kv_seqlens: one per sequence"
    assert window_size is not None and window_size >= 0 and num_sinks >= 0 and max_seqlen >= 0, \
        "window_size, num_sinks and max_seqlen must not be negative (there is no window_size for none: pass the longest context)"
    q_start_loc, q_seqlens, kv_seqlens = q_start_loc.contiguous(), q_seqlens.contiguous(), kv_seqlens.contiguous()
    wide = (is64(block_offsets, "block_offsets"), is64(q_start_loc, "q_start_loc"), is64(q_seqlens, "q_seqlens"),
            is64(kv_seqlens, "kv_seqlens"))
    lib = _lib.load()
    with _lib.on_device(dev):
        rc = lib.dlb_sink_attention(
            q.data_ptr(), k.data_ptr(), v.data_ptr(), o.data_ptr(), block_offsets.data_ptr(), q_start_loc.data_ptr(),
            q_seqlens.data_ptr(), kv_seqlens.data_ptr(), batch, tokens, int(max_seqlen), hq, hkv, dk, dv, page, pages,
            columns, *strides, bt_stride, *wide, min(int(window_size), 2**31), min(int(num_sinks), 2**31),
            dk ** -0.5 if sm_scale is None else sm_scale, logit_softcapping or -1.0, _lib.dtype_code(q),
            _lib.status_word(dev).data_ptr(), _lib.stream_ptr(dev))
    _lib.check(rc, "sink_attention_fwd")
    return o
