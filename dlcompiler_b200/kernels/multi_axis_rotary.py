"""Rotary position embedding with several position axes (time, height, width for images and video).

No counterpart in the reference, whose rotary kernels take one row of cos / sin per token
(python/dlBLAS/dlblas/kernels/apply_rotary_pos_emb.py:98)."""
from __future__ import annotations

import ctypes
from functools import lru_cache
from typing import Sequence

import torch
from torch import Tensor
from torch.autograd import forward_ad

from .. import _lib


@lru_cache(maxsize=64)
def _axis_of_freq(sections: tuple, interleaved: bool, axes: int, freqs: int):
    """Axis of every frequency as a host byte array."""
    assert len(sections) == axes and all(n >= 0 for n in sections) and sum(sections) == freqs, \
        "sections: one count per axis, together as many as frequencies"
    if interleaved:
        order = [a for _, a in sorted((i, a) for a, n in enumerate(sections) for i in range(n))]
    else:
        order = [a for a, n in enumerate(sections) for _ in range(n)]
    return (ctypes.c_uint8 * max(freqs, 1))(*order)


def _launch(q, k, q_out, k_out, positions, inv_freq, axes, inverse):
    tokens, hq, dim = q.shape
    dev = q.device
    with _lib.on_device(dev):
        rc = _lib.load().dlb_multi_axis_rotary(
            q.data_ptr(), k.data_ptr(), q_out.data_ptr(), k_out.data_ptr(), positions.data_ptr(),
            positions.dtype is torch.int64, positions.stride(0), inv_freq.data_ptr(), axes, positions.size(0), tokens, hq,
            k.size(1), dim, 2 * inv_freq.numel(), *q.stride()[:2], *k.stride()[:2], *q_out.stride()[:2],
            *k_out.stride()[:2], inverse, _lib.dtype_code(q), _lib.stream_ptr(dev))
    _lib.check(rc, "apply_multi_axis_rotary")


def _dense(t):
    return t if t.stride(-1) == 1 or t.size(-1) == 1 else t.contiguous()


def _output(out, x):
    if out is None:
        return torch.empty_like(x, memory_format=torch.contiguous_format)
    assert out.shape == x.shape and out.dtype is x.dtype and (out.stride(-1) == 1 or out.size(-1) == 1), \
        "q_embed / k_embed must have their input's shape and dtype, the last dimension contiguous"
    return out


def _rotated(q, k, positions, inv_freq, axes, inverse, q_out=None, k_out=None):
    q, k = _dense(q), _dense(k)
    q_out, k_out = _output(q_out, q), _output(k_out, k)
    _launch(q, k, q_out, k_out, positions, inv_freq, axes, inverse)
    return q_out, k_out


def _has_tangent(*tensors):
    """Does one of them carry a tangent of forward-mode differentiation?"""
    return forward_ad._current_level >= 0 and any(
        t is not None and forward_ad.unpack_dual(t).tangent is not None for t in tensors)


class _MultiAxisRotary(torch.autograd.Function):
    """A rotation is linear and its transpose the rotation back: tangents take the same launch, gradients the one with the
    other sign (and, where they are to be differentiated again, this function)."""

    @staticmethod
    def forward(ctx, q, k, positions, inv_freq, axes, inverse):
        ctx.save_for_backward(positions, inv_freq)
        if forward_ad._current_level >= 0:
            ctx.save_for_forward(positions, inv_freq)
        ctx.axes, ctx.inverse, ctx.shapes = axes, inverse, (q.shape, k.shape)
        ctx.set_materialize_grads(False)
        return _rotated(q, k, positions, inv_freq, axes, inverse)

    @staticmethod
    def _rotate_some(ctx, q, k, inverse):
        """One of the two may be None: its heads are left out of the launch."""
        if q is None and k is None:
            return None, None
        positions, inv_freq = ctx.saved_tensors
        some = k if q is None else q
        none = some.new_empty((some.size(0), 0, some.size(2))) if q is None or k is None else None
        rotate = _MultiAxisRotary.apply if torch.is_grad_enabled() or _has_tangent(q, k) else _rotated
        q_out, k_out = rotate(none if q is None else q, none if k is None else k, positions, inv_freq, ctx.axes, inverse)
        return None if q is None else q_out, None if k is None else k_out

    @staticmethod
    def backward(ctx, grad_q, grad_k):
        # an output that nothing was made of has no gradient, an input may want none
        if not ctx.needs_input_grad[0]:
            grad_q = None
        if not ctx.needs_input_grad[1]:
            grad_k = None
        return *_MultiAxisRotary._rotate_some(ctx, grad_q, grad_k, not ctx.inverse), None, None, None, None

    @staticmethod
    def jvp(ctx, q_tangent, k_tangent, *_):
        some = k_tangent if q_tangent is None else q_tangent
        out = _MultiAxisRotary._rotate_some(ctx, q_tangent, k_tangent, ctx.inverse)
        return tuple(some.new_zeros(shape) if t is None else t for t, shape in zip(out, ctx.shapes))    # none is not taken


def apply_multi_axis_rotary(
    q: Tensor,
    k: Tensor,
    positions: Tensor,
    inv_freq: Tensor,
    sections: Sequence[int],
    interleaved: bool = False,
    q_embed: Tensor = None,
    k_embed: Tensor = None,
):
    """Rotate-half rotary embedding of query and key ([tokens, heads, dim]) at positions with several axes.

    `positions` [axes, tokens] (int32 or int64, 1 to 8 axes) holds each token's place on every axis, `inv_freq` (fp32,
    up to dim / 2 and 256 of them) the angle per step of each frequency; the first `2 * len(inv_freq)` columns are
    rotated (column f with column f + len(inv_freq)), the others pass through.  `sections[a]` frequencies follow axis
    a: the first sections[0] frequencies the first axis and so on, or, with `interleaved`, one frequency to each axis
    in turn, an axis dropping out once it has its number.  Angles are formed in twice 64 bits and the rotation in 32, with
    one rounding to the tensors' type (fp16, bf16, fp32): no cos / sin tables, and angles as good far out, up to position
    2^53, as near 0.

    Differentiable in q and k, backward and forward (`torch.autograd.forward_ad`), more than once; `q_embed` / `k_embed` (which may
    be q and k themselves) are for calls without a gradient or tangent.  Returns (q_embed, k_embed).
    """
    dev = _lib.require_cuda(q, k, positions, inv_freq, q_embed, k_embed)
    assert q.dim() == 3 and k.dim() == 3 and positions.dim() == 2, "q and k are [tokens, heads, dim], positions [axes, tokens]"
    (tokens, _, dim), (tokens_k, _, dim_k), (n_axes, places) = q.shape, k.shape, positions.shape
    assert tokens_k == tokens and places == tokens and dim_k == dim, "q, k and positions need the same tokens, q and k the same dim"
    assert k.dtype is q.dtype, "q and k must have one dtype"
    assert positions.dtype is torch.int64 or positions.dtype is torch.int32, "positions must be int32 or int64"
    assert inv_freq.dim() == 1 and inv_freq.dtype is torch.float32, "inv_freq is a vector of fp32"
    dual = forward_ad._current_level >= 0              # tangents are looked for only where there may be some
    assert not (inv_freq.requires_grad or dual and _has_tangent(inv_freq)), "there is no gradient for inv_freq"
    axes = _axis_of_freq(tuple(sections), bool(interleaved), n_axes, inv_freq.numel())
    if positions.stride(1) != 1:
        positions = positions.contiguous()
    inv_freq = inv_freq.contiguous()
    if (q.requires_grad or k.requires_grad) and torch.is_grad_enabled() or dual and _has_tangent(q, k):
        assert q_embed is None and k_embed is None, "outputs cannot be given where a gradient or tangent is wanted"
        return _MultiAxisRotary.apply(q, k, positions, inv_freq, axes, False)
    return _rotated(q, k, positions, inv_freq, axes, False, q_embed, k_embed)
