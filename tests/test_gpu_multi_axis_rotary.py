"""GPU: rotary positions of several axes against complex numbers in 64 bits, forward, gradient and refusals of layouts."""
import math
from fractions import Fraction

import pytest
import torch
import torch.autograd.forward_ad as fwAD

from dlcompiler_b200 import apply_multi_axis_rotary, apply_rotary_pos_emb

pytestmark = pytest.mark.gpu


def _axes_of(sections, interleaved):
    if not interleaved:
        return [a for a, n in enumerate(sections) for _ in range(n)]
    left, out = list(sections), []
    while sum(left):
        for a in range(len(left)):
            if left[a]:
                out.append(a)
                left[a] -= 1
    return out


def _exact(x, positions, inv_freq, sections, interleaved, back=False):
    half = inv_freq.numel()
    angle = positions[_axes_of(sections, interleaved)].t().double() * inv_freq.double()
    turn = torch.polar(torch.ones_like(angle), -angle if back else angle)[:, None]
    x = x.detach().double()
    z = torch.complex(x[..., :half], x[..., half:2 * half]) * turn
    return torch.cat([z.real, z.imag, x[..., 2 * half:]], -1)


def _close(out, x, ref, half):
    """sin and cos are off by 2^-24 (their function) + 2^-25 (the first-order term) at most, each of the two products and
    the sum rounds once in 32 bits: together below 2^-22 (|lo| + |hi|); then half a step of the output's type, or of its
    smallest number.  Columns behind the rotated ones are copies."""
    x = x.detach().double()
    size = x[..., :half].abs() + x[..., half:2 * half].abs()
    slack = torch.cat([size, size, torch.zeros_like(x[..., 2 * half:])], -1) * 2.0 ** -22
    info = torch.finfo(out.dtype)
    step = info.eps / 2 * (ref.abs() + slack) + info.smallest_normal * info.eps / 2
    assert ((out.double() - ref).abs() <= slack + step).all()
    assert torch.equal(out[..., 2 * half:].double(), x[..., 2 * half:])


def _inputs(dev, tokens, hq, hk, dim, half, axes, dtype, far=0, idx=torch.int64, seed=0):
    g = torch.Generator().manual_seed(seed * 7919 + tokens * 31 + dim)
    q, k = (torch.randn(tokens, h, dim, generator=g).to(dtype).to(dev) for h in (hq, hk))
    pos = (torch.randint(0, 300, (axes, tokens), generator=g) + far).to(idx).to(dev)
    inv = (10000.0 ** (-torch.arange(half, dtype=torch.float64) / half)).float().to(dev)
    return q, k, pos, inv


CASES = [  # tokens, hq, hk, dim, half, sections, interleaved, dtype, far
    (1, 1, 1, 2, 1, [1], False, torch.float32, 0),
    (1, 32, 8, 128, 64, [16, 24, 24], False, torch.bfloat16, 5000),
    (5, 3, 1, 10, 5, [2, 2, 1], True, torch.float16, 0),
    (7, 4, 4, 80, 20, [8, 6, 6], True, torch.bfloat16, 10 ** 6),
    (600, 6, 2, 96, 32, [32], False, torch.float16, 10 ** 7),
    (601, 5, 3, 72, 36, [9, 9, 9, 9], True, torch.float32, 10 ** 6),
    (1000, 4, 1, 128, 64, [24, 20, 20], True, torch.bfloat16, 2 ** 24 - 7),
    (593, 2, 2, 512, 256, [0, 256, 0], False, torch.float32, 3),
    (33, 2, 1, 520, 250, [100, 150], True, torch.bfloat16, 3),
    (2, 1, 1, 64, 8, [1] * 8, True, torch.float16, 40),
]


@pytest.mark.parametrize("tokens,hq,hk,dim,half,sections,interleaved,dtype,far", CASES)
@pytest.mark.parametrize("idx", [torch.int32, torch.int64])
def test_against_complex_numbers(cuda_device, tokens, hq, hk, dim, half, sections, interleaved, dtype, far, idx):
    q, k, pos, inv = _inputs(cuda_device, tokens, hq, hk, dim, half, len(sections), dtype, far, idx)
    qe, ke = apply_multi_axis_rotary(q, k, pos, inv, sections, interleaved)
    for out, x in ((qe, q), (ke, k)):
        _close(out, x, _exact(x, pos, inv, sections, interleaved), half)
    # negative positions turn the other way
    qn, _ = apply_multi_axis_rotary(q, k, -pos, inv, sections, interleaved)
    _close(qn, q, _exact(q, pos, inv, sections, interleaved, back=True), half)


@pytest.mark.parametrize("dtype,dim,half", [(torch.bfloat16, 128, 64), (torch.float16, 80, 20), (torch.float32, 36, 18)])
def test_layouts_and_outputs(cuda_device, dtype, dim, half):
    """Views of a fused projection, heads outside tokens, odd offsets, a transposed last dimension, in place, given
    outputs: the bits of the contiguous call, and nothing beside the outputs written."""
    q, k, pos, inv = _inputs(cuda_device, 9, 4, 2, dim, half, 2, dtype)
    sections = [half // 2, half - half // 2]
    ref = apply_multi_axis_rotary(q, k, pos, inv, sections)
    qkv = torch.cat([q.flatten(1), k.flatten(1)], 1)
    views = [t.view(9, -1, dim) for t in qkv.split([4 * dim, 2 * dim], 1)]
    outside = [t.transpose(0, 1).contiguous().transpose(0, 1) for t in (q, k)]
    shifted = []
    for t in (q, k):
        buf = torch.zeros(t.numel() + 1, dtype=dtype, device=cuda_device)
        buf[1:] = t.flatten()
        shifted.append(buf[1:].view(t.shape))
    turned = [t.transpose(1, 2).contiguous().transpose(1, 2) for t in (q, k)]
    strided_pos = torch.stack([pos, pos + 1], -1)[..., 0]
    for a, b in (views, outside, shifted, turned):
        out = apply_multi_axis_rotary(a, b, strided_pos, inv, sections)
        assert all(torch.equal(x, y) for x, y in zip(out, ref))
    canvas = torch.full((9, 9, dim + 8), 7.0, dtype=dtype, device=cuda_device)
    qe, ke = canvas[:, 1:5, :dim], canvas[:, 6:8, :dim]
    out = apply_multi_axis_rotary(q, k, pos, inv, sections, q_embed=qe, k_embed=ke)
    assert out[0] is qe and torch.equal(qe, ref[0]) and torch.equal(ke, ref[1])
    assert (canvas[:, [0, 5, 8]] == 7).all() and (canvas[..., dim:] == 7).all()
    apply_multi_axis_rotary(*views, pos, inv, sections, q_embed=views[0], k_embed=views[1])
    assert torch.equal(views[0], ref[0]) and torch.equal(views[1], ref[1])
    empty = q[:0]
    assert apply_multi_axis_rotary(empty, k[:0], pos[:, :0], inv, sections)[0].shape == empty.shape


def test_one_axis_is_the_plain_rotary(cuda_device):
    """All tokens on one line: apply_rotary_pos_emb with its tables in 32 bits."""
    q, k, pos, inv = _inputs(cuda_device, 50, 4, 2, 64, 32, 1, torch.float32)
    a = (pos[0][:, None].double() * inv.double()).repeat(1, 2)
    ref = apply_rotary_pos_emb(q, k, a.cos().float(), a.sin().float())
    out = apply_multi_axis_rotary(q, k, pos, inv, [32])
    for x, r in zip(out, ref):
        # tables rounded to 2^-25 each, two products and a sum of 2^-24 each there; 2^-22 (|lo| + |hi|) here
        assert ((x - r).abs() <= 2.0 ** -21 * 2 * q.abs().max()).all()


@pytest.mark.parametrize("dtype,dim,half,sections,interleaved", [
    (torch.bfloat16, 128, 64, [16, 24, 24], False), (torch.float16, 80, 20, [8, 6, 6], True),
    (torch.float32, 72, 36, [9, 9, 9, 9], True), (torch.float32, 13, 4, [1, 3], False)])
def test_gradient_is_the_rotation_back(cuda_device, dtype, dim, half, sections, interleaved):
    q, k, pos, inv = _inputs(cuda_device, 37, 4, 2, dim, half, len(sections), dtype)
    q.requires_grad_(), k.requires_grad_()
    gq, gk = (torch.randn_like(t) for t in (q, k))
    qe, ke = apply_multi_axis_rotary(q, k, pos, inv, sections, interleaved)
    plain = apply_multi_axis_rotary(q.detach(), k.detach(), pos, inv, sections, interleaved)
    assert torch.equal(qe, plain[0]) and torch.equal(ke, plain[1])
    dq, dk = torch.autograd.grad((qe, ke), (q, k), (gq, gk), retain_graph=True)
    for d, g in ((dq, gq), (dk, gk)):
        _close(d, g, _exact(g, pos, inv, sections, interleaved, back=True), half)
    # one of the two outputs unused, and a gradient broadcast over heads
    one, = torch.autograd.grad(qe, q, gq, retain_graph=True)
    assert torch.equal(one, dq)
    wide = gk[:, :1].expand_as(gk)
    one, = torch.autograd.grad(ke, k, wide, retain_graph=True)
    _close(one, wide, _exact(wide, pos, inv, sections, interleaved, back=True), half)
    # only k wants one
    _, ke = apply_multi_axis_rotary(q.detach(), k, pos, inv, sections, interleaved)
    assert torch.equal(torch.autograd.grad(ke, k, gk)[0], dk)


def test_gradient_against_differences(cuda_device):
    """<g, f(x + d) - f(x - d)> / 2 = <df, d>, the inputs shared by heads (one head expanded to four)."""
    q, k, pos, inv = _inputs(cuda_device, 21, 1, 1, 24, 8, 2, torch.float32, far=1000)
    base = q.clone().requires_grad_()
    g, d = torch.randn(21, 4, 24, device=cuda_device), torch.randn_like(q)
    f = lambda x: apply_multi_axis_rotary(x.expand(21, 4, 24), k, pos, inv, [5, 3], True)[0]
    dx, = torch.autograd.grad(f(base), base, g)
    with torch.no_grad():
        up, down = f(q + d).double(), f(q - d).double()
    left = (g.double() * (up - down)).sum() / 2
    right = (dx.double() * d.double()).sum()
    # 2^-22 (|lo| + |hi|) and one rounding per value on the left, the same with a sum over four heads on the right
    bound = 2.0 ** -20 * (g.abs().double() * ((q.abs() + d.abs()).amax() * 4)).sum()
    assert abs(left - right) <= bound


def test_second_derivative(cuda_device):
    """The map is linear: the gradient's own derivative by the incoming gradient is the forward rotation."""
    q, k, pos, inv = _inputs(cuda_device, 6, 2, 1, 16, 8, 2, torch.float32)
    q.requires_grad_()
    g = torch.randn_like(q).requires_grad_()
    qe, _ = apply_multi_axis_rotary(q, k, pos, inv, [4, 4])
    dq, = torch.autograd.grad(qe, q, g, create_graph=True)
    v = torch.randn_like(q)
    dg, = torch.autograd.grad(dq, g, v)
    assert torch.equal(dg, apply_multi_axis_rotary(v, k, pos, inv, [4, 4])[0])


def test_other_stream_and_graph(cuda_device):
    q, k, pos, inv = _inputs(cuda_device, 40, 4, 2, 64, 32, 3, torch.bfloat16)
    ref = apply_multi_axis_rotary(q, k, pos, inv, [16, 8, 8])
    qe, ke = torch.empty_like(q), torch.empty_like(k)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        apply_multi_axis_rotary(q, k, pos, inv, [16, 8, 8], q_embed=qe, k_embed=ke)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(qe, ref[0]) and torch.equal(ke, ref[1])
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        apply_multi_axis_rotary(q, k, pos, inv, [16, 8, 8], q_embed=qe, k_embed=ke)
    pos += 17
    qe.zero_()
    graph.replay()
    assert torch.equal(qe, apply_multi_axis_rotary(q, k, pos, inv, [16, 8, 8])[0])


@pytest.mark.parametrize("idx,far", [(torch.int32, 2 ** 31 - 1), (torch.int64, 2 ** 31), (torch.int64, 2 ** 40 + 12345),
                                     (torch.int64, 2 ** 53 - 1)])
def test_positions_far_out(cuda_device, idx, far):
    """Angles from whole numbers and fractions: position x frequency (each exact) x 1 / 2 pi to 60 digits, whole turns dropped."""
    turn = Fraction("0.159154943091895335768883763372514362034459645740456448747667")
    q, k, pos, inv = _inputs(cuda_device, 24, 2, 1, 32, 16, 1, torch.float32)
    pos = torch.tensor([[(far - i * (far // 1000)) * (-1) ** i for i in range(24)]], dtype=idx, device=cuda_device)
    inv[3:6] = torch.tensor([1.9999998, 1.0 / 3, 1000.123])
    angles = []
    for p in pos[0].tolist():
        turns = [p * Fraction(f) * turn for f in inv.tolist()]
        angles.append([2 * math.pi * float(t - round(t)) for t in turns])
    angle = torch.tensor(angles, dtype=torch.float64, device=cuda_device)[:, None]
    for out, x in zip(apply_multi_axis_rotary(q, k, pos, inv, [16]), (q, k)):
        lo, hi = x.double().chunk(2, -1)
        _close(out, x, torch.cat([lo * angle.cos() - hi * angle.sin(), hi * angle.cos() + lo * angle.sin()], -1), 16)


@pytest.mark.parametrize("dtype,dim,half", [(torch.bfloat16, 64, 32), (torch.float32, 13, 4)])
def test_forward_mode(cuda_device, dtype, dim, half):
    """The map is linear: an output's tangent is the rotation of the input's, an input without one gives none."""
    q, k, pos, inv = _inputs(cuda_device, 11, 4, 2, dim, half, 2, dtype)
    sections, (tq, tk) = [half // 2, half - half // 2], (torch.randn_like(t) for t in (q, k))
    plain, turned = (apply_multi_axis_rotary(a, b, pos, inv, sections) for a, b in ((q, k), (tq, tk)))
    for wants in (False, True):
        with fwAD.dual_level():
            for with_q, with_k in ((True, True), (True, False), (False, True)):
                a = fwAD.make_dual(q.clone().requires_grad_(wants), tq) if with_q else q
                b = fwAD.make_dual(k.clone().requires_grad_(wants), tk) if with_k else k
                for out, value, tangent, has in zip(apply_multi_axis_rotary(a, b, pos, inv, sections), plain, turned, (with_q, with_k)):
                    out = fwAD.unpack_dual(out)
                    assert torch.equal(out.primal, value)
                    if has:
                        assert torch.equal(out.tangent, tangent)
                    else:
                        assert out.tangent is None or not out.tangent.any()
            with torch.no_grad():
                out, _ = apply_multi_axis_rotary(fwAD.make_dual(q, tq), k, pos, inv, sections)
                assert torch.equal(fwAD.unpack_dual(out).tangent, turned[0])


def test_forward_mode_of_the_gradient(cuda_device):
    """The gradient is linear in the incoming one: its tangent is turned back."""
    q, k, pos, inv = _inputs(cuda_device, 11, 4, 2, 16, 8, 2, torch.float32)
    q.requires_grad_()
    g, tg = torch.randn_like(q), torch.randn_like(q)
    back, = torch.autograd.grad(apply_multi_axis_rotary(q, k, pos, inv, [4, 4])[0], q, tg)
    for create in (False, True):
        with fwAD.dual_level():
            out, _ = apply_multi_axis_rotary(q, k, pos, inv, [4, 4])
            dq, = torch.autograd.grad(out, q, fwAD.make_dual(g, tg), create_graph=create)
            assert torch.equal(fwAD.unpack_dual(dq).tangent, back)


def test_forward_mode_refusals(cuda_device):
    """A tangent that would be lost: into given outputs, and of the frequencies."""
    q, k, pos, inv = _inputs(cuda_device, 3, 2, 1, 16, 8, 1, torch.float32)
    with fwAD.dual_level():
        with pytest.raises(AssertionError, match="outputs"):
            apply_multi_axis_rotary(fwAD.make_dual(q, q), k, pos, inv, [8], q_embed=torch.empty_like(q))
        with pytest.raises(AssertionError, match="inv_freq"):
            apply_multi_axis_rotary(q, k, pos, fwAD.make_dual(inv, inv), [8])


def test_training_step_in_a_graph(cuda_device):
    """Forward and backward captured together and replayed with other inputs, positions and incoming gradients."""
    q, k, pos, inv = _inputs(cuda_device, 40, 4, 2, 64, 32, 3, torch.bfloat16)
    q.requires_grad_(), k.requires_grad_()
    gq, gk = (torch.randn_like(t) for t in (q, k))

    def step():
        qe, ke = apply_multi_axis_rotary(q, k, pos, inv, [16, 8, 8])
        return (qe, ke) + torch.autograd.grad((qe, ke), (q, k), (gq, gk))

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        outs = step()
    with torch.no_grad():
        pos += 17
        q.mul_(-2), gk.mul_(3)
    graph.replay()
    assert all(torch.equal(a, b) for a, b in zip(outs, step()))
