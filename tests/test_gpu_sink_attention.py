"""GPU: paged attention with a sliding window and sinks against 64 bits, in the form for single tokens and the one for
several, with everything that no query sees poisoned."""
import pytest
import torch

import dlcompiler_b200 as dl
from dlcompiler_b200 import check_device_status, paged_attention_fwd, sink_attention_fwd
from dlcompiler_b200._lib import DlblasError
from tests.paged_reference import attend, close, rows_of

pytestmark = pytest.mark.gpu
BF, FP = torch.bfloat16, torch.float16


class Batch:
    """A paged cache for sequences of `new` tokens after `past` ones, pages in random order.  Keys and values that no query
    of their sequence sees are NaN, the pages that hold nothing else are -1 in the table."""

    def __init__(self, dev, new, past, window, sinks, page=16, hq=8, hkv=2, d=64, dv=None, dtype=BF, idx=torch.int32,
                 seed=0, poison=True, head_first=False):
        g = torch.Generator().manual_seed(seed + 1000 * len(new) + sum(new) + window)
        dv = dv or d
        self.new, self.past, self.window, self.sinks, self.page, self.d = new, past, window, sinks, page, d
        full = [a + b for a, b in zip(new, past)]
        need = [max(-(-n // page), 1) for n in full]
        total = sum(need) + 3
        perm = torch.randperm(total, generator=g)
        self.q = torch.randn(sum(new), hq, d, generator=g).to(dtype).to(dev)
        k = torch.randn(total * page, hkv, d, generator=g).to(dtype)
        v = torch.randn(total * page, hkv, dv, generator=g).to(dtype)
        visible = torch.zeros(total * page, dtype=torch.bool)
        self.table = torch.zeros(len(new), max(need) + 1, dtype=torch.int64) - 1
        at = 0
        for b, n in enumerate(need):
            self.table[b, :n] = perm[at:at + n]
            at += n
            if new[b]:
                seen = self.seen(b).any(0)
                visible[rows_of(self.table[b], full[b], page)] = seen
                if poison:
                    for c in range(n):
                        if not seen[c * page:(c + 1) * page].any():
                            self.table[b, c] = -1 if c % 2 else 2 ** 30
        self.clean = self.table.clamp(0, total - 1)
        if poison:
            k[~visible], v[~visible] = float("nan"), float("nan")
        k, v = k.view(total, page, hkv, d).to(dev), v.view(total, page, hkv, dv).to(dev)
        if head_first:
            k, v = (t.transpose(1, 2).contiguous().transpose(1, 2) for t in (k, v))
        self.k, self.v = k, v
        self.table, self.clean = self.table.to(idx).to(dev), self.clean.to(dev)
        starts, s = [], 0
        for n in new:
            starts.append(s)
            s += n
        self.start, self.lens, self.kv = (torch.tensor(x, dtype=idx, device=dev) for x in (starts, new, full))
        self.o = torch.full((sum(new), hq, dv), 7.0, dtype=dtype, device=dev)

    def seen(self, b, dev="cpu"):
        n, past = self.new[b], self.past[b]
        pos, key = torch.arange(past, past + n, device=dev)[:, None], torch.arange(past + n, device=dev)
        return (key <= pos) & ((key >= pos - self.window) | (key < self.sinks))

    def run(self, scale=None, cap=None, most=None, o=None, q=None):
        return sink_attention_fwd(self.q if q is None else q, self.k, self.v, self.o if o is None else o, self.table,
                                  self.start, self.lens, self.kv, max(self.new) if most is None else most, self.window,
                                  self.sinks, scale, cap)

    def check(self, o, scale=None, cap=0.0):
        at, scale = 0, scale or self.d ** -0.5
        hkv = self.k.size(2)
        k, v = (t.reshape(-1, hkv, t.size(3)) for t in (self.k, self.v))
        for b, (n, past) in enumerate(zip(self.new, self.past)):
            if n == 0:
                continue
            rows = rows_of(self.clean[b], n + past, self.page)
            ref, bound = attend(self.q[at:at + n], k[rows], v[rows], self.seen(b, self.q.device), scale, cap, o.dtype)
            close(o[at:at + n], ref, bound, f"sequence {b}")
            at += n


ONE = [  # past, window, sinks, page, hq, hkv, d, dv, dtype, cap
    ([0], 0, 0, 16, 1, 1, 8, 8, BF, 0.0),
    ([0, 1, 15, 16, 17, 62, 63, 64, 65, 127, 128, 200], 63, 4, 16, 8, 2, 64, 64, FP, 0.0),
    ([5, 900, 1023, 1024, 1025, 3000], 1000, 17, 16, 28, 4, 128, 128, BF, 0.0),
    ([5, 900, 3000], 1, 64, 64, 32, 8, 128, 128, FP, 30.0),
    ([4100, 3, 77], 4095, 100, 32, 24, 8, 96, 80, BF, 0.0),
    ([700, 12], 64, 0, 128, 16, 16, 128, 64, FP, 0.0),
    ([2222], 129, 1, 256, 40, 1, 40, 128, BF, 20.0),
    ([333, 50], 5000, 8, 16, 34, 2, 72, 8, FP, 0.0),
    ([999], 0, 1000, 64, 4, 4, 128, 128, BF, 0.0),
    ([130, 70, 64], 0, 3, 64, 128, 1, 64, 64, BF, 0.0),
    ([20000], 16384, 4, 64, 8, 1, 128, 128, BF, 0.0),
]


@pytest.mark.parametrize("past,window,sinks,page,hq,hkv,d,dv,dtype,cap", ONE)
@pytest.mark.parametrize("idx", [torch.int32, torch.int64])
def test_single_tokens(cuda_device, past, window, sinks, page, hq, hkv, d, dv, dtype, cap, idx):
    b = Batch(cuda_device, [1] * len(past), past, window, sinks, page, hq, hkv, d, dv, dtype, idx)
    o = b.run(cap=cap or None)
    b.check(o, cap=cap)
    check_device_status()


@pytest.mark.parametrize("past,window,sinks,page,hq,hkv,d,dv,dtype,cap", ONE)
def test_single_tokens_in_the_form_for_several(cuda_device, past, window, sinks, page, hq, hkv, d, dv, dtype, cap):
    b = Batch(cuda_device, [1] * len(past), past, window, sinks, page, hq, hkv, d, dv, dtype)
    b.check(b.run(cap=cap or None, most=2), cap=cap)


SEVERAL = [  # new, past, window, sinks, page, hq, hkv, d, dv, dtype, cap
    ([2], [0], 0, 0, 16, 1, 1, 8, 8, BF, 0.0),
    ([5, 3, 1, 4], [70, 0, 400, 63], 50, 4, 16, 28, 4, 128, 128, FP, 0.0),
    ([33, 64, 65, 128, 129], [0, 1, 64, 200, 31], 64, 16, 16, 8, 8, 64, 64, BF, 0.0),
    ([300, 1, 77], [0, 1000, 513], 127, 130, 64, 24, 8, 96, 80, BF, 30.0),
    ([257], [0], 1000, 4, 32, 4, 1, 128, 128, FP, 0.0),
    ([400], [321], 31, 70, 128, 6, 2, 128, 64, BF, 0.0),
    ([31], [900], 300, 1, 256, 128, 1, 64, 128, FP, 0.0),
    ([40], [90], 17, 3, 16, 100, 1, 40, 48, BF, 15.0),
    ([7] * 40, [13 * i for i in range(40)], 100, 5, 16, 4, 2, 64, 64, BF, 0.0),
    ([(5 * i) % 4 for i in range(301)], [7 * i % 90 for i in range(301)], 40, 5, 16, 4, 2, 64, 64, BF, 0.0),
    ([1500], [0], 700, 4, 64, 8, 2, 128, 128, BF, 0.0),
    ([5, 2, 9], [5000, 700, 0], 4095, 4, 16, 28, 4, 128, 128, FP, 0.0),
    ([3], [2500], 1023, 70, 64, 4, 4, 64, 64, BF, 20.0),
    ([2500, 1, 2400], [0, 30, 333], 300, 4, 64, 8, 8, 64, 64, BF, 0.0),
    ([700, 19, 691], [1000, 0, 5], 200, 70, 16, 28, 4, 128, 128, FP, 25.0),
    ([3, 200], [50, 3], 5000, 10 ** 6, 64, 8, 2, 128, 128, BF, 0.0),
]


@pytest.mark.parametrize("new,past,window,sinks,page,hq,hkv,d,dv,dtype,cap", SEVERAL)
@pytest.mark.parametrize("idx", [torch.int32, torch.int64])
def test_several_tokens(cuda_device, new, past, window, sinks, page, hq, hkv, d, dv, dtype, cap, idx):
    b = Batch(cuda_device, new, past, window, sinks, page, hq, hkv, d, dv, dtype, idx)
    o = b.run(cap=cap or None)
    b.check(o, cap=cap)
    check_device_status()


@pytest.mark.parametrize("most", [1, 6])
def test_sequences_without_tokens_and_rows_of_nobody(cuda_device, most):
    """Empty sequences are passed over, rows between and behind the sequences keep what they hold."""
    new = [1, 0, 1, 0, 1] if most == 1 else [3, 0, 6, 0, 2]
    b = Batch(cuda_device, new, [40, 300, 0, 7, 99], 30, 4)
    gap = 2
    starts = [0, 50, new[0] + gap, -3, new[0] + new[2] + 2 * gap]
    total = sum(new) + 3 * gap
    q = torch.full((total, 8, 64), float("nan"), dtype=BF, device=cuda_device)
    o = torch.full((total, 8, 64), 7.0, dtype=BF, device=cuda_device)
    at, mine = 0, torch.zeros(total, dtype=torch.bool, device=cuda_device)
    for n, s in zip(new, starts):
        if n:
            q[s:s + n] = b.q[at:at + n]
            mine[s:s + n] = True
            at += n
    b.start = torch.tensor(starts, dtype=torch.int32, device=cuda_device)
    b.run(o=o, q=q, most=most)
    b.check(o[mine])
    assert (o[~mine] == 7).all()


@pytest.mark.parametrize("most", [1, 4])
def test_cache_shorter_than_the_new_tokens(cuda_device, most):
    """kv_seqlens below q_seqlens: the first tokens lie before the cache and see nothing, so they get zeros."""
    new = [1, 1] if most == 1 else [4, 2]
    b = Batch(cuda_device, new, [0, 0], 30, 4, poison=False)
    b.kv = torch.zeros(2, dtype=torch.int32, device=cuda_device)
    assert not b.run(most=most).any()


@pytest.mark.parametrize("new", [[1, 1, 1], [9, 150, 4]])
def test_layouts(cuda_device, new):
    """Views of a fused projection, rows that cannot be fetched as they are, strided outputs, caches with the heads outside
    the slots, a table that is a view: the bits of the plain call, nothing beside the output written."""
    b = Batch(cuda_device, new, [333, 20, 65], 100, 20, d=64, seed=3)
    ref = b.run().clone()
    total = sum(new)
    fused = torch.cat([b.q.flatten(1), torch.zeros(total, 256, dtype=BF, device=cuda_device)], 1)
    odd = torch.zeros(total, 8, 65, dtype=BF, device=cuda_device)
    odd[..., 1:] = b.q
    turned = b.q.transpose(1, 2).contiguous().transpose(1, 2)
    for q in (fused[:, :512].view(total, 8, 64), odd[..., 1:], turned):
        assert torch.equal(b.run(q=q, o=torch.empty_like(b.q)), ref)
    canvas = torch.full((total + 2, 10, 72), 7.0, dtype=BF, device=cuda_device)
    b.run(o=canvas[1:-1, 1:9, :64])
    assert torch.equal(canvas[1:-1, 1:9, :64], ref)
    canvas[1:-1, 1:9, :64] = 7
    assert (canvas == 7).all()
    b.table = torch.stack([b.table, b.table * 0], -1)[..., 0]
    assert torch.equal(b.run(), ref)
    h = Batch(cuda_device, new, [333, 20, 65], 100, 20, d=64, seed=3, head_first=True)
    assert h.k.stride(2) > h.k.stride(1) and torch.equal(h.run(), ref)


@pytest.mark.parametrize("new,past", [([1, 1, 1], [100, 40, 0]), ([90, 5, 17], [100, 40, 0])])
def test_wide_window_is_plain_attention(cuda_device, new, past):
    """A window past every context: what paged_attention_fwd computes, within both bounds; and its window without sinks."""
    for window, plain in ((10 ** 6, None), (25, 25)):
        b = Batch(cuda_device, new, past, window, 0)
        b.table = b.clean.int()
        if plain:
            b.k, b.v = b.k.nan_to_num(0.0), b.v.nan_to_num(0.0)
        o, other = b.run(), torch.empty_like(b.o)
        paged_attention_fwd(b.q, b.k.nan_to_num(0.0), b.v.nan_to_num(0.0), other, b.table, b.start, b.lens, b.kv, max(new),
                            window_size=plain)
        b.check(o)
        b.check(other)


@pytest.mark.parametrize("most", [1, 3])
def test_page_outside_the_cache(cuda_device, most):
    """Where a visible token should be: an error for the call, the other sequences as without it."""
    b = Batch(cuda_device, [most] * 3, [100, 120, 140], 64, 4, poison=False)
    ref = b.run().clone()
    check_device_status()
    for bad in (-1, b.k.size(0), 2 ** 31 - 1):
        table = b.table.clone()
        b.table[1, 6] = bad
        o = b.run(o=torch.empty_like(b.o))
        with pytest.raises(DlblasError, match=f"row 1, column 6 .* page {bad},"):
            check_device_status()
        check_device_status()
        assert torch.equal(o[:most], ref[:most]) and torch.equal(o[2 * most:], ref[2 * most:])
        b.table = table


@pytest.mark.parametrize("most", [1, 3])
def test_64_bit_indices_past_32_bits(cuda_device, most):
    """A page 2^32 is not page 0, nor a row or a length of that size one of 0."""
    b = Batch(cuda_device, [most] * 3, [100, 120, 140], 64, 4, idx=torch.int64, poison=False)
    ref = b.run().clone()
    b.table[1, 6] = 2 ** 32
    b.run(o=torch.empty_like(b.o))
    with pytest.raises(DlblasError, match=f"row 1, column 6 .* page {2 ** 31 - 1},"):
        check_device_status()
    b.table[1, 6] = -2 ** 32
    b.run(o=torch.empty_like(b.o))
    with pytest.raises(DlblasError, match=f"row 1, column 6 .* page {-2 ** 31},"):
        check_device_status()
    b.table = b.clean
    for far in (2 ** 32, 2 ** 32 + most, -2 ** 32):
        start = b.start
        b.start = start.clone()
        b.start[1] = far
        o = b.run(o=torch.full_like(b.o, 7.0))
        assert (o[most:2 * most] == 7).all() and torch.equal(o[:most], ref[:most]) and torch.equal(o[2 * most:], ref[2 * most:])
        b.start = start
    b.kv = b.kv.clone()
    b.kv[1] = -2 ** 32 + 100
    assert not b.run(o=torch.empty_like(b.o))[most:2 * most].any()
    check_device_status()


@pytest.mark.parametrize("most", [1, 40])
def test_graph_streams_and_repeats(cuda_device, most):
    """The same bits every time, on another stream, and from a graph replayed with other lengths."""
    b = Batch(cuda_device, [most] * 6, [10, 500, 90, 1000, 64, 3], 200, 4, poison=False)
    ref = b.run().clone()
    for _ in range(3):
        assert torch.equal(b.run(), ref)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    o = torch.empty_like(b.o)
    with torch.cuda.stream(side):
        b.run(o=o)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(o, ref)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        b.run(o=o)
    b.kv -= 3
    o.zero_()
    graph.replay()
    assert torch.equal(o, b.run()) and not torch.equal(o, ref)


@pytest.mark.parametrize("most", [1, 3])
def test_cache_past_2_31_elements(cuda_device, most):
    pages, page, hkv, d = 140000, 16, 8, 128                        # 2.3e9 elements
    k, v = (torch.empty(pages, page, hkv, d, dtype=BF, device=cuda_device) for _ in range(2))
    b = Batch(cuda_device, [most, most], [100, 700], 300, 4, hq=16, hkv=8, d=128, poison=False)
    far = pages - 1 - torch.arange(b.k.size(0), device=cuda_device) * 7
    k[far], v[far] = b.k, b.v
    ref = b.run().clone()
    b.table = far[b.clean.long()].int()
    b.k, b.v = k, v
    assert torch.equal(b.run(), ref)


def test_large_scores_and_infinite_values_behind_the_window(cuda_device):
    """Scores of +-100 (a maximum that grows and falls), -inf and the type's lowest value where nobody looks."""
    for new in ([1, 1], [70, 3]):
        b = Batch(cuda_device, new, [500, 300], 150, 5, dtype=FP, poison=False)
        b.q *= 12
        hidden = rows_of(b.clean[0], 300, 16)[5:]
        flat_k, flat_v = b.k.view(-1, 2, 64), b.v.view(-1, 2, 64)
        flat_k[hidden], flat_v[hidden] = float("-inf"), torch.finfo(FP).min
        b.check(b.run())
        b.check(b.run(cap=20.0), cap=20.0)                   # scores on both sides of the cap


@pytest.mark.parametrize("new", [[1, 1], [70, 3]])
@pytest.mark.parametrize("size", [-12.0, -1.0, -0.05, 0.0, 0.05, 1.0, 12.0])
def test_scores_of_one_sign(cuda_device, new, size):
    """All scores of a row far below zero (about -60, -5, -0.3) or above: the reference that P is taken against has to follow."""
    b = Batch(cuda_device, new, [500, 300], 150, 5, dtype=FP, poison=False)
    b.q, b.k = b.q.abs() * size, b.k.abs()
    b.check(b.run())


@pytest.mark.parametrize("new", [[1, 1, 1], [70, 3, 20]])
@pytest.mark.parametrize("cap", [1e6, 1e30, float("inf")])
def test_cap_far_above_the_scores(cuda_device, new, cap):
    """Takes off x^2 / 3 of a score, x its size over the cap: nothing here (10^-10 of it at most)."""
    b = Batch(cuda_device, new, [500, 30, 1], 150, 5)
    b.check(b.run(cap=cap))


@pytest.mark.parametrize("new", [[1, 1, 1], [70, 3, 20]])
@pytest.mark.parametrize("cap", [0.0, 30.0])
def test_no_numbers_in_visible_places(cuda_device, new, cap):
    """A head of q that is no number: its row of the output is none either, the others are as without it.  A key that is no
    number: so are the queries that see it, and no other."""
    b = Batch(cuda_device, new, [500, 30, 1], 150, 5, poison=False)
    q = b.q.clone()
    for t, h in ((0, 0), (0, 5), (sum(new) - 1, 7)):
        q[t, h, 3] = float("nan")
    o = b.run(cap=cap or None, q=q)
    lost = q.isnan().any(-1)
    assert o[lost].isnan().all()
    o[lost] = b.run(cap=cap or None, o=torch.empty_like(b.o))[lost]
    b.check(o, cap=cap)

    whole = b.run(cap=cap or None, o=torch.empty_like(b.o))
    at = 0
    for s, past in enumerate(b.past):
        b.k.view(-1, 2, 64)[rows_of(b.clean[s], past + 1, 16)[-1], 1] = float("nan")      # the first new token
    o = b.run(cap=cap or None)
    for s, (n, past) in enumerate(zip(new, b.past)):
        sees = b.seen(s, cuda_device)[:, past]
        assert sees[0] and o[at:at + n][sees, 4:].isnan().all()
        assert not o[at:at + n, :4].isnan().any() and not o[at:at + n][~sees].isnan().any()
        at += n
    keep = ~o.isnan()
    # two results of the same scores, each off by a rounding of P and one of the output
    assert (o[keep].float() - whole[keep].float()).abs().max() <= 2 * 2 * 2 ** -8 * b.v.abs().max()


def test_empty_calls(cuda_device):
    b = Batch(cuda_device, [2], [10], 5, 1)
    e = b.q[:0]
    out = sink_attention_fwd(e, b.k, b.v, e.clone(), b.table[:0], b.start[:0], b.lens[:0], b.kv[:0], 0, 5, 1)
    assert out.shape == e.shape
    b.o.fill_(7)
    b.run(most=0)
    assert (b.o == 7).all() and dl.is_built()


@pytest.mark.parametrize("value", [float("nan"), float("inf")])
@pytest.mark.parametrize("hq,past", [(43, 1), (48, 1), (65, 0), (71, 0), (96, 5)])
def test_no_number_behind_a_tile(cuda_device, hq, past, value):
    """43 to 48 or 65 to 96 q-heads to a kv head leave the last warp of a tile without rows.  The token after a tile, at the end of
    a block of 64 keys, is fetched with it and seen by nobody there: its values change no bit of the rows in front."""
    b = Batch(cuda_device, [70], [past], 1000, 4, hq=hq, hkv=1, poison=False)
    ref = b.run().clone()
    b.v.view(-1, 1, 64)[rows_of(b.clean[0], 64, 16)[63]] = value
    o = b.run(o=torch.empty_like(b.o))
    assert torch.equal(o[:63 - past], ref[:63 - past]) and not o[63 - past:].isfinite().any()


@pytest.mark.parametrize("page", [16, 64])
def test_sequences_past_max_seqlen(cuda_device, page):
    """Tiles as for two tokens, half of whose warps have no rows, and a sequence of 200; what lies in shared memory from the call
    before, here no numbers, is nobody's value."""
    b = Batch(cuda_device, [200, 7, 90], [40, 0, 13], 1000, 4, page=page, hq=4, hkv=4)
    v = b.v
    b.v = torch.full_like(v, float("nan"))
    assert b.run(most=2).isnan().all()
    b.v = v
    b.check(b.run(most=2))


@pytest.mark.parametrize("most", [1, 3])
@pytest.mark.parametrize("window,sinks", [(40, 5), (40, 0), (33, 70), (0, 100)])
def test_lengths_past_the_table(cuda_device, most, window, sinks):
    """A query keeps its position, and the tokens that the table has no room for are not there, in both forms."""
    b = Batch(cuda_device, [most] * 5, [60, 93, 130, 200, 400], window, sinks, poison=False)
    b.table = b.clean[:, :6].int()
    o, k, v = b.run(), b.k.view(-1, 2, 64), b.v.view(-1, 2, 64)
    for s in range(5):
        n = min(b.past[s] + most, 96)
        rows = rows_of(b.clean[s], n, 16)
        ref, bound = attend(b.q[s * most:(s + 1) * most], k[rows], v[rows], b.seen(s, cuda_device)[:, :n], 64 ** -0.5, 0.0, BF)
        close(o[s * most:(s + 1) * most], ref, bound, f"sequence {s}")


def test_first_token_of_a_sequence_before_the_cache(cuda_device):
    """max_seqlen 1 and sequences of two tokens: a length far below zero has no key."""
    b = Batch(cuda_device, [2, 2], [40, 50], 30, 4, idx=torch.int64, poison=False)
    b.kv[1] = -2 ** 40
    o = b.run(most=1)
    assert not o[2].any() and (o[[1, 3]] == 7).all() and o[0].any()


@pytest.mark.parametrize("most", [1, 3])
def test_window_past_2_30(cuda_device, most):
    """Positions past 2^30 over a table of 112 tokens: the window is not cut short."""
    b = Batch(cuda_device, [most] * 2, [100, 90], 0, 3, poison=False)
    for window in (2 ** 30 + 180, 2 ** 31 - 1):
        b.window = window
        b.kv = torch.tensor([min(window + n, 2 ** 31 - 1) for n in (20, 60)], dtype=torch.int32, device=cuda_device)
        b.table = b.clean.int()[:, :6]
        o = b.run(o=torch.empty_like(b.o))
        k, v = b.k.view(-1, 2, 64), b.v.view(-1, 2, 64)
        for s, kv in enumerate(b.kv.tolist()):
            pos, key = torch.arange(kv - most, kv, device=cuda_device)[:, None], torch.arange(96, device=cuda_device)
            rows = rows_of(b.clean[s], 96, 16)
            ref, bound = attend(b.q[s * most:(s + 1) * most], k[rows], v[rows], (key >= pos - window) | (key < 3), 64 ** -0.5, 0.0, BF)
            close(o[s * most:(s + 1) * most], ref, bound, f"window {window}, sequence {s}")
