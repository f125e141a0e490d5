"""GPU: decode attention of groups that share a prefix against 64 bits, with everything that no token sees poisoned."""
import pytest
import torch

from dlcompiler_b200 import check_device_status, paged_attention_fwd, shared_prefix_attention_fwd
from dlcompiler_b200._lib import DlblasError
from tests.paged_reference import attend, close, rows_of

pytestmark = pytest.mark.gpu
BF, FP = torch.bfloat16, torch.float16


class Groups:
    def __init__(self, dev, members, prefix, own, page=16, hq=8, hkv=2, d=64, dv=None, dtype=BF, idx=torch.int32, seed=0,
                 poison=True, room=0):
        g = torch.Generator().manual_seed(seed + sum(own) * 17 + sum(prefix))
        dv = dv or d
        batch = sum(members)
        assert len(own) == batch
        self.members, self.prefix, self.own, self.page, self.d = members, prefix, own, page, d
        need = [[max(-(-n // page), 0) for n in x] for x in (prefix, own)]
        total = sum(map(sum, need)) + 2
        perm, at = torch.randperm(total, generator=g), 0
        tables = []
        for n in need:
            t = torch.full((len(n), max(max(n), 1) + room), -1 if poison else 0, dtype=torch.int64)
            for i, m in enumerate(n):
                t[i, :m] = perm[at:at + m]
                at += m
            tables.append(t)
        self.q = torch.randn(batch, hq, d, generator=g).to(dtype).to(dev)
        k, v = torch.randn(total * page, hkv, d, generator=g).to(dtype), torch.randn(total * page, hkv, dv, generator=g).to(dtype)
        if poison:
            live = torch.cat([rows_of(t[i], n, page) for t, ns in zip(tables, (prefix, own)) for i, n in enumerate(ns)])
            dead = torch.ones(total * page, dtype=torch.bool)
            dead[live] = False
            k[dead], v[dead] = float("nan"), float("nan")
        self.k, self.v = k.view(total, page, hkv, d).to(dev), v.view(total, page, hkv, dv).to(dev)
        starts = [0]
        for m in members:
            starts.append(starts[-1] + m)
        self.starts = starts
        to = lambda x: torch.as_tensor(x).to(idx).to(dev)
        self.prefix_table, self.table = to(tables[0]), to(tables[1])
        self.prefix_lens, self.lens, self.group_start = to(prefix), to(own), to(starts)
        self.o = torch.full((batch, hq, dv), 7.0, dtype=dtype, device=dev)

    def run(self, scale=None, cap=None, o=None, q=None):
        return shared_prefix_attention_fwd(self.q if q is None else q, self.k, self.v, self.o if o is None else o,
                                           self.prefix_table, self.prefix_lens, self.group_start, self.table, self.lens,
                                           scale, cap)

    def check(self, o, cap=0.0):
        hkv = self.k.size(2)
        k, v = (t.reshape(-1, hkv, t.size(3)) for t in (self.k, self.v))
        for g, m in enumerate(self.members):
            first = rows_of(self.prefix_table[g], self.prefix[g], self.page)
            for b in range(self.starts[g], self.starts[g] + m):
                rows = torch.cat([first, rows_of(self.table[b], self.own[b], self.page)])
                seen = torch.ones(1, rows.numel(), dtype=torch.bool, device=o.device)
                if rows.numel() == 0:
                    assert not o[b].any()
                    continue
                ref, bound = attend(self.q[b:b + 1], k[rows], v[rows], seen, self.d ** -0.5, cap, o.dtype)
                close(o[b:b + 1], ref, bound, f"sequence {b} of group {g}")


CASES = [  # members, prefix, own, page, hq, hkv, d, dv, dtype, cap
    ([1], [1], [1], 16, 1, 1, 8, 8, BF, 0.0),
    ([3], [64], [1, 2, 0], 16, 8, 2, 64, 64, FP, 0.0),
    ([33], [1000], list(range(1, 34)), 16, 28, 4, 128, 128, BF, 0.0),
    ([2, 5, 1, 40], [65, 0, 4001, 127], [17 * i % 301 for i in range(48)], 64, 24, 8, 96, 80, FP, 0.0),
    ([70], [2500], [i % 7 for i in range(70)], 32, 8, 8, 128, 64, BF, 30.0),
    ([1, 1, 1], [0, 0, 63], [0, 70, 0], 128, 40, 1, 40, 128, BF, 0.0),
    ([4] * 40, [50 + 3 * i for i in range(40)], [1 + i % 50 for i in range(160)], 16, 4, 2, 64, 64, BF, 0.0),
    ([i % 3 for i in range(150)], [20 + i for i in range(150)], [1 + i % 20 for i in range(150)], 16, 4, 2, 64, 64, BF, 0.0),
    ([3, 2], [300, 200], [900, 5, 2000, 64, 63], 256, 128, 1, 72, 72, FP, 10.0),
    ([2], [40000], [3, 700], 64, 32, 8, 128, 128, BF, 0.0),
    ([150], [700], [5] * 150, 64, 16, 16, 64, 64, FP, 0.0),
]


@pytest.mark.parametrize("members,prefix,own,page,hq,hkv,d,dv,dtype,cap", CASES)
@pytest.mark.parametrize("idx", [torch.int32, torch.int64])
def test_groups(cuda_device, members, prefix, own, page, hq, hkv, d, dv, dtype, cap, idx):
    b = Groups(cuda_device, members, prefix, own, page, hq, hkv, d, dv, dtype, idx)
    b.check(b.run(cap=cap or None), cap=cap)
    check_device_status()


def test_same_as_the_whole_context(cuda_device):
    """A prefix that ends on a page: the table of the whole context through paged_attention_fwd, within both bounds."""
    b = Groups(cuda_device, [6], [320], [1, 30, 64, 65, 200, 16], poison=False)
    o, other = b.run(), torch.empty_like(b.o)
    whole = torch.cat([b.prefix_table.expand(6, -1), b.table], 1)
    one = torch.ones(6, dtype=torch.int32, device=cuda_device)
    paged_attention_fwd(b.q, b.k, b.v, other, whole, one, one, b.lens + 320, 1)
    b.check(o)
    b.check(other)


def test_sequences_outside_the_groups(cuda_device):
    """No prefix for them: their own tokens alone, and zeros where there are none."""
    b = Groups(cuda_device, [2, 3], [300, 100], [5, 80, 3, 0, 40], seed=2)
    b.group_start = torch.tensor([0, 2, 3], dtype=torch.int32, device=cuda_device)
    o = b.run()
    alone = Groups(cuda_device, [2, 1, 2], [300, 100, 0], b.own, seed=2)
    for name in ("q", "k", "v", "table"):
        setattr(alone, name, getattr(b, name))
    alone.prefix_table = torch.cat([b.prefix_table, b.prefix_table[:1]])
    alone.check(o)
    assert not o[3].any()


@pytest.mark.parametrize("starts", [[0, 9, 5], [-4, 2, 100], [3, 1, 5], [5, 5, 5]])
def test_starts_out_of_order_or_range_touch_nothing_else(cuda_device, starts):
    """Rows that no group holds keep their own tokens' result; nothing outside the output is written."""
    b = Groups(cuda_device, [2, 3], [300, 100], [5, 80, 3, 7, 40], poison=False)
    b.group_start = torch.tensor(starts, dtype=torch.int32, device=cuda_device)
    canvas = torch.full((7, 8, 64), 7.0, dtype=BF, device=cuda_device)
    b.run(o=canvas[1:-1])
    assert (canvas[[0, -1]] == 7).all()
    if starts == [5, 5, 5]:
        alone = Groups(cuda_device, [5], [0], b.own, poison=False)
        alone.q, alone.k, alone.v, alone.table = b.q, b.k, b.v, b.table
        alone.check(canvas[1:-1])


def test_lengths_beside_the_tables(cuda_device):
    """Negative lengths count as none, lengths past a table as what it holds."""
    b = Groups(cuda_device, [2, 1], [32, 48], [16, 32, 16], poison=False)
    ref = b.run().clone()
    b.prefix_lens = torch.tensor([32, 10 ** 9], dtype=torch.int32, device=cuda_device)
    b.lens = torch.tensor([16, 10 ** 9, 16], dtype=torch.int32, device=cuda_device)
    assert torch.equal(b.run(), ref)
    b.prefix_lens.fill_(-5)
    b.lens.fill_(-(2 ** 31))
    assert not b.run().any()


def test_layouts(cuda_device):
    b = Groups(cuda_device, [3, 2], [130, 500], [10, 200, 1, 64, 33])
    ref = b.run().clone()
    fused = torch.cat([b.q.flatten(1), torch.zeros(5, 256, dtype=BF, device=cuda_device)], 1)
    odd = torch.zeros(5, 8, 65, dtype=BF, device=cuda_device)
    odd[..., 1:] = b.q
    for q in (fused[:, :512].view(5, 8, 64), odd[..., 1:]):
        assert torch.equal(b.run(q=q, o=torch.empty_like(b.q)), ref)
    canvas = torch.full((7, 10, 72), 7.0, dtype=BF, device=cuda_device)
    b.run(o=canvas[1:-1, 1:9, :64])
    assert torch.equal(canvas[1:-1, 1:9, :64], ref)
    canvas[1:-1, 1:9, :64] = 7
    assert (canvas == 7).all()
    b.k, b.v = (t.transpose(1, 2).contiguous().transpose(1, 2) for t in (b.k, b.v))
    b.table, b.prefix_table = (torch.stack([t, t * 0], -1)[..., 0] for t in (b.table, b.prefix_table))
    assert torch.equal(b.run(), ref)


def test_page_outside_the_cache(cuda_device):
    b = Groups(cuda_device, [2, 2], [100, 200], [20, 40, 60, 80], poison=False)
    ref = b.run().clone()
    check_device_status()
    for table, r, c, other in ((b.prefix_table, 1, 3, slice(0, 2)), (b.table, 2, 1, [0, 1, 3])):
        keep = table.clone()
        for bad in (-7, b.k.size(0)):
            table[r, c] = bad
            o = b.run(o=torch.empty_like(b.o))
            with pytest.raises(DlblasError, match=f"row {r}, column {c} .* page {bad},"):
                check_device_status()
            check_device_status()
            assert torch.equal(o[other], ref[other])
        table.copy_(keep)


def test_graphs_streams_and_repeats(cuda_device):
    """The same bits every time and on another stream; two graphs in one memory pool replayed in turn with other lengths."""
    a = Groups(cuda_device, [9, 4], [900, 2000], [3 + 40 * i for i in range(13)], poison=False, room=1)
    b = Groups(cuda_device, [5], [3000], [5] * 5, poison=False, room=1)
    refs = [x.run().clone() for x in (a, b)]
    for _ in range(3):
        assert torch.equal(a.run(), refs[0])
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        o = a.run(o=torch.empty_like(a.o))
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(o, refs[0])
    torch.cuda.synchronize()
    pool, graphs = torch.cuda.graph_pool_handle(), []
    for x in (a, b):
        graphs.append(torch.cuda.CUDAGraph())
        with torch.cuda.graph(graphs[-1], pool=pool):
            x.run()
    for step in range(2):
        for x, graph in zip((a, b), graphs):
            x.lens += 1
            x.own = [n + 1 for n in x.own]
            x.o.zero_()
            graph.replay()
            got = x.o.clone()
            assert torch.equal(got, x.run())


def test_large_scores(cuda_device):
    b = Groups(cuda_device, [20], [700], list(range(20)), dtype=FP)
    b.q *= 12
    b.check(b.run())
    b.check(b.run(cap=20.0), cap=20.0)                       # scores on both sides of the cap


@pytest.mark.parametrize("size", [-12.0, -0.05, 12.0])
def test_scores_of_one_sign(cuda_device, size):
    b = Groups(cuda_device, [20], [700], list(range(20)), dtype=FP)
    b.q, b.k = b.q.abs() * size, b.k.abs()
    b.check(b.run())


@pytest.mark.parametrize("cap", [None, 20.0, float("inf")])
def test_no_numbers_in_visible_places(cuda_device, cap):
    """Heads of q that are no number, a key of a prefix and one of a sequence: their rows of the output are none either, and no
    other."""
    b = Groups(cuda_device, [7, 5], [700, 65], list(range(12)), poison=False)
    ref = b.run(cap=cap).clone()
    b.q[2, 3, 1] = b.q[11, 0, 0] = float("nan")
    b.k.view(-1, 2, 64)[rows_of(b.prefix_table[1], 65, 16)[64], 1] = float("nan")
    b.k.view(-1, 2, 64)[rows_of(b.table[4], 4, 16)[0], 0] = float("nan")
    lost = torch.zeros(12, 8, dtype=torch.bool, device=cuda_device)
    lost[2, 3] = lost[11, 0] = lost[4, :4] = lost[7:, 4:] = True
    o = b.run(cap=cap, o=torch.empty_like(b.o))
    assert o[lost].isnan().all() and not o[~lost].isnan().any()
    # two results of the same scores, each off by a rounding of P and one of the output
    assert (o[~lost].float() - ref[~lost].float()).abs().max() <= 2 * 2 * 2 ** -8 * b.v.abs().max()
