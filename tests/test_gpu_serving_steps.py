"""GPU: the serving operators together, as a server calls them: rotary positions of several axes for q and k, the keys and
values into the paged cache, attention over it, with a window and sinks or behind a shared prefix."""
import os
import subprocess
import sys

import pytest
import torch

from dlcompiler_b200 import (apply_multi_axis_rotary, check_device_status, fill_kv_cache, paged_attention_fwd,
                             shared_prefix_attention_fwd, sink_attention_fwd)
from tests.paged_reference import attend, close, rows_of

pytestmark = pytest.mark.gpu
HQ, HKV, D, PAGE, SECTIONS = 8, 2, 64, 16, [8, 12, 12]


def _ints(x, dev):
    return torch.tensor(x, dtype=torch.int32, device=dev)


class Server:
    def __init__(self, dev, batch, pages, columns, dtype, seed):
        self.dev, self.g = dev, torch.Generator().manual_seed(seed)
        self.k, self.v = (torch.full((pages, PAGE, HKV, D), float("nan"), dtype=dtype, device=dev) for _ in range(2))
        self.free = torch.randperm(pages, generator=self.g).tolist()
        self.table = torch.full((batch, columns), -1, dtype=torch.int32, device=dev)
        self.inv = (10000.0 ** (-torch.arange(D // 2, dtype=torch.float64) / (D // 2))).float().to(dev)
        self.dtype = dtype

    def need(self, table, row, tokens):
        for c in range(-(-tokens // PAGE)):
            if int(table[row, c]) < 0:
                table[row, c] = self.free.pop()

    def project(self, tokens):
        qkv = torch.randn(tokens, (HQ + 2 * HKV) * D, generator=self.g).to(self.dtype).to(self.dev)
        return [t.view(tokens, -1, D) for t in qkv.split([HQ * D, HKV * D, HKV * D], 1)]

    def rotated(self, q, k, positions):
        return apply_multi_axis_rotary(q, k, positions.to(self.dev), self.inv, SECTIONS)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_prompts_with_images_then_tokens_behind_a_window(cuda_device, dtype):
    """Prompts (a grid of patches between text), drafted tokens and single ones; pages behind the window are given back and
    their entries go stale, so that other sequences' tokens land there."""
    window, sinks, lens = 40, 5, [70, 33, 1]
    s = Server(cuda_device, 3, 24, 12, dtype, 1)
    grid = torch.cartesian_prod(torch.arange(2), torch.arange(4), torch.arange(3)).t()
    done = [0, 0, 0]
    keys, values = [[], [], []], [[], [], []]
    for step, new in enumerate([lens, [4, 2, 3]] + [[1, 1, 1]] * 6):
        total = sum(new)
        q, k, v = s.project(total)
        pos = []
        for b, n in enumerate(new):
            p = (done[b] + torch.arange(n)).repeat(3, 1)
            if step == 0 and n > 40:
                p[:, 5:29] = 5 + grid
            pos.append(p)
            done[b] += n
            s.need(s.table, b, done[b])
        q, k = s.rotated(q, k, torch.cat(pos, 1))
        start = _ints([0, new[0], new[0] + new[1]], s.dev)
        args = (start, _ints(new, s.dev), _ints(done, s.dev), max(new))
        fill_kv_cache(k, v, s.k, s.v, *args, s.table)
        o = torch.empty_like(q)
        sink_attention_fwd(q, s.k, s.v, o, s.table, *args, window, sinks)
        at = 0
        for b, n in enumerate(new):
            keys[b].append(k[at:at + n])
            values[b].append(v[at:at + n])
            kk, vv = torch.cat(keys[b]), torch.cat(values[b])
            row, key = torch.arange(done[b] - n, done[b], device=s.dev)[:, None], torch.arange(done[b], device=s.dev)
            seen = (key <= row) & ((key >= row - window) | (key < sinks))
            ref, bound = attend(q[at:at + n], kk, vv, seen, D ** -0.5, 0.0, dtype)
            close(o[at:at + n], ref, bound, f"step {step}, sequence {b}")
            at += n
            # what no later token sees is given back
            for c in range(-(-sinks // PAGE), (done[b] - window) // PAGE):
                if int(s.table[b, c]) >= 0:
                    s.free.append(int(s.table[b, c]))
                    s.table[b, c] = -1
    check_device_status()


def test_answers_behind_one_prompt_in_a_graph(cuda_device):
    """The prompt once, then a step of all answers captured into a graph and replayed: each like paged_attention_fwd over the
    whole context, whose pages the prompt fills."""
    dtype, prompt, batch, steps = torch.bfloat16, 96, 5, 20
    s = Server(cuda_device, batch, 40, 3, dtype, 2)
    prefix = torch.full((1, prompt // PAGE), -1, dtype=torch.int32, device=s.dev)
    s.need(prefix, 0, prompt)
    for b in range(batch):
        s.need(s.table, b, steps + 1)
    q, k, v = s.project(prompt)
    q, k = s.rotated(q, k, torch.arange(prompt).repeat(3, 1))
    fill_kv_cache(k, v, s.k, s.v, _ints([0], s.dev), _ints([prompt], s.dev), _ints([prompt], s.dev), prompt, prefix)
    qkv = torch.zeros(batch, (HQ + 2 * HKV) * D, dtype=dtype, device=s.dev)
    q, k, v = (t.view(batch, -1, D) for t in qkv.split([HQ * D, HKV * D, HKV * D], 1))
    pos = torch.full((3, batch), prompt, dtype=torch.int64, device=s.dev)
    own, one, start = _ints([1] * batch, s.dev), _ints([1] * batch, s.dev), _ints(list(range(batch)), s.dev)
    plen, groups = _ints([prompt], s.dev), _ints([0, batch], s.dev)
    o = torch.empty(batch, HQ, D, dtype=dtype, device=s.dev)

    def step():
        qr, kr = apply_multi_axis_rotary(q, k, pos, s.inv, SECTIONS)
        fill_kv_cache(kr, v, s.k, s.v, start, one, own, 1, s.table)
        shared_prefix_attention_fwd(qr, s.k, s.v, o, prefix, plen, groups, s.table, own)
        return qr

    s.k.nan_to_num_(0.0), s.v.nan_to_num_(0.0)
    step()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        qr = step()
    whole = torch.cat([prefix.expand(batch, -1), s.table], 1).contiguous()
    other = torch.empty_like(o)
    for t in range(steps):
        qkv.copy_(torch.randn(qkv.shape, generator=s.g).to(dtype))
        own.fill_(t + 1)
        pos.fill_(prompt + t)
        graph.replay()
        got = o.clone()
        assert torch.equal(got, shared_prefix_attention_fwd(qr, s.k, s.v, torch.empty_like(o), prefix, plen, groups, s.table, own))
        paged_attention_fwd(qr, s.k, s.v, other, whole, start, one, own + prompt, 1)
        kk, vv = s.k.view(-1, HKV, D), s.v.view(-1, HKV, D)
        for b in range(batch):
            rows = rows_of(whole[b], prompt + t + 1, PAGE)
            seen = torch.ones(1, rows.numel(), dtype=torch.bool, device=s.dev)
            ref, bound = attend(qr[b:b + 1], kk[rows], vv[rows], seen, D ** -0.5, 0.0, dtype)
            close(got[b:b + 1], ref, bound, f"step {t}, sequence {b}")
            close(other[b:b + 1], ref, bound, f"whole context, step {t}, sequence {b}")
    check_device_status()


@pytest.mark.parametrize("streams", [1, 3])
def test_calls_from_several_threads(cuda_device, streams):
    """Threads that call at the same time, on streams of their own or with their launches mixed on one: the bits of one after
    the other."""
    import threading

    dtype, batch = torch.bfloat16, 6
    servers, refs = [], []
    for seed in range(3):
        s = Server(cuda_device, batch, 60, 8, dtype, 10 + seed)
        s.k.copy_(torch.randn(s.k.shape, generator=s.g)), s.v.copy_(torch.randn(s.v.shape, generator=s.g))
        for b in range(batch):
            s.need(s.table, b, 8 * PAGE)
        s.q = torch.randn(batch, HQ, D, generator=s.g).to(dtype).to(s.dev)
        s.lens, s.start, s.one = _ints([5 + 20 * b for b in range(batch)], s.dev), _ints(range(batch), s.dev), _ints([1] * batch, s.dev)
        servers.append(s)

    def step(s):
        q, _ = s.rotated(s.q, s.q[:, :2], s.lens.long().repeat(3, 1))
        a = sink_attention_fwd(q, s.k, s.v, torch.empty_like(q), s.table, s.start, s.one, s.lens, 1, 31, 4)
        b = sink_attention_fwd(q, s.k, s.v, torch.empty_like(q), s.table, s.start, s.one, s.lens, 2, 31, 4)
        c = shared_prefix_attention_fwd(q, s.k, s.v, torch.empty_like(q), s.table[:2], s.lens[4:], _ints([0, 2, 6], s.dev),
                                        s.table, s.lens)
        return a, b, c

    refs = [step(s) for s in servers]
    torch.cuda.synchronize()
    pool = [torch.cuda.Stream() for _ in range(streams)]
    wrong = []

    def work(i):
        with torch.cuda.stream(pool[i % streams]):
            for _ in range(50):
                got = step(servers[i])
                if not all(torch.equal(x, y) for x, y in zip(got, refs[i])):
                    wrong.append(i)

    threads = [threading.Thread(target=work, args=(i,)) for i in range(3)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not wrong
    check_device_status()


def test_every_thread_gets_through(cuda_device):
    """Threads on streams of their own from a process's first call on; an exception in one of them is a failure."""
    code = """
import threading
from concurrent.futures import ThreadPoolExecutor
import torch
from dlcompiler_b200 import apply_multi_axis_rotary, check_device_status, shared_prefix_attention_fwd, sink_attention_fwd
dev, n = torch.device("cuda:0"), 4
g = torch.Generator().manual_seed(5)
k, v = (torch.randn(30, 16, 2, 64, generator=g).to(torch.bfloat16).to(dev) for _ in range(2))
q = torch.randn(6, 8, 64, generator=g).to(torch.bfloat16).to(dev)
table = torch.randperm(30, generator=g).view(6, 5).int().to(dev)
lens, start, one = (torch.tensor(x, dtype=torch.int32, device=dev) for x in ([5, 17, 33, 48, 70, 79], list(range(6)), [1] * 6))
groups, inv = torch.tensor([0, 2, 6], dtype=torch.int32, device=dev), torch.ones(32, device=dev)
torch.cuda.synchronize()
gate = threading.Barrier(n)

def step():
    a, _ = apply_multi_axis_rotary(q, q[:, :2], lens.long()[None], inv, [32])
    b = sink_attention_fwd(a, k, v, torch.empty_like(a), table, start, one, lens, 1, 31, 4)
    c = sink_attention_fwd(a, k, v, torch.empty_like(a), table, start, one, lens, 2, 31, 4)
    return a, b, c, shared_prefix_attention_fwd(a, k, v, torch.empty_like(a), table[:2], lens[4:], groups, table, lens)

def work(i):
    gate.wait()
    with torch.cuda.stream(torch.cuda.Stream()):
        outs = [step() for _ in range(50)]
    torch.cuda.synchronize()
    return outs

with ThreadPoolExecutor(n) as pool:
    done = [f.result() for f in [pool.submit(work, i) for i in range(n)]]
ref = step()
assert len(done) == n and all(len(outs) == 50 for outs in done)
assert all(torch.equal(x, y) for outs in done for got in outs for x, y in zip(got, ref))
check_device_status()
print("all through")
"""
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    res = subprocess.run([sys.executable, "-c", code], cwd=root, capture_output=True, text=True, timeout=600)
    assert res.returncode == 0 and "all through" in res.stdout, res.stdout + res.stderr
