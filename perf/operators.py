"""Attention with a window and sinks, attention over a shared prefix and rotary positions of several axes, as
measurable cases.

  rotary   rotary positions of several axes (time, height, width) for q and k, forward, and with its gradient
  sink     attention over the paged cache with a sliding window and a few first tokens that stay visible:
           single tokens, a few tokens per sequence, chunks of prompts
  prefix   one token per sequence over its own pages and over a prefix that its group of sequences shares

Where `own` is false `run` computes each from elementary torch operations in 32 bits (the rotation's angles in 64),
with one rounding at the end.  Lengths of a batch are spread evenly over their range and shuffled by the seed, so
that a case's work does not depend on the seed while its inputs do.
"""
from __future__ import annotations

import math

import torch

own = False

DEVICE = "cuda"
DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
SIZE = {"bf16": 2, "fp16": 2, "fp32": 4}


def listed():
    return [
        # One decode step of a server that also takes images: 16 running requests.  The smallest call there is.
        {"name": "rotary_decode", "kind": "rotary", "tokens": 16, "hq": 32, "hkv": 8, "dim": 128, "rot": 128,
         "sections": "16,24,24", "interleaved": False, "offset": 5000, "grad": False, "dtype": "bf16"},
        # Prefill of long video prompts, far into the context.
        {"name": "rotary_video", "kind": "rotary", "tokens": 32768, "hq": 32, "hkv": 8, "dim": 128, "rot": 128,
         "sections": "16,24,24", "interleaved": False, "offset": 200000, "grad": False, "dtype": "bf16"},
        # A training step of a vision tower: axes dealt out in turn, half the head rotated, an odd number of tokens.
        {"name": "rotary_training", "kind": "rotary", "tokens": 9217, "hq": 16, "hkv": 16, "dim": 80, "rot": 40,
         "sections": "8,6,6", "interleaved": True, "offset": 0, "grad": True, "dtype": "bf16"},
        # One decode step for four running requests, some shorter than the window.
        {"name": "sink_decode_small", "kind": "sink", "batch": 4, "lo": 1, "hi": 1, "past": 4000, "page": 16,
         "window": 1023, "sinks": 4, "hq": 32, "hkv": 8, "dim": 128, "dtype": "fp16", "softcap": 0.0},
        # One decode step of a full server: 64 requests of up to 32k tokens.
        {"name": "sink_decode_large", "kind": "sink", "batch": 64, "lo": 1, "hi": 1, "past": 32768, "page": 64,
         "window": 4095, "sinks": 4, "hq": 32, "hkv": 8, "dim": 128, "dtype": "bf16", "softcap": 0.0},
        # Drafted tokens checked in one pass: five per sequence, seven query heads to a key head.
        {"name": "sink_verify", "kind": "sink", "batch": 24, "lo": 2, "hi": 5, "past": 7001, "page": 16,
         "window": 2047, "sinks": 16, "hq": 28, "hkv": 4, "dim": 128, "dtype": "bf16", "softcap": 0.0},
        # Chunks of running prompts of odd lengths, a short window.
        {"name": "sink_chunks", "kind": "sink", "batch": 7, "lo": 100, "hi": 1500, "past": 9000, "page": 64,
         "window": 511, "sinks": 130, "hq": 24, "hkv": 8, "dim": 96, "dtype": "bf16", "softcap": 30.0},
        # Two long prompts in one go.
        {"name": "sink_prefill_long", "kind": "sink", "batch": 2, "lo": 16384, "hi": 16384, "past": 0, "page": 64,
         "window": 4095, "sinks": 4, "hq": 32, "hkv": 8, "dim": 128, "dtype": "bf16", "softcap": 0.0},
        # Eight requests behind one system prompt, at their first tokens.
        {"name": "prefix_small", "kind": "prefix", "groups": 1, "batch": 8, "prefix": 1000, "own_lo": 1, "own_hi": 40,
         "page": 16, "hq": 32, "hkv": 8, "dim": 128, "dtype": "bf16", "softcap": 0.0},
        # Several answers to each of 16 questions.
        {"name": "prefix_groups", "kind": "prefix", "groups": 16, "batch": 128, "prefix": 4000, "own_lo": 1,
         "own_hi": 701, "page": 16, "hq": 28, "hkv": 4, "dim": 128, "dtype": "fp16", "softcap": 0.0},
        # A few questions to one long document.
        {"name": "prefix_document", "kind": "prefix", "groups": 1, "batch": 16, "prefix": 120001, "own_lo": 20,
         "own_hi": 900, "page": 64, "hq": 32, "hkv": 8, "dim": 128, "dtype": "bf16", "softcap": 30.0},
        # A full server behind one long prompt with examples.
        {"name": "prefix_large", "kind": "prefix", "groups": 1, "batch": 256, "prefix": 32768, "own_lo": 16,
         "own_hi": 512, "page": 64, "hq": 32, "hkv": 8, "dim": 128, "dtype": "bf16", "softcap": 0.0},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["rotary", "sink", "sink", "prefix", "prefix"])
    hq, hkv = rng.choice([(32, 8), (32, 8), (16, 16), (24, 8), (28, 4), (16, 1)])
    dtype = rng.choice(["bf16", "bf16", "fp16"])
    if kind == "rotary":
        dim, rot, sections = rng.choice([(128, 128, "16,24,24"), (128, 128, "24,20,20"), (80, 40, "8,6,6"),
                                         (64, 64, "16,16"), (96, 64, "32"), (72, 72, "9,9,9,9")])
        grad, dtype = rng.random() < 0.4, rng.choice([dtype, dtype, "fp32"])
        most = 30000 // ((2 if grad else 1) * (2 if dtype == "fp32" else 1))
        return {"kind": kind, "tokens": _log(rng, 1, most), "hq": hq, "hkv": hkv, "dim": dim, "rot": rot,
                "sections": sections, "interleaved": rng.random() < 0.5, "offset": _log(rng, 1, 1000000),
                "grad": grad, "dtype": dtype}
    dim = rng.choice([64, 80, 96, 128, 128, 128])
    softcap = rng.choice([0.0, 0.0, 0.0, 30.0])
    page = rng.choice([16, 32, 64, 128])
    if kind == "sink":
        window = _log(rng, 32, 4096)
        past = rng.choice([1, 1, 1, 0]) * _log(rng, 64, 32768)
        form = rng.choice(["one", "one", "few", "chunk", "chunk"])
        if form == "one":
            lo, hi, batch = 1, 1, _log(rng, 1, 64)
        elif form == "few":
            hi = rng.randint(2, 9)
            lo, batch = rng.randint(1, hi), _log(rng, 1, 64)
        else:
            hi = _log(rng, 10, 8192)
            lo, batch = max(hi // rng.choice([1, 4, 40]), 1), min(_log(rng, 1, 16), 32768 // hi)
            past = min(past, 16000)
        batch = max(1, min(batch, (64 * 8) // hkv)) if form != "chunk" else batch
        return {"kind": kind, "batch": batch, "lo": lo, "hi": hi, "past": past, "page": page, "window": window,
                "sinks": rng.choice([0, 1, 4, 4, 16, 100]), "hq": hq, "hkv": hkv, "dim": dim, "dtype": dtype,
                "softcap": softcap}
    groups = rng.choice([1, 1, 1, _log(rng, 1, 24)])
    prefix = min(_log(rng, 30, 120000), 960000 // (groups * hkv))
    batch = max(groups, min(_log(rng, 1, 256), 180 * 32768 // prefix))
    own_hi = min(_log(rng, 1, 4000), 320000 // (batch * hkv))
    return {"kind": kind, "groups": groups, "batch": batch, "prefix": prefix,
            "own_lo": max(own_hi // rng.choice([1, 4, 40]), 1), "own_hi": own_hi, "page": page, "hq": hq, "hkv": hkv,
            "dim": dim, "dtype": dtype, "softcap": softcap}


# ------------------------------------------------------------------------------------------------- inputs
def _spread(n, lo, hi):
    """n whole numbers spread evenly over [lo, hi], both ends included."""
    return [hi] if n == 1 else [lo + (hi - lo) * i // (n - 1) for i in range(n)]


def _sizes(case):
    """Lengths of a case before they are shuffled."""
    if case["kind"] == "sink":
        return _spread(case["batch"], case["lo"], case["hi"]), _spread(case["batch"], case["past"] // 8, case["past"])
    groups, batch = case["groups"], case["batch"]
    members = [batch * (i + 1) // groups - batch * i // groups for i in range(groups)]
    return members, _spread(groups, max(case["prefix"] // 4, 1), case["prefix"]), \
        _spread(batch, case["own_lo"], case["own_hi"])


class _Inputs:
    def __init__(self, seed):
        self.g = torch.Generator(device=DEVICE)
        self.g.manual_seed(seed)

    def normal(self, *shape, dtype):
        return torch.randn(shape, generator=self.g, device=DEVICE, dtype=dtype)

    def shuffled(self, values):
        order = torch.randperm(len(values), generator=self.g, device=DEVICE).tolist()
        return [values[i] for i in order]

    def pages(self, lens, page, taken=0):
        """(block table int32 [len(lens), most pages], pages used): a random permutation of the pool behind `taken`."""
        need = [(n + page - 1) // page for n in lens]
        pool = taken + torch.randperm(sum(need), generator=self.g, device=DEVICE).to(torch.int32)
        table = torch.zeros(len(lens), max(max(need), 1), dtype=torch.int32, device=DEVICE)
        at = 0
        for b, n in enumerate(need):
            table[b, :n] = pool[at:at + n]
            at += n
        return table, taken + at


def _ints(values, dtype=torch.int32):
    return torch.tensor(values, dtype=dtype, device=DEVICE)


def _starts(lens):
    at, out = 0, []
    for n in lens:
        out.append(at)
        at += n
    return out


def _positions(tokens, axes, offset):
    """int64 [axes, tokens]: runs of text (all axes alike) and grids of patches in turn, from `offset` on."""
    cols, at, n, turn = [], offset, 0, 0
    while n < tokens:
        if turn % 2 == 0:
            p = (at + torch.arange(37 + 5 * turn)).repeat(axes, 1)
        else:
            grid = [2, 14 + turn % 5, 11 + turn % 7, 2][:axes]
            p = at + torch.cartesian_prod(*[torch.arange(m) for m in grid]).reshape(-1, axes).t()
        cols.append(p)
        at, n, turn = int(p.max()) + 1, n + p.shape[1], turn + 1
    return torch.cat(cols, 1)[:, :tokens].contiguous()


def prepare(case, seed):
    kind, rnd = case["kind"], _Inputs(seed)
    dtype = DTYPES[case["dtype"]]
    hq, hkv, d = case["hq"], case["hkv"], case["dim"]
    s = {"case": case}
    if kind == "rotary":
        t, sections = case["tokens"], [int(x) for x in case["sections"].split(",")]
        # q and k as a fused projection leaves them: views of one buffer
        qkv = rnd.normal(t, (hq + 2 * hkv) * d, dtype=dtype)
        s["q"], s["k"] = (x.view(t, -1, d) for x in qkv.split([hq * d, hkv * d, hkv * d], dim=-1)[:2])
        if case["grad"]:
            s["q"], s["k"] = (x.detach().clone().requires_grad_() for x in (s["q"], s["k"]))
            s["gq"], s["gk"] = rnd.normal(t, hq, d, dtype=dtype), rnd.normal(t, hkv, d, dtype=dtype)
        shift = int(torch.randint(0, 1000, (1,), generator=rnd.g, device=DEVICE))
        s["sections"] = sections
        s["positions"] = _positions(t, len(sections), case["offset"] + shift).to(DEVICE)
        half = case["rot"] // 2
        s["inv_freq"] = (10000.0 ** (-torch.arange(half, device=DEVICE, dtype=torch.float64) / half)).float()
        return s
    s["scale"] = d ** -0.5
    if kind == "sink":
        new, past = (rnd.shuffled(x) for x in _sizes(case))
        full = [a + b for a, b in zip(new, past)]
        s["new"], s["full"] = new, full
        s["q"] = rnd.normal(sum(new), hq, d, dtype=dtype)
        s["table"], pages = rnd.pages(full, case["page"])
        s["start"], s["lens"], s["kv_lens"], s["most"] = _ints(_starts(new)), _ints(new), _ints(full), max(new)
    else:
        members, prefix, mine = (rnd.shuffled(x) for x in _sizes(case))
        s["members"], s["prefix"], s["mine"] = members, prefix, mine
        s["q"] = rnd.normal(sum(members), hq, d, dtype=dtype)
        s["prefix_table"], pages = rnd.pages(prefix, case["page"])
        s["table"], pages = rnd.pages(mine, case["page"], pages)
        s["prefix_lens"], s["lens"] = _ints(prefix), _ints(mine)
        s["group_start"] = _ints(_starts(members) + [sum(members)])
    s["k_cache"] = rnd.normal(pages, case["page"], hkv, d, dtype=dtype)
    s["v_cache"] = rnd.normal(pages, case["page"], hkv, d, dtype=dtype)
    s["o"] = torch.empty_like(s["q"])
    return s


# ------------------------------------------------------------------------------------------------- plain forms
def _axis_of(sections, interleaved):
    """Axis of every frequency: one axis after the other, or dealt out in turn until an axis has its number."""
    if not interleaved:
        return [a for a, n in enumerate(sections) for _ in range(n)]
    left, out = list(sections), []
    while any(left):
        for a in range(len(left)):
            if left[a]:
                out.append(a)
                left[a] -= 1
    return out


def _rotated(x, cos, sin, rot):
    lo, hi, rest = x[..., :rot // 2].float(), x[..., rot // 2:rot].float(), x[..., rot:].float()
    return torch.cat([lo * cos - hi * sin, hi * cos + lo * sin, rest], -1).to(x.dtype)


def _plain_rotary(s):
    case = s["case"]
    axis = torch.tensor(_axis_of(s["sections"], case["interleaved"]), device=DEVICE)
    angle = s["positions"][axis].t().to(torch.float64) * s["inv_freq"].to(torch.float64)      # [tokens, rot / 2]
    cos, sin = angle.cos().float()[:, None], angle.sin().float()[:, None]
    return [_rotated(s[n], cos, sin, case["rot"]) for n in ("q", "k")]


def _cap(scores, cap):
    return cap * torch.tanh(scores / cap) if cap > 0 else scores


def _softmax_parts(scores):
    m = scores.amax(-1, keepdim=True)
    e = torch.exp(scores - m)
    return m, e, e.sum(-1, keepdim=True)


def _plain_sink(s):
    """Per sequence, a piece of the queries at a time against the keys that some of them see."""
    case = s["case"]
    hq, hkv, d, w, sinks = case["hq"], case["hkv"], case["dim"], case["window"], case["sinks"]
    k_rows, v_rows = s["k_cache"].view(-1, hkv, d), s["v_cache"].view(-1, hkv, d)
    out, at = s["o"], 0
    for b, (n, full) in enumerate(zip(s["new"], s["full"])):
        for i0 in range(0, n, 1024):
            i1 = min(n, i0 + 1024)
            pos = torch.arange(full - n + i0, full - n + i1, device=DEVICE)
            first, last = max(full - n + i0 - w, 0), full - n + i1 - 1
            key = torch.cat([torch.arange(min(sinks, first), device=DEVICE),
                             torch.arange(first, last + 1, device=DEVICE)])
            row = s["table"][b, key // case["page"]].long() * case["page"] + key % case["page"]
            k, v = k_rows[row].float(), v_rows[row].float()                                  # [keys, hkv, d]
            q = s["q"][at + i0:at + i1].float().view(i1 - i0, hkv, hq // hkv, d)
            scores = _cap(torch.einsum("thgd,khd->hgtk", q, k) * s["scale"], case["softcap"])
            seen = (key <= pos[:, None]) & ((key >= pos[:, None] - w) | (key < sinks))
            _, e, total = _softmax_parts(scores.masked_fill_(~seen, float("-inf")))
            o = torch.einsum("hgtk,khd->hgtd", e, v) / total
            out[at + i0:at + i1] = o.permute(2, 0, 1, 3).reshape(i1 - i0, hq, d).to(out.dtype)
        at += n
    return out


def _plain_prefix(s):
    """Scores of a group against its prefix and of every sequence against its own tokens, joined by their sums."""
    case = s["case"]
    hq, hkv, d, page = case["hq"], case["hkv"], case["dim"], case["page"]
    k_rows, v_rows = s["k_cache"].view(-1, hkv, d), s["v_cache"].view(-1, hkv, d)
    out, at = s["o"], 0
    for g, (n, size) in enumerate(zip(s["members"], s["prefix"])):
        key = torch.arange(size, device=DEVICE)
        row = s["prefix_table"][g, key // page].long() * page + key % page
        q = s["q"][at:at + n].float().view(n, hkv, hq // hkv, d)
        scores = _cap(torch.einsum("bhgd,khd->hbgk", q, k_rows[row].float()) * s["scale"], case["softcap"])
        m1, e, l1 = _softmax_parts(scores)
        o1 = torch.einsum("hbgk,khd->hbgd", e, v_rows[row].float())
        key = torch.arange(max(s["mine"][at:at + n]), device=DEVICE)
        row = s["table"][at:at + n, key // page].long() * page + key % page                   # [n, keys]
        scores = _cap(torch.einsum("bhgd,bkhd->hbgk", q, k_rows[row].float()) * s["scale"], case["softcap"])
        seen = key < s["lens"][at:at + n, None]
        m2, e, l2 = _softmax_parts(scores.masked_fill_(~seen[None, :, None], float("-inf")))
        o2 = torch.einsum("hbgk,bkhd->hbgd", e, v_rows[row].float())
        m = torch.maximum(m1, m2)
        a1, a2 = torch.exp(m1 - m), torch.exp(m2 - m)
        o = (o1 * a1 + o2 * a2) / (l1 * a1 + l2 * a2)
        out[at:at + n] = o.transpose(0, 1).reshape(n, hq, d).to(out.dtype)
        at += n
    return out


# ------------------------------------------------------------------------------------------------- one pass
def run(s):
    case = s["case"]
    kind = case["kind"]
    if own:
        import dlcompiler_b200 as dl
    if kind == "rotary":
        if own:
            q, k = dl.apply_multi_axis_rotary(s["q"], s["k"], s["positions"], s["inv_freq"], s["sections"],
                                              interleaved=case["interleaved"])
        else:
            q, k = _plain_rotary(s)
        if not case["grad"]:
            return q, k
        dq, dk = torch.autograd.grad((q, k), (s["q"], s["k"]), (s["gq"], s["gk"]))
        return q.detach(), k.detach(), dq, dk
    if kind == "sink":
        if not own:
            return _plain_sink(s)
        dl.sink_attention_fwd(s["q"], s["k_cache"], s["v_cache"], s["o"], s["table"], s["start"], s["lens"],
                              s["kv_lens"], s["most"], case["window"], case["sinks"], sm_scale=s["scale"],
                              logit_softcapping=case["softcap"] or None)
        return s["o"]
    if not own:
        return _plain_prefix(s)
    dl.shared_prefix_attention_fwd(s["q"], s["k_cache"], s["v_cache"], s["o"], s["prefix_table"], s["prefix_lens"],
                                   s["group_start"], s["table"], s["lens"], sm_scale=s["scale"],
                                   logit_softcapping=case["softcap"] or None)
    return s["o"]


# ------------------------------------------------------------------------------------------------- its work
def work(case):
    es, hq, hkv, d = SIZE[case["dtype"]], case["hq"], case["hkv"], case["dim"]
    if case["kind"] == "rotary":
        t, axes, passes = case["tokens"], case["sections"].count(",") + 1, 2 if case["grad"] else 1
        return {"bytes": passes * 2 * t * (hq + hkv) * d * es + axes * t * 8,
                "flops": passes * 3 * t * (hq + hkv) * case["rot"]}
    if case["kind"] == "sink":
        w, sinks = case["window"], case["sinks"]
        pairs = keys = 0
        for n, past in zip(*_sizes(case)):
            lo = max(past - w, 0)                                     # first key inside the first query's window
            keys += past + n - lo + min(sinks, lo)
            for p in range(past, past + n):
                lo = max(p - w, 0)
                pairs += p + 1 - lo + min(sinks, lo)
        rows = sum(_sizes(case)[0])
        return {"bytes": 2 * keys * hkv * d * es + 2 * rows * hq * d * es, "flops": 4 * pairs * hq * d}
    members, prefix, mine = _sizes(case)
    # which group has which prefix follows the seed: the mean over the ways to pair them
    pairs = sum(members) * sum(prefix) / len(prefix) + sum(mine)
    return {"bytes": 2 * (sum(prefix) + sum(mine)) * hkv * d * es + 2 * sum(members) * hq * d * es,
            "flops": 4 * pairs * hq * d}


# ------------------------------------------------------------------------------------------------- in 64 bits
def exact(case, seed):
    """The definitions in 64 bits: the rotation as a product of complex numbers, each query's softmax over all keys
    of its sequence in order, those it does not see at minus infinity."""
    s = prepare(case, seed)
    hq, hkv, d = case["hq"], case["hkv"], case["dim"]
    if case["kind"] == "rotary":
        half, inv = case["rot"] // 2, s["inv_freq"].double()
        place = torch.zeros(case["tokens"], half, dtype=torch.float64, device=DEVICE)
        if case["interleaved"]:
            order = sorted((i, a) for a, n in enumerate(s["sections"]) for i in range(n))     # (turn, axis)
            for f, (_, a) in enumerate(order):
                place[:, f] = s["positions"][a].double()
        else:
            f = 0
            for a, n in enumerate(s["sections"]):
                place[:, f:f + n] = s["positions"][a].double()[:, None]
                f += n
        turn = torch.polar(torch.ones_like(place), place * inv)[:, None]

        def rotate(x, by):
            x = x.detach().double()
            z = torch.complex(x[..., :half], x[..., half:2 * half]) * by
            return torch.cat([z.real, z.imag, x[..., 2 * half:]], -1)

        out = [rotate(s["q"], turn), rotate(s["k"], turn)]
        return tuple(out + ([rotate(s["gq"], turn.conj()), rotate(s["gk"], turn.conj())] if case["grad"] else []))

    def gathered(cache, pages, n):
        return cache[pages.long()].reshape(-1, hkv, d)[:n].double().transpose(0, 1)          # [hkv, n, d]

    def attend(q, k, v, seen):
        """q [rows, hq, d] in 64 bits; seen [rows, keys] or None."""
        rows = q.shape[0]
        q = q.reshape(rows, hkv, hq // hkv, d).permute(1, 2, 0, 3).reshape(hkv, -1, d)
        x = torch.bmm(q, k.transpose(1, 2)) * d ** -0.5
        if case["softcap"]:
            x = (x / case["softcap"]).tanh() * case["softcap"]
        x = x.reshape(hkv, hq // hkv, rows, -1)
        if seen is not None:
            x = torch.where(seen, x, torch.full((), -math.inf, dtype=torch.float64, device=DEVICE))
        x = torch.softmax(x, -1).reshape(hkv, -1, k.shape[1])
        return torch.bmm(x, v).reshape(hkv, hq // hkv, rows, d).permute(2, 0, 1, 3).reshape(rows, hq, d)

    out, at = torch.zeros(s["q"].shape, dtype=torch.float64, device=DEVICE), 0
    if case["kind"] == "sink":
        for b, (n, full) in enumerate(zip(s["new"], s["full"])):
            k, v = gathered(s["k_cache"], s["table"][b], full), gathered(s["v_cache"], s["table"][b], full)
            key = torch.arange(full, device=DEVICE)
            for i in range(0, n, 256):
                q = s["q"][at + i:at + min(i + 256, n)].double()
                back = full - n + i + torch.arange(q.shape[0], device=DEVICE)[:, None] - key  # how far behind the query
                seen = (back >= 0) & ((back <= case["window"]) | (key < case["sinks"]))
                out[at + i:at + i + q.shape[0]] = attend(q, k, v, seen)
            at += n
        return out
    for g, n in enumerate(s["members"]):
        first = [gathered(s[c], s["prefix_table"][g], s["prefix"][g]) for c in ("k_cache", "v_cache")]
        for b in range(at, at + n):
            rest = [gathered(s[c], s["table"][b], s["mine"][b]) for c in ("k_cache", "v_cache")]
            k, v = (torch.cat(x, 1) for x in zip(first, rest))
            out[b:b + 1] = attend(s["q"][b:b + 1].double(), k, v, None)
        at += n
    return out
