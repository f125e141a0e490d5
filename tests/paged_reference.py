"""Attention over a paged cache in 64 bits for the tests, one query row at a time over the keys that it sees, with the
error that an implementation in the cache's type may make."""
import torch


def rows_of(table_row, n, page):
    """Cache rows of tokens 0 .. n - 1."""
    key = torch.arange(n, device=table_row.device)
    return table_row[key // page].long() * page + key % page


def attend(q, k, v, seen, scale, cap, dtype):
    """q [rows, Hq, D], k / v [keys, Hkv, D], seen [rows, keys] -> (exact output, bound on an implementation's error).

    Keys that a row does not see take no part, whatever they hold.  The bound: a score is a sum of D products, each exact
    in 32 bits, so it is off by (D + 8) 2^-24 sum |q k| scale (8 for the scale, the maximum and their roundings), a
    soft-cap adds 2^-21 cap, an exponential 2^-22; weights move by twice that (they are divided by their sum); P is
    rounded to the type (half a step, for fp16 at least 2^-25 of the largest, and never below a sum of 1); adding n
    terms in 32 bits costs n 2^-24; the output is rounded once."""
    rows, hq, d = q.shape
    hkv = k.shape[1]
    q, k, v = q.double(), k.double(), v.double()
    live = seen.any(0)
    k, v = (torch.where(live[:, None, None], t, torch.zeros((), dtype=t.dtype, device=t.device)) for t in (k, v))
    q = q.view(rows, hkv, hq // hkv, d)
    x = torch.einsum("rhgd,khd->rhgk", q, k) * scale
    size = torch.einsum("rhgd,khd->rhgk", q.abs(), k.abs()) * scale
    if cap:
        x = cap * torch.tanh(x / cap)
    mask = seen[:, None, None]
    some = seen.any(1)
    x = torch.where(mask, x, torch.full((), -float("inf"), dtype=x.dtype, device=x.device))
    x[~some] = 0.0
    w = torch.where(mask, torch.softmax(x, -1), torch.zeros((), dtype=x.dtype, device=x.device))
    out = torch.einsum("rhgk,khd->rhgd", w, v)
    mass = torch.einsum("rhgk,khd->rhgd", w, v.abs())
    n = seen.sum(1).clamp(min=1)[:, None, None, None].double()
    off = torch.where(mask, size, torch.zeros((), dtype=x.dtype, device=x.device)).amax(-1, keepdim=True)
    off = 2 * ((d + 8) * 2.0 ** -24 * off + 2.0 ** -21 * cap + 2.0 ** -22)
    half = torch.finfo(dtype).eps / 2
    bound = mass * (half + off + n * 2.0 ** -24)
    if dtype == torch.float16:
        most = torch.where(live[:, None, None], v.abs(), torch.zeros((), dtype=v.dtype, device=v.device)).amax((0, 2))
        bound = bound + (n * 2.0 ** -25 * most[None, :, None, None])
        bound = bound + 2.0 ** -25
    bound = bound + half * (out.abs() + bound) + torch.finfo(dtype).tiny
    return out.reshape(rows, hq, -1), bound.reshape(rows, hq, -1)


def close(o, ref, bound, what=""):
    err = (o.double() - ref).abs()
    bad = ~(err <= bound)
    assert not bad.any(), f"{what}: {int(bad.sum())} of {bad.numel()} off, worst {float((err / bound).nan_to_num(9e9).max()):.3g} bounds"
