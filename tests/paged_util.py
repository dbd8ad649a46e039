"""Inputs and definitions for the tests of the paged cache: pools with what real ones hold (numbers that nobody wrote in unused places), tables,
and attention in 64 bits."""
import math

import torch

TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}


def pools(pages, page, kv_heads, dim, dtype, g, order="page pos head", fill=None):
    """k, v [pages][page][kv_heads][dim] of normal values (or `fill`), laid out in another order of dimensions where asked."""
    def make():
        shape = dict(page=pages, pos=page, head=kv_heads)
        names = order.split()
        t = torch.randn([shape[n] for n in names] + [dim], generator=g, device="cuda").to(dtype)
        if fill is not None:
            t.fill_(fill)
        return t.permute([names.index(n) for n in ("page", "pos", "head")] + [3])
    return make(), make()


def tables(lengths, page, pages, g, width=None):
    """Page tables of sequences of these lengths, over distinct pages in random order; entries that hold nothing are far out of range."""
    need = [-(-n // page) for n in lengths]
    assert sum(need) <= pages
    place = torch.randperm(pages, generator=g)[:sum(need)].to(torch.int32)
    t = torch.full((len(lengths), width or max(1, max(need, default=1))), 0x7ffffff0, dtype=torch.int32)
    at = 0
    for i, n in enumerate(need):
        t[i, :n] = place[at:at + n]
        at += n
    return t


def rows_of(pool, table_row, page, n):
    """The first n positions of a sequence, [n][kv_heads][dim] in 64 bits."""
    if n == 0:
        return torch.zeros(0, *pool.shape[2:], dtype=torch.float64, device=pool.device)
    return pool[table_row[:-(-n // page)].long().to(pool.device)].flatten(0, 1)[:n].double()


def seen(p, n, window, sinks, device):
    """Which of n positions the queries at positions p see."""
    j, p = torch.arange(n, device=device)[None], p[:, None]
    vis = j <= p
    return vis & ((j > p - window) | (j < sinks)) if window else vis


def attention(q, k, v, table, page, kv_len, starts, scale, window=0, sinks=0):
    """(out, lse, size) in 64 bits of rows starts[0] .. starts[-1] of q [tokens][heads][dim].  size: the sum of |p v| and the largest |score|
    of every row, which rounding errors are counted by."""
    heads, group = q.shape[1], q.shape[1] // k.shape[2]
    out = torch.zeros(q.shape, dtype=torch.float64, device=q.device)
    lse = torch.full(q.shape[:2], -math.inf, dtype=torch.float64, device=q.device)
    mass = torch.zeros(q.shape, dtype=torch.float64, device=q.device)
    for s, n in enumerate(kv_len):
        lo, hi = starts[s], starts[s + 1]
        if hi == lo or n == 0:
            continue
        kk, vv = rows_of(k, table[s], page, n), rows_of(v, table[s], page, n)
        p = torch.arange(n - (hi - lo), n, device=q.device)
        vis = seen(p, n, window, sinks, q.device)
        for h in range(heads):
            x = (q[lo:hi, h].double() @ kk[:, h // group].T * scale).masked_fill(~vis, -math.inf)
            m = x.amax(1, keepdim=True)
            e = torch.where(vis, torch.exp(x - torch.where(m == -math.inf, 0.0, m)), 0.0)
            l = e.sum(1, keepdim=True)
            w = torch.where(l > 0, e / l, 0.0)
            used = vis.any(0)
            out[lo:hi, h] = w[:, used] @ vv[used, h // group]
            mass[lo:hi, h] = w[:, used] @ vv[used, h // group].abs()
            lse[lo:hi, h] = torch.where(l > 0, m + torch.log(l), -math.inf)[:, 0]
    return out, lse, mass


def poison(pool, table, page, kv_len, new, window=0, sinks=0):
    """Not-a-numbers in every place of a pool that no query of the call sees."""
    keep = torch.zeros(pool.shape[:2], dtype=torch.bool, device=pool.device)
    for s, (n, m) in enumerate(zip(kv_len, new)):
        if n == 0 or m == 0:
            continue
        j = torch.arange(n)
        j = j[(j > n - m - window) | (j < sinks)] if window else j
        keep[table[s, j // page].long().to(pool.device), (j % page).to(pool.device)] = True
    pool[~keep] = math.nan


def tolerance(out, mass, dtype):
    """What an output may be off, by arithmetic.  f32: a score is a sum of `dim` products whose absolute values come to about 7 for normal values
    and a scale of dim^-1/2 (tests with larger scores say so); with 2^-22 of each product (two f16 terms) and f32 sums it is off by at most
    7 * (2^-22 + 2^-19) < 1.6e-5, and so is the logarithm of a probability; its exponential adds 2^-21, the sums of probabilities and values
    2^-20 each, a probability in two f16 terms 2^-21: below 2e-5 of the mass sum |p v|, and again for the sum that it is divided by.  16 bits: a probability is
    rounded by at most half a step, and so is the output."""
    half = 0.0 if dtype == torch.float32 else torch.finfo(dtype).eps / 2
    least = 2.0 ** -24 if dtype == torch.float16 else 0.0   # a step among the subnormals
    return mass * (4e-5 + half) + out.abs() * half + least * half


LSE_OFF = 4e-5   # of lse: the scores' error, as above; and 2^-22 of its size


def worst(got, want, tol):
    """The largest error in units of its tolerance."""
    d = (got.double() - want).abs()
    return float(torch.where(d == 0, 0.0, d / tol.clamp(min=1e-300)).max()) if got.numel() else 0.0
