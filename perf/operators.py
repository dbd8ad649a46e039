"""The paged key-value cache as measurable cases: attention of new tokens and of prompts over pages, the pages' writes and copies.

A cache holds pages of `page` positions, [pages][page][kv heads][dim], for each of keys and values; a table per sequence says which page
holds which positions.  A query at position p sees position j where j <= p and, with a window, j > p - window or j < sinks.  Lengths of
a batch come from the case: position counts spread evenly from short to `kv` (`even`: all the same).
"""
from __future__ import annotations

import math

import torch

own = False

DT = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}


def _decode(name, seqs, kv, heads=32, kv_heads=8, dim=128, page=64, q="f32", cache="f16", window=0, sinks=0, even=False):
    return dict(name=name, kind="decode", seqs=seqs, kv=kv, heads=heads, kv_heads=kv_heads, dim=dim, page=page, q=q, cache=cache, window=window, sinks=sinks, even=even)


def _prompt(name, seqs, new, context, heads=32, kv_heads=8, dim=128, page=64, q="f32", cache="f16", window=0, sinks=0, even=False):
    return dict(name=name, kind="prompt", seqs=seqs, new=new, context=context, heads=heads, kv_heads=kv_heads, dim=dim, page=page, q=q, cache=cache, window=window,
                sinks=sinks, even=even)


def listed():
    return [
        # a chat's step right after a short question: launches and latency are everything
        _decode("decode-1x100", 1, 100, page=16, even=True),
        # one long document in the cache, one new token: eight key heads have to keep the whole chip busy
        _decode("decode-1x32768", 1, 32768, page=64, even=True),
        # a server's step: sequences of all ages, none to 16384 positions long
        _decode("decode-64x16384", 64, 16384, page=16, q="bf16", cache="bf16"),
        # window attention with the first tokens kept: long sequences of which a step reads a thousand positions
        _decode("decode-48x20000-window-1024", 48, 20000, heads=16, kv_heads=4, dim=64, page=32, q="f16", window=1024, sinks=4),
        # a short question behind a short history
        _prompt("prompt-33-behind-300", 1, 33, 300, heads=16, kv_heads=8, page=16, even=True),
        # the benchmark's prompt: 2048 tokens from position 0
        _prompt("prompt-2048", 1, 2048, 0, even=True),
        # pieces of several prompts in one step of a server, odd lengths, behind contexts of all lengths
        _prompt("prompt-5x512-behind-6000", 5, 512, 6000, page=32, q="bf16", cache="bf16"),
        # a long text through window attention with the first tokens kept
        _prompt("prompt-8191-window-1024", 1, 8191, 0, heads=16, kv_heads=4, dim=128, page=128, q="f16", window=1024, sinks=4, even=True),
        # the rows of a step's tokens go to their pages
        dict(name="append-64", kind="append", seqs=64, new=1, context=2000, kv_heads=8, dim=128, page=16, src="f32", cache="f16"),
        # the rows of prompts' tokens
        dict(name="append-4x3000", kind="append", seqs=4, new=3000, context=1000, kv_heads=8, dim=128, page=64, src="f32", cache="f16"),
        # beams part: their last pages are copied in all layers of an 8B-sized model
        dict(name="copy-8-pages-32-layers", kind="copy", pairs=8, layers=32, pages=64, kv_heads=8, dim=128, page=16, cache="f16", part=True),
        # a pool is compacted: the pages at its end move into the holes
        dict(name="copy-500-pages-4-layers", kind="copy", pairs=500, layers=4, pages=1024, kv_heads=8, dim=128, page=64, cache="bf16", part=False),
    ]


def _log(rng, lo, hi):
    return min(hi, int(math.exp(rng.uniform(math.log(lo), math.log(hi + 1)))))


def draw(rng):
    kind = rng.choice(["decode", "decode", "decode", "prompt", "prompt", "prompt", "append", "copy"])
    kv_heads, group = rng.choice([1, 2, 4, 8, 8, 16]), rng.choice([1, 2, 4, 4, 5, 7, 8, 16])
    size = dict(kv_heads=kv_heads, dim=rng.choice([64, 128, 128]), page=rng.choice([8, 16, 32, 64, 128, 256]))
    q, cache = rng.choice([("f32", "f16"), ("f32", "f16"), ("f16", "f16"), ("bf16", "bf16")])
    if kind in ("decode", "prompt"):
        if kv_heads * group > 64:
            group = 4
        size |= dict(heads=kv_heads * group, q=q, cache=cache, even=rng.random() < 0.3)
        size |= dict(window=_log(rng, 16, 4096), sinks=rng.choice([0, 1, 4, 64])) if rng.random() < 0.4 else dict(window=0, sinks=0)
    width = kv_heads * size["dim"]
    if kind == "decode":
        seqs = _log(rng, 1, 128)
        c = _decode("", seqs, _log(rng, 1, min(65536, 64 * 16384 * 1024 // (seqs * max(width, 128)))), **size)
    elif kind == "prompt":
        seqs, new = _log(rng, 1, 8), _log(rng, 1, 4096)
        most = 2048 * 2048 * 32 * 128 // (seqs * new * size["heads"] * size["dim"])   # keys that the largest listed prompt of this form would leave
        while new > 1 and most < 1.5 * new:
            new = new * 2 // 3
            most = 2048 * 2048 * 32 * 128 // (seqs * new * size["heads"] * size["dim"])
        c = _prompt("", seqs, new, _log(rng, 1, max(1, min(32768, most - new))) - 1, **size)
    elif kind == "append":
        seqs = _log(rng, 1, 64)
        c = dict(kind=kind, seqs=seqs, new=_log(rng, 1, 12000 * 1024 // (seqs * width)) if seqs * width < 1 << 20 else 1, context=_log(rng, 1, 500), src=q, cache=cache, **size)
    else:
        pages = _log(rng, 4, max(8, min(2048, (1 << 25) // (size["page"] * width))))
        c = dict(kind=kind, pairs=_log(rng, 1, pages // 2), layers=_log(rng, 1, 8), pages=pages, cache=cache, part=rng.random() < 0.5, **size)
    c.pop("name", None)
    return c


def _spread(n, most, even, least=0):
    """n counts up to `most`: all the same, or spread evenly from `least` on, in an order that is not sorted."""
    if even or n == 1:
        return [most] * n
    return [least + (i * 29 % n if math.gcd(29, n) == 1 else i) * (most - least) // (n - 1) for i in range(n)]


def _lengths(c):
    """(new tokens, positions in the cache behind them) of every sequence."""
    if c["kind"] == "decode":
        kv = _spread(c["seqs"], c["kv"], c["even"])
        return [1] * c["seqs"], kv
    if c["kind"] == "append":
        new = _spread(c["seqs"], c["new"], c["new"] == 1, 1)
        return new, [n + c["context"] * (i + 1) // c["seqs"] for i, n in enumerate(new)]
    new = _spread(c["seqs"], c["new"], c["even"], 1)
    return new, [n + x for n, x in zip(new, _spread(c["seqs"], c["context"], c["even"])[::-1])]


def _seen(p, window, sinks):
    """How many positions a query at position p sees."""
    if p < 0:
        return 0
    return p + 1 if window == 0 else min(p + 1, window) + min(sinks, max(0, p + 1 - window))


# ---- inputs --------------------------------------------------------------------------------------
def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed * 7 + 3)


def _randn(shape, dtype, g):
    """Normal values of a type, made a part at a time."""
    t = torch.empty(shape, dtype=dtype, device="cuda")
    flat = t.view(-1)
    for i in range(0, flat.numel(), 1 << 27):
        flat[i:i + (1 << 27)] = torch.randn(min(1 << 27, flat.numel() - i), device="cuda", generator=g).to(dtype)
    return t


def prepare(case, seed):
    c, g = case, _gen(seed)
    H, D, P = c["kv_heads"], c["dim"], c["page"]
    if c["kind"] == "copy":
        shape = (c["layers"], c["pages"], P, H, D)
        s = dict(case=c, k=_randn(shape, DT[c["cache"]], g), v=_randn(shape, DT[c["cache"]], g))
        # the plan of a program's book-keeping, on the host: distinct pages, some of which are only partly filled
        order = torch.randperm(c["pages"], generator=torch.Generator().manual_seed(seed)).to(torch.int32)
        s["src"], s["dst"] = order[:c["pairs"]].numpy(), order[c["pairs"]:2 * c["pairs"]].numpy()
        s["rows"] = (torch.arange(c["pairs"], dtype=torch.int32) * 5 % P + 1).numpy() if c["part"] else None
    else:
        new, kv = _lengths(c)
        need = [-(-n // P) for n in kv]
        total = sum(need)
        pages = total + total // 8 + 1
        place = torch.randperm(pages, generator=torch.Generator().manual_seed(seed)).to(torch.int32)
        table = torch.full((c["seqs"], max(1, max(need))), -1, dtype=torch.int32)
        at = 0
        for i, n in enumerate(need):
            table[i, :n] = place[at:at + n]
            at += n
        tokens = sum(new)
        start = torch.tensor([0] + new).cumsum(0).to(torch.int32)
        s = dict(case=c, k=_randn((pages, P, H, D), DT[c["cache"]], g), v=_randn((pages, P, H, D), DT[c["cache"]], g), table=table.cuda(),
                 kv_len=torch.tensor(kv, dtype=torch.int32).cuda(), start=start.cuda(), tokens=tokens, most=max(new))
        if c["kind"] == "append":
            s["k_new"], s["v_new"] = (_randn((tokens, H, D), DT[c["src"]], g) for _ in range(2))
        else:
            s["q"] = _randn((tokens, c["heads"], D), DT[c["q"]], g)
            s["out"] = torch.empty_like(s["q"])
            s["scale"] = D ** -0.5
    if own:   # what a serving program keeps: descriptions of its cache and batch, and a workspace
        from runnburn_b200 import paged
        s["cache"] = paged.PagedCache(s["k"], s["v"])
        if c["kind"] != "copy":
            s["batch"] = paged.PagedBatch(s["table"], s["kv_len"], None if c["kind"] == "decode" else s["start"], s["tokens"])
        if c["kind"] in ("decode", "prompt"):
            s["workspace"] = paged.Workspace()
    return s


# ---- the operators -------------------------------------------------------------------------------
def _places(s):
    """(sequence, index among its new tokens, position) of every token."""
    t = torch.arange(s["tokens"], device="cuda")
    seq = torch.searchsorted(s["start"][1:].long(), t, right=True)
    i = t - s["start"][seq]
    new = s["start"][1:] - s["start"][:-1]
    return seq, i, s["kv_len"][seq] - new[seq] + i


def _plain_attention(s):
    c = s["case"]
    B, G, D, P = c["seqs"], c["kv_heads"], c["dim"], c["page"]
    group, L = c["heads"] // G, s["table"].shape[1] * c["page"]
    at = s["table"].clamp(min=0).long()
    j = torch.arange(L, device="cuda")
    held = (j < s["kv_len"][:, None])[:, :, None, None]
    k = s["k"][at].view(B, L, G, D).float()
    v = torch.where(held, s["v"][at].view(B, L, G, D).float(), 0.0)
    seq, i, pos = _places(s)
    q = torch.zeros(B, s["most"], G, group, D, device="cuda")
    q[seq, i] = s["q"].view(-1, G, group, D).float() * s["scale"]
    p = torch.full((B, s["most"]), -1, dtype=torch.int64, device="cuda")
    p[seq, i] = pos.long()
    seen = j <= p[:, :, None]
    if c["window"]:
        seen &= (j > p[:, :, None] - c["window"]) | (j < c["sinks"])
    x = q.permute(0, 2, 3, 1, 4).reshape(B, G, -1, D) @ k.permute(0, 2, 3, 1)                   # [B, G, group * most, L]
    x = x.view(B, G, group, s["most"], L).masked_fill_(~seen[:, None, None], -math.inf)
    m = x.amax(-1, keepdim=True)
    e = x.sub_(torch.where(m == -math.inf, 0.0, m)).exp_()
    l = e.sum(-1, keepdim=True)
    o = (e.view(B, G, -1, L) @ v.permute(0, 2, 1, 3)).view(B, G, group, s["most"], D)
    o = torch.where(l > 0, o / l, 0.0).permute(0, 3, 1, 2, 4)[seq, i]
    return o.reshape(-1, c["heads"], D).to(DT[c["q"]])


def run(state):
    s, c = state, state["case"]
    if c["kind"] in ("decode", "prompt"):
        if own:
            from runnburn_b200 import paged
            call = paged.attention_decode_paged if c["kind"] == "decode" else paged.attention_prefill_paged
            return call(s["cache"], s["batch"], s["q"], s["scale"], out=s["out"], window=c["window"], sinks=c["sinks"], workspace=s["workspace"])
        return _plain_attention(s)
    if c["kind"] == "append":
        if own:
            from runnburn_b200 import paged
            paged.paged_kv_append(s["cache"], s["batch"], s["k_new"], s["v_new"])
        else:
            seq, _, pos = _places(s)
            page = s["table"][seq, (pos // c["page"]).long()].long()
            s["k"][page, (pos % c["page"]).long()] = s["k_new"].to(s["k"].dtype)
            s["v"][page, (pos % c["page"]).long()] = s["v_new"].to(s["v"].dtype)
    elif own:
        from runnburn_b200 import paged
        paged.paged_kv_copy(s["cache"], s["src"], s["dst"], s["rows"])
    else:
        src, dst = (torch.from_numpy(s[n]).cuda().long() for n in ("src", "dst"))
        rows = torch.from_numpy(s["rows"]).cuda() if s["rows"] is not None else torch.full_like(dst, c["page"])
        keep = (torch.arange(c["page"], device="cuda") < rows[:, None])[None, :, :, None, None]
        for t in (s["k"], s["v"]):
            t[:, dst] = torch.where(keep, t[:, src], t[:, dst])
    return {"k": s["k"], "v": s["v"]}


# ---- what a pass cannot do without ---------------------------------------------------------------
def work(case):
    c = case
    row = c["kv_heads"] * c["dim"]
    if c["kind"] == "copy":
        rows = sum(i * 5 % c["page"] + 1 for i in range(c["pairs"])) if c["part"] else c["pairs"] * c["page"]
        return dict(bytes=rows * c["layers"] * row * 2 * 2 * 2, flops=0)
    new, kv = _lengths(c)
    if c["kind"] == "append":
        return dict(bytes=sum(new) * row * 2 * (2 + (4 if c["src"] == "f32" else 2)), flops=0)
    w, z = c["window"], c["sinks"]
    seen = sum(_seen(n - m + i, w, z) for m, n in zip(new, kv) for i in range(m))
    # positions that some query of the call sees: the last ones and the first ones
    read = sum(n if w == 0 else min(n, m + w - 1) + min(z, max(0, n - m - w + 1)) for m, n in zip(new, kv) if n)
    return dict(bytes=read * row * 2 * 2 + sum(new) * c["heads"] * c["dim"] * 2 * (4 if c["q"] == "f32" else 2), flops=4 * c["dim"] * c["heads"] * seen)


# ---- the definition in 64 bits -------------------------------------------------------------------
def exact(case, seed):
    c, s = case, prepare(case, seed)
    P = c["page"]
    if c["kind"] == "copy":
        out = {}
        for n in ("k", "v"):
            t = s[n].double()
            for i, (a, b) in enumerate(zip(s["src"].tolist(), s["dst"].tolist())):
                m = P if s["rows"] is None else int(s["rows"][i])
                t[:, b, :m] = s[n][:, a, :m].double()
            out[n] = t
        return out
    new, kv = _lengths(c)
    table = s["table"].cpu()
    if c["kind"] == "append":
        out, at = {n: s[n].double() for n in ("k", "v")}, 0
        for b, (m, n) in enumerate(zip(new, kv)):
            j = torch.arange(n - m, n)
            page, row = table[b, j // P].long().cuda(), (j % P).cuda()
            for t in ("k", "v"):
                out[t][page, row] = s[t + "_new"][at:at + m].double()
            at += m
        return out
    out, at, group = torch.zeros(s["tokens"], c["heads"], c["dim"], dtype=torch.float64, device="cuda"), 0, c["heads"] // c["kv_heads"]
    for b, (m, n) in enumerate(zip(new, kv)):
        pages = table[b, :-(-n // P)].long().cuda()
        k, v = (s[t][pages].flatten(0, 1)[:n].double() for t in ("k", "v"))
        for lo in range(0, m if n else 0, 1024):
            hi = min(m, lo + 1024)
            p = torch.arange(n - m + lo, n - m + hi, device="cuda")[:, None]
            j = torch.arange(n, device="cuda")[None]
            hidden = j > p
            if c["window"]:
                hidden = hidden | ((p - j >= c["window"]) & (j >= c["sinks"]))
            for h in range(c["heads"]):
                w = (s["q"][at + lo:at + hi, h].double() @ k[:, h // group].T * s["scale"]).masked_fill(hidden, -math.inf)
                out[at + lo:at + hi, h] = torch.softmax(w, -1) @ v[:, h // group]
        at += m
    return out
