"""The paged cache on the GPU against its definition in 64 bits (tests/paged_util.py): sizes at the edges of pages and tiles, sequences of
length zero, windows and sinks, layouts, and not-a-numbers in every place that no query sees."""
import math

import pytest

import paged_util as pu
from paged_util import LSE_OFF, TYPES, tolerance, worst

pytestmark = pytest.mark.gpu

PAIRS = [("f32", "f16"), ("f16", "f16"), ("bf16", "bf16")]
EDGES = [0, 1, 7, 8, 9, 63, 64, 65, 127, 128, 129, 191, 0]


@pytest.fixture(scope="module")
def P():
    import torch  # noqa: F401

    from runnburn_b200 import build
    build.build_library()
    from runnburn_b200 import ops, paged
    ops.open()
    ops.dev_error_flag()
    return paged


@pytest.fixture(scope="module")
def ws(P):
    return P.Workspace()


@pytest.fixture(autouse=True)
def no_flag(P):
    from runnburn_b200 import ops
    yield
    assert ops.dev_error_flag() == 0


class Case:
    def __init__(self, P, kv_len, new=None, heads=4, kv_heads=2, dim=128, page=16, q="f32", cache="f16", window=0, sinks=0, order="page pos head", seed=0, nan=True, padding=0,
                 gain=1.0):
        import torch
        g, h = torch.Generator("cuda").manual_seed(seed + 1), torch.Generator().manual_seed(seed)
        self.P, self.kv, self.new, self.page = P, kv_len, new or [1] * len(kv_len), page
        n_pages = sum(-(-n // page) for n in kv_len) + 3
        self.table = pu.tables(kv_len, page, n_pages, h)
        self.k, self.v = pu.pools(n_pages, page, kv_heads, dim, TYPES[cache], g, order)
        if nan:
            for t in (self.k, self.v):
                pu.poison(t, self.table, page, kv_len, self.new, window, sinks)
        self.starts = [0]
        for n in self.new:
            self.starts.append(self.starts[-1] + n)
        self.tokens = self.starts[-1] + padding
        self.q = (torch.randn(self.tokens, heads, dim, device="cuda", generator=g) * gain).to(TYPES[q])
        self.scale, self.window, self.sinks = dim ** -0.5, window, sinks
        self.cache = P.PagedCache(self.k, self.v)
        i32 = dict(dtype=torch.int32, device="cuda")
        self.batch = P.PagedBatch(self.table.cuda(), torch.tensor(kv_len, **i32), None if new is None else torch.tensor(self.starts, **i32), self.tokens)
        self.call = P.attention_decode_paged if new is None else P.attention_prefill_paged
        self.lse = torch.full((self.tokens, heads), 7.0, device="cuda")

    def run(self, ws, **kw):
        return self.call(self.cache, self.batch, self.q, self.scale, window=self.window, sinks=self.sinks, workspace=ws, **({"lse": self.lse} | kw))

    def want(self):
        return pu.attention(self.q, self.k, self.v, self.table, self.page, self.kv, self.starts, self.scale, self.window, self.sinks)

    def check(self, got, more=1.0):
        import torch
        out, lse, mass = self.want()
        n = self.starts[-1]
        assert not torch.isnan(got[:n]).any()
        tol = tolerance(out, mass, got.dtype) * more
        assert (off := worst(got[:n], out[:n], tol[:n])) <= 1, off
        empty = lse[:n] == -math.inf
        assert torch.equal(self.lse[:n] == -math.inf, empty) and not got[:n][empty].any()
        d = (self.lse[:n].double() - lse[:n])[~empty].abs()
        assert bool((d <= more * LSE_OFF + lse[:n][~empty].abs() * 2.0 ** -22).all()), float(d.max())


# ---- one token per sequence ---------------------------------------------------------------------------------------------
@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("q,cache", PAIRS)
@pytest.mark.parametrize("heads,kv_heads", [(4, 2), (1, 1), (8, 1), (7, 1), (9, 1), (32, 2), (40, 1), (15, 3), (64, 1), (130, 2)])
def test_decode_heads(P, ws, heads, kv_heads, dim, q, cache):
    c = Case(P, EDGES, heads=heads, kv_heads=kv_heads, dim=dim, q=q, cache=cache, seed=heads)
    c.check(c.run(ws))


@pytest.mark.parametrize("page", [8, 16, 32, 64, 128, 256])
@pytest.mark.parametrize("q,cache,dim", [("f32", "f16", 128), ("bf16", "bf16", 64)])
@pytest.mark.parametrize("order", ["page pos head", "page head pos", "head page pos", "pos head page"])
def test_decode_pages_and_layouts(P, ws, page, q, cache, dim, order):
    c = Case(P, EDGES + [255, 256, 257, 700], page=page, q=q, cache=cache, dim=dim, order=order, seed=page)
    c.check(c.run(ws))


@pytest.mark.parametrize("window,sinks", [(1, 0), (1, 1), (64, 0), (100, 4), (63, 65), (128, 64), (500, 1), (1, 1000), (2000, 3)])
@pytest.mark.parametrize("dim", [64, 128])
def test_decode_windows(P, ws, window, sinks, dim):
    c = Case(P, EDGES + [500, 501, 640, 777, 1500], window=window, sinks=sinks, dim=dim, page=32, seed=window)
    c.check(c.run(ws))


@pytest.mark.parametrize("kv_len,heads,kv_heads", [([1], 8, 8), ([0], 8, 8), ([37], 2, 2), ([9000], 8, 1), ([20011], 16, 2), ([9000, 3, 0, 12345], 8, 2), ([5000] * 9, 4, 4),
                                                   ([70001], 1, 1), (list(range(300)), 4, 1), ([1] * 700, 2, 2), ([4000, 0, 0, 0, 1], 32, 8)])
@pytest.mark.parametrize("q,cache,dim", [("f32", "f16", 128), ("f16", "f16", 64), ("bf16", "bf16", 128)])
def test_decode_split_and_joined(P, ws, kv_len, heads, kv_heads, q, cache, dim):
    c = Case(P, kv_len, heads=heads, kv_heads=kv_heads, page=64, q=q, cache=cache, dim=dim, seed=len(kv_len))
    first = c.run(ws)
    c.check(first)
    assert (c.run(ws) == first).all()   # the sums' order does not depend on who comes first


@pytest.mark.parametrize("kv_len", [[128, 192], [192, 128, 64, 1, 130, 64, 192, 65], [64] * 5 + [192], [1, 192] * 40])
@pytest.mark.parametrize("q,cache,dim,heads", [("f32", "f16", 128, 3), ("bf16", "bf16", 64, 8), ("f16", "f16", 128, 16)])
def test_decode_of_short_sequences_that_differ(P, ws, kv_len, q, cache, dim, heads):
    """One key head and sequences of one to three tiles, some of which the equal runs cut."""
    c = Case(P, kv_len, heads=heads, kv_heads=1, q=q, cache=cache, dim=dim, seed=len(kv_len))
    first = c.run(ws)
    c.check(first)
    assert (c.run(ws) == first).all()


# ---- prompts ------------------------------------------------------------------------------------------------------------
PROMPTS = [
    ([1], [1]), ([5], [5]), ([64], [64]), ([129], [65]), ([300, 0, 77], [33, 0, 77]), ([1000, 130, 7, 64], [1, 130, 2, 63]), ([257], [256]), ([513, 700], [513, 31]),
    ([2100], [16]), ([6000, 0, 40], [3, 0, 40]), ([40, 8], [41, 9]), ([5, 600], [70, 1]),
]


@pytest.mark.parametrize("kv,new", PROMPTS)
@pytest.mark.parametrize("q,cache,dim", [("f32", "f16", 128), ("f32", "f16", 64), ("f16", "f16", 128), ("bf16", "bf16", 64), ("bf16", "bf16", 128)])
def test_prompts(P, ws, kv, new, q, cache, dim):
    """Among them tokens before position 0 (more tokens than positions), which see nothing."""
    c = Case(P, kv, new, q=q, cache=cache, dim=dim, seed=sum(kv))
    c.check(c.run(ws))


@pytest.mark.parametrize("heads,kv_heads", [(1, 1), (8, 1), (7, 1), (5, 5), (12, 4), (32, 1), (48, 1), (130, 2), (160, 1)])
@pytest.mark.parametrize("q,cache", [("f32", "f16"), ("bf16", "bf16")])
def test_prompt_heads(P, ws, heads, kv_heads, q, cache):
    c = Case(P, [200, 0, 333, 64], [70, 0, 1, 64], heads=heads, kv_heads=kv_heads, q=q, cache=cache, seed=heads)
    c.check(c.run(ws))


@pytest.mark.parametrize("page", [8, 16, 32, 64, 128, 256])
@pytest.mark.parametrize("order", ["page pos head", "page head pos", "head page pos", "pos head page"])
@pytest.mark.parametrize("q,cache,dim", [("f32", "f16", 128), ("f16", "f16", 64)])
def test_prompt_pages_and_layouts(P, ws, page, order, q, cache, dim):
    c = Case(P, [300, 77, 640], [129, 77, 5], page=page, order=order, q=q, cache=cache, dim=dim, seed=page)
    c.check(c.run(ws))


@pytest.mark.parametrize("window,sinks", [(1, 0), (1, 1), (64, 0), (100, 4), (63, 65), (128, 64), (300, 1), (1, 1000), (2000, 3), (37, 130)])
@pytest.mark.parametrize("q,cache,dim", [("f32", "f16", 128), ("bf16", "bf16", 64)])
def test_prompt_windows(P, ws, window, sinks, q, cache, dim):
    c = Case(P, [700, 129, 1500, 64], [700, 1, 140, 64], page=32, window=window, sinks=sinks, q=q, cache=cache, dim=dim, seed=window)
    c.check(c.run(ws))


@pytest.mark.parametrize("q,cache", PAIRS)
def test_long_prompt(P, ws, q, cache):
    """Sums over many tiles."""
    c = Case(P, [9001], [300], heads=2, kv_heads=1, page=64, q=q, cache=cache)
    c.check(c.run(ws))


# ---- both ---------------------------------------------------------------------------------------------------------------
BOTH = [(None, [300, 0, 77, 2000]), ([33, 0, 77, 200], [300, 0, 77, 2000])]


@pytest.mark.parametrize("new,kv", BOTH)
@pytest.mark.parametrize("q,cache", PAIRS)
@pytest.mark.parametrize("scale", [0.0, -0.2, 1e-3])
def test_any_scale(P, ws, new, kv, q, cache, scale):
    c = Case(P, kv, new, q=q, cache=cache)
    c.scale = scale
    c.check(c.run(ws), more=3)   # |scores| of 0.2 * 81 instead of 7


@pytest.mark.parametrize("new,kv", BOTH)
@pytest.mark.parametrize("gain", [1e6, 1e-6, 3e30])
def test_f32_queries_of_any_size(P, ws, new, kv, gain):
    """Queries far outside of f16: what counts is the score."""
    c = Case(P, kv, new, gain=gain)
    c.scale = 128 ** -0.5 / gain
    c.check(c.run(ws))


@pytest.mark.parametrize("new,kv", BOTH)
@pytest.mark.parametrize("factor", [1e2, 1e3, 1e4, 1e5, 1e6])
@pytest.mark.parametrize("gain", [1.0, 1e-30, 1e20])
def test_f32_queries_with_one_large_element(P, ws, new, kv, factor, gain):
    """Where the keys have nothing it says nothing about the score, which keeps the bound of 19 bits of every other element (2^20 times smaller)."""
    c = Case(P, kv, new, gain=gain)
    c.scale = 128 ** -0.5 / gain
    c.q[..., 77] *= factor
    c.k[..., 77] = 0
    c.check(c.run(ws))


@pytest.mark.parametrize("new,kv", BOTH)
@pytest.mark.parametrize("q,cache", PAIRS)
@pytest.mark.parametrize("way", ["growing", "falling", "sharp"])
def test_maxima_that_move(P, ws, new, kv, q, cache, way):
    """Scores that grow or fall by some 60 over the sequence, and single keys that take everything.  A score of size 60 has errors nine times
    those of the bound's 7."""
    import torch
    c = Case(P, kv, new, q=q, cache=cache, nan=False)
    c.q += 1.0
    for s, n in enumerate(kv):
        j = torch.arange(n)
        page, row = c.table[s, j // c.page].long().cuda(), (j % c.page).cuda()
        ramp = torch.linspace(0, 5, max(n, 2), device="cuda")[:n]
        ramp = ramp.flip(0) if way == "falling" else ramp
        if way == "sharp":
            ramp = torch.where(torch.arange(n, device="cuda") % 50 == 17, 5.0, 0.0)
        c.k[page, row] = (c.k[page, row].float() + ramp[:, None, None]).to(c.k.dtype)
    c.check(c.run(ws), more=9)


@pytest.mark.parametrize("new,kv", BOTH)
@pytest.mark.parametrize("q", ["f32", "bf16"])
def test_views_and_padding(P, ws, new, kv, q):
    """Queries and outputs as slices of wider rows; what lies beside and behind the batch's tokens stays."""
    import torch
    c = Case(P, kv, new, q=q, cache="f16" if q == "f32" else "bf16", padding=5 if new else 0)
    n = c.starts[-1]
    wide_q, wide_o = torch.full((c.tokens, 16, 128), math.nan, device="cuda", dtype=c.q.dtype), torch.full((c.tokens, 9, 128), 3.0, device="cuda", dtype=c.q.dtype)
    wide_q[:n, 2:6] = c.q[:n]
    c.q = wide_q[:, 2:6]
    got = c.run(ws, out=wide_o[:, 3:7])
    c.check(got)
    assert (wide_o[:, :3] == 3).all() and (wide_o[:, 7:] == 3).all() and (wide_o[n:] == 3).all() and (c.lse[n:] == 7).all()
    assert torch.equal(c.run(ws, lse=None)[:n], got[:n])


@pytest.mark.parametrize("new,kv", BOTH)
def test_values_that_are_not_finite_where_seen(P, ws, new, kv):
    """An infinite or undefined value reaches the queries that see it, in its own dimension, and no other."""
    import torch
    c = Case(P, kv, new, heads=4, kv_heads=2)
    spots = [(0, 290, 1, 5, math.inf), (0, 280, 0, 9, math.nan), (3, 1990, 1, 77, -math.inf), (3, 1855, 0, 64, math.nan), (2, 60, 0, 0, math.inf)]
    clean = c.v.clone()
    for s, j, h, d, x in spots:
        c.v[c.table[s, j // c.page], j % c.page, h, d] = x
        clean[c.table[s, j // c.page], j % c.page, h, d] = 0
    got = c.run(ws)
    out, _, mass = pu.attention(c.q, c.k, clean, c.table, c.page, c.kv, c.starts, c.scale)
    strange = torch.zeros_like(got, dtype=torch.bool)
    for s, j, h, d, x in spots:
        n = c.new[s]
        for i in range(n):
            if c.kv[s] - n + i >= j:
                row = got[c.starts[s] + i, 2 * h:2 * h + 2, d]
                assert (torch.isnan(row).all() if x != x else (row == x).all()), (s, j, i, row)
                strange[c.starts[s] + i, 2 * h:2 * h + 2, d] = True
    ok = torch.where(strange, 0.0, got.double())
    assert worst(ok, torch.where(strange, 0.0, out), tolerance(out, mass, got.dtype)) <= 1


@pytest.mark.parametrize("new,kv", BOTH)
def test_graphs_streams_and_one_workspace(P, new, kv):
    """A captured call follows what its buffers hold when it is replayed; two graphs take turns on a workspace, with eager calls between."""
    import torch
    cases = [Case(P, kv, new, seed=1), Case(P, kv[::-1], new[::-1] if new else None, heads=16, kv_heads=1, q="bf16", cache="bf16", dim=64, seed=2)]
    ws, graphs, outs = P.Workspace(), [], []
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        for c in cases:
            out = torch.empty_like(c.q)
            g = torch.cuda.CUDAGraph()
            with torch.cuda.graph(g, stream=stream):
                c.run(ws, out=out)
            graphs.append(g), outs.append(out)
        for _ in range(2):
            for c, g, out in zip(cases, graphs, outs):
                out.zero_()
                g.replay()
                eager = c.run(ws)
                g.replay()
                assert torch.equal(out, eager)
    stream.synchronize()
    for c, out in zip(cases, outs):
        c.check(out)
    # other lengths, pages and queries in the same buffers
    c = cases[0]
    c.kv = [max(0, n - 7) for n in kv]
    c.batch.kv_len.copy_(torch.tensor(c.kv, dtype=torch.int32))
    c.table = c.table.flip(1).contiguous() if new is None else c.table
    if new is None:   # every entry is used by now
        c.table = torch.randint(0, c.k.shape[0], c.table.shape, dtype=torch.int32, generator=torch.Generator().manual_seed(3))
        c.k.normal_(), c.v.normal_()
        c.batch.table.copy_(c.table)
    c.q.normal_()
    torch.cuda.synchronize()
    with torch.cuda.stream(stream):
        graphs[0].replay()
    stream.synchronize()
    c.check(outs[0])


@pytest.mark.parametrize("new,kv", BOTH)
def test_what_points_outside_is_flagged(P, ws, new, kv):
    """Entries out of range, lengths beyond the table and starts out of order are reported, and the other sequences come out right."""
    import torch
    from runnburn_b200 import ops
    for spoil in ("entry", "negative entry", "length", "negative length") + (("start", "too many tokens") if new else ()):
        c = Case(P, kv, new, nan=False)
        if "entry" in spoil:
            c.batch.table[3, 1] = -1 if "negative" in spoil else c.k.shape[0]
        elif "length" in spoil:
            c.batch.kv_len[3] = -5 if "negative" in spoil else c.table.shape[1] * c.page + 1
        elif spoil == "start":
            c.batch.q_start[3] = c.batch.q_start[4] + 3
        else:
            c.batch.q_start[4] = c.tokens + 40
        got = c.run(ws)
        torch.cuda.synchronize()
        assert ops.dev_error_flag() == P.DEVICE_BAD_PAGE, spoil
        out, _, mass = c.want()
        m = c.starts[2]
        assert worst(got[:m], out[:m], tolerance(out, mass, got.dtype)[:m]) <= 1


@pytest.mark.parametrize("q,cache", PAIRS)
@pytest.mark.parametrize("new,kv", BOTH)
def test_scores_that_are_not_finite(P, ws, new, kv, q, cache):
    """Undefined keys and queries, and scores of plus infinity, leave rows undefined in all dimensions; a score of minus infinity has no weight."""
    import torch
    c = Case(P, kv, new, heads=4, kv_heads=2, q=q, cache=cache)
    keys = [(0, 290, 1, math.nan), (3, 1990, 0, math.inf), (3, 1855, 1, -math.inf), (2, 60, 0, math.inf)]   # sequence, position, head, its element 7
    for s, j, h, x in keys:
        c.k[c.table[s, j // c.page], j % c.page, h, 7] = x
    c.q[c.starts[3], 2] = math.nan
    c.q[c.starts[4] - 1, 1, 64] = math.nan
    got = c.run(ws)
    for s in range(len(c.kv)):
        n = c.new[s]
        if not n or not c.kv[s]:
            continue
        k, v = pu.rows_of(c.k, c.table[s], c.page, c.kv[s]), pu.rows_of(c.v, c.table[s], c.page, c.kv[s])
        seen = pu.seen(torch.arange(c.kv[s] - n, c.kv[s], device="cuda"), c.kv[s], 0, 0, "cuda")
        for h in range(4):
            x = (c.q[c.starts[s]:c.starts[s + 1], h].double() @ k[:, h // 2].double().T * c.scale).masked_fill(~seen, -math.inf)
            bad = (torch.isnan(x) | (x == math.inf)).any(1)
            row, lse = got[c.starts[s]:c.starts[s + 1], h], c.lse[c.starts[s]:c.starts[s + 1], h]
            assert torch.isnan(row[bad]).all() and torch.isnan(lse[bad]).all(), (s, h)
            w = torch.softmax(x[~bad], 1)
            out, mass = w @ v[:, h // 2].double(), w @ v[:, h // 2].double().abs()
            assert worst(row[~bad], out, tolerance(out, mass, got.dtype)) <= 1, (s, h)


@pytest.mark.parametrize("q,cache", PAIRS)
@pytest.mark.parametrize("window,sinks", [(0, 0), (20, 3)])
@pytest.mark.parametrize("copies", [1, 40])
def test_more_tokens_than_positions(P, ws, copies, window, sinks, q, cache):
    """Tokens before the first position see nothing: zeros, with minus infinity for the sum; the others are as ever."""
    new, kv = [40, 5, 300, 1] * copies, [10, 0, 280, 1] * copies
    c = Case(P, kv, new, q=q, cache=cache, window=window, sinks=sinks, nan=False)
    c.check(c.run(ws))


@pytest.mark.parametrize("q,cache", PAIRS)
@pytest.mark.parametrize("window,sinks", [(2 ** 31 - 1, 0), (2 ** 31 - 1, 3), (2 ** 31 - 6, 0), (2 ** 31 - 41, 0)])
def test_windows_without_an_end(P, ws, window, sinks, q, cache):
    """Windows near 2^31 hide nothing, in front of the first position neither."""
    c = Case(P, [10, 0, 280, 1], [40, 5, 300, 1], window=window, sinks=sinks, q=q, cache=cache, nan=False)
    c.check(c.run(ws))
    c = Case(P, [10, 0, 280, 1], window=window, sinks=sinks, q=q, cache=cache)
    c.check(c.run(ws))


@pytest.mark.parametrize("q,cache", PAIRS)
@pytest.mark.parametrize("dim,window", [(64, 0), (128, 0), (128, 1500)])
def test_prompts_whose_longest_decides(P, ws, dim, window, q, cache):
    """Several prompts of very unlike lengths, whose keys pairs of CTAs share."""
    new = [100, 1, 70, 33, 0, 5, 99, 128, 2, 64]
    kv = [5001, 1, 70, 3000, 900, 4000, 131, 128, 2600, 65]
    c = Case(P, kv, new, heads=16, kv_heads=8, dim=dim, page=32, q=q, cache=cache, window=window, sinks=4, padding=9)
    c.check(c.run(ws))


def test_a_workspace_that_was_not_initialised_is_flagged(P, ws):
    """And nothing is written, to it or to the output; one that was initialised then serves."""
    import torch
    from runnburn_b200 import ops
    c, bare = Case(P, [3000, 5, 0, 700]), P.Workspace()
    bare.buffer.zero_()
    out = torch.full_like(c.q, 3.0)
    c.run(bare, out=out)
    torch.cuda.synchronize()
    assert ops.dev_error_flag() == P.DEVICE_BAD_WORKSPACE
    assert bool((out == 3.0).all()) and bool((c.lse == 7.0).all()) and int(bare.buffer.count_nonzero()) == 0
    c.check(c.run(ws, out=out))


def test_streams_side_by_side(P):
    """Calls on streams of their own, with a workspace each, that overlap as they like."""
    import torch
    cases = [Case(P, [20000, 9], seed=1), Case(P, [5, 9000, 0, 300], q="bf16", cache="bf16", dim=64, seed=2), Case(P, [900, 40], [700, 3], seed=3)]
    streams, spaces = [torch.cuda.Stream() for _ in cases], [P.Workspace() for _ in cases]
    torch.cuda.synchronize()
    outs = [[c.run(w, stream=s) for c, s, w in zip(cases, streams, spaces)] for _ in range(4)]
    torch.cuda.synchronize()
    for turn in outs:
        for c, out, first in zip(cases, turn, outs[0]):
            assert torch.equal(out, first)
    for c, out in zip(cases, outs[0]):
        c.check(out)


@pytest.mark.parametrize("new,kv", BOTH)
@pytest.mark.parametrize("number", [False, True])
def test_memory_of_a_given_stream(P, ws, new, kv, number):
    """What a call allocates is of the stream that writes it, not a block that work of the current stream may still be using."""
    import torch
    c, s = Case(P, kv, new), torch.cuda.Stream()
    stream = s.cuda_stream if number else s
    torch.cuda.synchronize()
    block = torch.empty_like(c.q)   # the block that the next one of its size on the current stream gets
    at = block.data_ptr()
    del block
    out = c.run(ws, stream=stream)
    assert out.data_ptr() != at
    s.synchronize()
    c.check(out)
    space = P.Workspace()
    at = space.ptr
    del space
    assert P.Workspace(stream=stream).ptr != at
    torch.cuda.synchronize()


def test_a_workspace_that_goes_while_another_stream_uses_it(P):
    import torch
    c, s, space = Case(P, [3000, 5]), torch.cuda.Stream(), P.Workspace()
    out, at, n = torch.empty_like(c.q), space.ptr, space.bytes
    torch.cuda.synchronize()
    with torch.cuda.stream(s):
        torch.cuda._sleep(50_000_000)
    c.run(space, out=out, stream=s)
    del space
    block = torch.empty(n, dtype=torch.uint8, device="cuda")
    assert block.data_ptr() != at
    s.synchronize()
    c.check(out)


def test_a_workspace_outlives_a_foreign_stream(P):
    """A stream that PyTorch does not know, given by its handle, may be gone before the workspace."""
    import ctypes as C

    import torch
    rt, handle, c, space = C.CDLL("libcudart.so.12"), C.c_void_p(), Case(P, [3000, 5]), P.Workspace()
    torch.cuda.synchronize()
    assert rt.cudaStreamCreate(C.byref(handle)) == 0
    out = c.run(space, stream=handle.value)
    again = c.run(space, stream=handle)
    torch.cuda.synchronize()
    assert rt.cudaStreamDestroy(handle) == 0
    n = space.bytes
    del space
    torch.empty(n, dtype=torch.uint8, device="cuda").zero_()
    torch.cuda.synchronize()
    assert torch.equal(out, again)
    c.check(out)


@pytest.mark.parametrize("bare", [False, True])
def test_a_new_workspace_serves_any_stream(P, bare):
    """Without a wait of the caller's between its making and its use."""
    import torch
    c = Case(P, [9000, 3])
    torch.cuda.synchronize()
    torch.cuda._sleep(50_000_000)
    space, s = P.Workspace(), torch.cuda.Stream()
    assert not torch.cuda.current_stream().query()   # it does not wait itself
    out = c.run(space, stream=s.cuda_stream if bare else s)
    s.synchronize()
    c.check(out)


@pytest.mark.parametrize("q,cache", PAIRS)
@pytest.mark.parametrize("prompt", [False, True])
def test_a_captured_step_with_room(P, prompt, q, cache):
    """Append and attention captured once, with tables as wide as the longest sequence may become, sequences that are not there (of length zero, or
    without tokens) and rows of padding; replayed with other lengths, starts and pages, two graphs on one workspace in turns."""
    import torch
    page, kvh, heads, dim, n_pages, width, i32 = 16, 2, 8, 64, 400, 2000, dict(dtype=torch.int32, device="cuda")
    g, h = torch.Generator("cuda").manual_seed(3), torch.Generator().manual_seed(3)
    n_seq, tokens, dt = 6, 90 if prompt else 6, TYPES[q]
    steps = [([200, 0, 33, 700, 5, 0], [40, 0, 33, 1, 2, 0]), ([64, 128, 0, 0, 0, 1], [64, 20, 0, 0, 0, 1]), ([0] * 6, [0] * 6), ([1500, 1, 1, 1, 1, 1], [85, 1, 1, 1, 1, 1])]
    if not prompt:
        steps = [(kv, [int(n > 0) for n in kv]) for kv, _ in steps]
    stream, space, sides = torch.cuda.Stream(), P.Workspace(), []
    for window in (0, 50):
        k, v = (torch.randn(n_pages, page, kvh, dim, device="cuda", generator=g).to(TYPES[cache]) for _ in range(2))
        s = dict(k=k, v=v, window=window, table=torch.zeros(n_seq, width, **i32), kv=torch.zeros(n_seq, **i32), start=torch.zeros(n_seq + 1, **i32),
                 q=torch.zeros(tokens, heads, dim, device="cuda", dtype=dt), rows=torch.zeros(2, tokens, kvh, dim, device="cuda", dtype=dt),
                 out=torch.zeros(tokens, heads, dim, device="cuda", dtype=dt), lse=torch.zeros(tokens, heads, device="cuda"), graph=torch.cuda.CUDAGraph())
        one, ragged = P.PagedCache(k, v), P.PagedBatch(s["table"], s["kv"], s["start"], tokens)
        batch = ragged if prompt else P.PagedBatch(s["table"], s["kv"])
        torch.cuda.synchronize()
        with torch.cuda.graph(s["graph"], stream=stream):
            P.paged_kv_append(one, ragged, s["rows"][0], s["rows"][1])   # (a sequence that is not there has no token here)
            (P.attention_prefill_paged if prompt else P.attention_decode_paged)(one, batch, s["q"], dim ** -0.5, out=s["out"], lse=s["lse"], window=window, sinks=2, workspace=space)
        sides.append(s)
    for kv, new in steps * 2:
        table = pu.tables(kv, page, n_pages, h, width)
        start = torch.tensor([0] + new).cumsum(0)
        used = int(start[-1])
        for s in sides:
            s["table"].copy_(table), s["kv"].copy_(torch.tensor(kv)), s["start"].copy_(start)
            s["q"].normal_(generator=g), s["rows"].normal_(generator=g), s["out"].fill_(3), s["lse"].fill_(3)
        # of a step of single tokens, the rows of append follow each other, those of attention go by sequence
        torch.cuda.synchronize()
        with torch.cuda.stream(stream):
            for _ in range(2):
                for s in sides:
                    s["graph"].replay()
        torch.cuda.synchronize()
        for s in sides:
            for i, (n, m) in enumerate(zip(kv, new)):
                j = torch.arange(n - m, n)
                at = table[i, j // page].long().cuda(), (j % page).cuda()
                for t, rows in zip((s["k"], s["v"]), s["rows"]):
                    assert torch.equal(t[at], rows[start[i]:start[i + 1]].to(t.dtype))
            rows = list(range(used)) if prompt else [i for i in range(n_seq) if kv[i]]
            starts = start.tolist() if prompt else list(range(n_seq + 1))
            out, lse, mass = pu.attention(s["q"], s["k"], s["v"], table, page, kv, starts, dim ** -0.5, s["window"], 2)
            assert worst(s["out"][rows], out[rows], tolerance(out, mass, dt)[rows]) <= 1 if rows else True
            assert bool(((s["lse"][rows].double() - lse[rows]).abs() <= LSE_OFF + lse[rows].abs() * 2.0 ** -22).all())
            rest = [i for i in range(tokens) if i not in rows]
            assert (s["out"][rest] == (3 if prompt else 0)).all() and (s["lse"][rest] == (3 if prompt else -math.inf)).all()


def test_threads_that_call_at_once(P):
    """Each with a stream and a workspace of its own."""
    import threading

    import torch
    kinds = [dict(kv_len=[3000, 5, 700]), dict(kv_len=[300, 0, 77], new=[33, 0, 77], q="bf16", cache="bf16"), dict(kv_len=[900, 40], new=[700, 3], dim=64),
             dict(kv_len=[64] * 30, q="f16", heads=16, kv_heads=1)]
    cases = [Case(P, **k, seed=i) for i, k in enumerate(kinds * 2)]
    torch.cuda.synchronize()
    outs, failed = [[] for _ in cases], []

    def work(i):
        try:
            c, s, space = cases[i], torch.cuda.Stream(), P.Workspace()
            n, kvh, dim = c.batch.n_tokens, c.k.shape[2], c.k.shape[3]
            k, v = (torch.zeros(4, 16, kvh, dim, device="cuda", dtype=c.k.dtype) for _ in range(2))
            mine = P.PagedCache(k, v)
            s.wait_stream(torch.cuda.current_stream())
            for turn in range(30):
                out = torch.empty_like(c.q)
                s.wait_stream(torch.cuda.current_stream())
                c.run(space, out=out, stream=s, lse=None)
                P.paged_kv_copy(mine, [0, 1], [2, 3], stream=s)
                outs[i].append(out)
                pages = P.KvPages(20, 16)
                a = pages.new()
                pages.extend(a, 50 + turn)
                pages.free(a)
            s.synchronize()
        except Exception as e:  # noqa: BLE001 - told by the main thread
            failed.append(e)
    threads = [threading.Thread(target=work, args=(i,)) for i in range(len(cases))]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    torch.cuda.synchronize()
    assert not failed, failed
    for c, got in zip(cases, outs):
        for out in got:
            assert torch.equal(out, got[0])
        c.run(P.Workspace(), out=got[1])   # the sums beside it
        c.check(got[0])


def test_a_sequence_in_more_parts_than_a_join_has_weights_for(P, ws):
    """One key head and so many tiles that every CTA of the launch leaves a part."""
    for dim, heads in ((64, 2), (128, 5)):
        c = Case(P, [64 * 15000 + 3], heads=heads, kv_heads=1, dim=dim, page=256, nan=False)
        c.check(c.run(ws))


def test_offsets_past_32_bits(P, ws):
    """Pages 2^31 elements and more apart."""
    import torch
    stride, page, dim = 2 ** 31 + 64, 16, 64
    big = torch.empty(3 * stride, dtype=torch.float16, device="cuda")
    for new in (None, [9]):
        c = Case(P, [40], new, kv_heads=1, heads=2, dim=dim, page=page, nan=False)
        k, v = (big[o:].as_strided((3, page, 1, dim), (stride, 2 * dim, dim, 1)) for o in (0, dim))
        c.table = torch.tensor([[2, 0, 1]], dtype=torch.int32)
        c.batch.table.copy_(c.table)
        k.copy_(torch.randn(k.shape)), v.copy_(torch.randn(v.shape))
        c.k, c.v, c.cache = k, v, P.PagedCache(k, v)
        c.check(c.run(ws))
    k_new = torch.randn(1, 1, dim, device="cuda")
    one = P.PagedBatch(c.batch.table[:, :2], torch.tensor([16], dtype=torch.int32, device="cuda"))
    P.paged_kv_append(c.cache, one, k_new, -k_new)
    assert torch.equal(k[2, 15], k_new[0].half()) and torch.equal(v[2, 15], -k_new[0].half())
    P.paged_kv_copy(c.cache, [2], [1])
    assert torch.equal(k[1], k[2]) and torch.equal(v[1], v[2])


@pytest.mark.parametrize("prompt", [False, True])
def test_positions_up_to_the_last(P, ws, prompt):
    """A table of 2^31 positions, all in one page: 2^31 - 256 of them are a length, more are flagged."""
    import torch
    from runnburn_b200 import ops
    page, window, dim, i32 = 256, 300, 64, dict(dtype=torch.int32, device="cuda")
    k, v = (torch.randn(1, page, 1, dim, device="cuda").half() for _ in range(2))
    q = torch.randn(1, 2, dim, device="cuda")
    cache, table = P.PagedCache(k, v), torch.zeros(1, 1 << 23, **i32)
    j = torch.arange(2 ** 31 - 256 - window, 2 ** 31 - 256) % page
    for n in (2 ** 31 - 256, 2 ** 31 - 255, 2 ** 31 - 1):
        batch = P.PagedBatch(table, torch.tensor([n], **i32), torch.tensor([0, 1], **i32) if prompt else None, 1)
        got = (P.attention_prefill_paged if prompt else P.attention_decode_paged)(cache, batch, q, 0.125, window=window, workspace=ws)
        torch.cuda.synchronize()
        assert ops.dev_error_flag() == (0 if n == 2 ** 31 - 256 else P.DEVICE_BAD_PAGE)
        if n == 2 ** 31 - 256:
            w, vv = torch.softmax(q[0].double() @ k[0, j, 0].double().T * 0.125, 1), v[0, j, 0].double()
            assert worst(got[0], w @ vv, tolerance(w @ vv, w @ vv.abs(), got.dtype)) <= 1


# ---- append and copy ----------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("src,cache", [("f32", "f16"), ("f32", "bf16"), ("f16", "f16"), ("bf16", "bf16")])
@pytest.mark.parametrize("page,kv_heads,dim,order", [(16, 8, 128, "page pos head"), (8, 1, 64, "page head pos"), (64, 3, 8, "head page pos"), (256, 5, 200, "pos head page"),
                                                     (32, 40, 128, "page pos head")])
def test_append(P, src, cache, page, kv_heads, dim, order):
    """Every row to its place, to the bit, and nothing else is touched."""
    import torch
    g, h = torch.Generator("cuda").manual_seed(5), torch.Generator().manual_seed(5)
    for new, kv in (([1, 1, 1, 1], [1, 17, 400, 256]), ([3, 0, 150, 40], [3, 0, 300, 41])):
        n_pages = sum(-(-n // page) for n in kv) + 2
        table = pu.tables(kv, page, n_pages, h)
        k, v = pu.pools(n_pages, page, kv_heads, dim, TYPES[cache], g, order)
        starts = [0]
        for n in new:
            starts.append(starts[-1] + n)
        wide = torch.randn(starts[-1] + 3, 2 * kv_heads + 1, dim, device="cuda", generator=g) * 300
        wide[0, 0, :8] = torch.tensor([math.inf, -math.inf, 1e9, 65519.0, 65520.0, 1e-8, 2.0 ** -25, 6e-8])
        wide = wide.to(TYPES[src])
        k_new, v_new = wide[:, :kv_heads], wide[:, kv_heads + 1:]
        want_k, want_v = k.clone(), v.clone()
        for s, (m, n) in enumerate(zip(new, kv)):
            for i in range(m):
                j = n - m + i
                want_k[table[s, j // page], j % page] = k_new[starts[s] + i].to(k.dtype)
                want_v[table[s, j // page], j % page] = v_new[starts[s] + i].to(v.dtype)
        i32 = dict(dtype=torch.int32, device="cuda")
        decode = new == [1] * 4
        batch = P.PagedBatch(table.cuda(), torch.tensor(kv, **i32), None if decode else torch.tensor(starts, **i32), starts[-1] + (0 if decode else 3))
        m = batch.n_tokens
        P.paged_kv_append(P.PagedCache(k, v), batch, k_new[:m], v_new[:m])
        assert torch.equal(k, want_k) and torch.equal(v, want_v)


def test_append_flags_what_has_no_place(P):
    import torch
    from runnburn_b200 import ops
    for kv, table, new in (([40], [[0, 1]], None), ([0], [[0, 1]], None), ([20], [[0, 9]], None), ([20], [[0, -1]], None), ([2], [[0, 1]], [0, 3])):
        k, v = torch.zeros(4, 16, 1, 64, device="cuda", dtype=torch.float16), torch.zeros(4, 16, 1, 64, device="cuda", dtype=torch.float16)
        i32 = dict(dtype=torch.int32, device="cuda")
        n = 1 if new is None else 3
        batch = P.PagedBatch(torch.tensor(table, **i32), torch.tensor(kv, **i32), None if new is None else torch.tensor(new, **i32), n)
        P.paged_kv_append(P.PagedCache(k, v), batch, torch.ones(n, 1, 64, device="cuda"), torch.ones(n, 1, 64, device="cuda"))
        torch.cuda.synchronize()
        assert ops.dev_error_flag() == P.DEVICE_BAD_PAGE
        assert int(k.sum()) == (2 * 64 if new else 64 if kv == [40] else 0)


@pytest.mark.parametrize("layers,order", [(1, "page pos head"), (3, "page pos head"), (2, "page head pos"), (2, "pos head page")])
@pytest.mark.parametrize("page,kv_heads,dim,pages,n", [(16, 8, 128, 40, 17), (8, 1, 8, 300, 140), (256, 3, 72, 9, 4), (64, 2, 64, 5000, 2500)])
def test_copy(P, layers, order, page, kv_heads, dim, pages, n):
    import torch
    g = torch.Generator().manual_seed(n)
    both = [pu.pools(pages, page, kv_heads, dim, torch.bfloat16, torch.Generator("cuda").manual_seed(i), order) for i in range(layers)]
    k, v = (torch.stack([b[i] for b in both]) if order == "page pos head" else torch.stack([b[i].permute(2, 0, 1, 3) for b in both]).permute(0, 2, 3, 1, 4) for i in range(2))
    if layers == 1:
        k, v = k[0], v[0]
    perm = torch.randperm(pages, generator=g)
    src, dst, rows = perm[:n].clone(), perm[n:2 * n], torch.randint(0, page + 1, (n,), generator=g)
    src[-1] = src[0]   # one page to two places
    for use in (None, rows):
        want_k, want_v = k.clone(), v.clone()
        for w, t in ((want_k, k), (want_v, v)):
            a = w if layers > 1 else w[None]
            b = t if layers > 1 else t[None]
            keep = torch.ones(n, page, dtype=torch.bool) if use is None else torch.arange(page) < use[:, None]
            a[:, dst.cuda()] = torch.where(keep.cuda()[None, :, :, None, None], b[:, src.cuda()], b[:, dst.cuda()])
        P.paged_kv_copy(P.PagedCache(k, v), src, dst, use)
        assert torch.equal(k, want_k) and torch.equal(v, want_v)


# ---- together -----------------------------------------------------------------------------------------------------------
def test_a_server_s_steps(P, ws):
    """Two prompts with a common beginning, then steps with window attention: append, attention, fork, copy on write, release, free and
    compaction, against sequences that are kept whole."""
    import torch
    g = torch.Generator("cuda").manual_seed(9)
    L, page, kvh, H, D, window, sinks, n_pages = 2, 16, 2, 8, 64, 40, 3, 30
    pool = torch.full((2, L, n_pages, page, kvh, D), math.nan, device="cuda", dtype=torch.bfloat16)
    cache, pages = P.PagedCache(pool[0], pool[1]), P.KvPages(n_pages, page)
    whole = {}   # seq -> rows [L][2][n][kvh][D]
    i32 = dict(dtype=torch.int32, device="cuda")

    def step(seqs, new):
        for s, n in zip(seqs, new):
            P.paged_kv_copy(cache, *pages.extend(s, n))
        table, lens = pages.tables(seqs)
        start = torch.tensor([0] + new).cumsum(0).to(torch.int32)
        batch = P.PagedBatch(torch.tensor(table, **i32), torch.tensor(lens, **i32), None if new == [1] * len(new) else start.cuda(), sum(new))
        for layer in range(L):
            q, k, v = (torch.randn(sum(new), h, D, device="cuda", generator=g).bfloat16() for h in (H, kvh, kvh))
            one = cache.layer(layer)
            P.paged_kv_append(one, batch, k, v)
            out = (P.attention_decode_paged if batch.q_start is None else P.attention_prefill_paged)(one, batch, q, D ** -0.5, window=window, sinks=sinks, workspace=ws)
            for i, s in enumerate(seqs):
                lo, hi = int(start[i]), int(start[i + 1])
                rows = whole.setdefault(s, [[torch.empty(0, kvh, D, device="cuda", dtype=torch.bfloat16)] * 2 for _ in range(L)])
                rows[layer] = [torch.cat([rows[layer][0], k[lo:hi]]), torch.cat([rows[layer][1], v[lo:hi]])]
                n = rows[layer][0].shape[0]
                one_page = -(-n // 8) * 8
                kk, vv = (torch.cat([t, torch.zeros(one_page - n, kvh, D, device="cuda", dtype=t.dtype)])[None] for t in rows[layer])
                want, _, mass = pu.attention(q[lo:hi], kk, vv, torch.zeros(1, 1, dtype=torch.int32), one_page, [n], [0, hi - lo], D ** -0.5, window, sinks)
                assert worst(out[lo:hi], want, tolerance(want, mass, out.dtype)) <= 1

    a, b = pages.new(), pages.new()
    step([a, b], [70, 21])
    c = pages.fork(a)
    whole[c] = [list(x) for x in whole[a]]
    step([a, b, c], [1, 1, 1])
    step([c], [19])
    for s in (a, b, c):
        pages.release(s, window, sinks)
    step([c, a, b], [1, 1, 1])
    pages.free(a)
    before = pages.info()["free_pages"]
    P.paged_kv_copy(cache, *pages.compact())
    assert pages.info()["free_pages"] == before
    for _ in range(3):
        step([b, c], [1, 1])
    d = pages.fork(c)
    whole[d] = [list(x) for x in whole[c]]
    step([d, b], [33, 7])
    step([c, d, b], [1, 1, 1])
