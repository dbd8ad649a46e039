"""The paged cache without a GPU: book-keeping of the pages against a model of it, and calls that are refused before anything runs."""
import ctypes as C
import random

import numpy as np
import pytest


@pytest.fixture(scope="module")
def r():
    from runnburn_b200 import build
    build.build_library()
    import runnburn_b200
    return runnburn_b200


class Model:
    """What the pages hold, position by position: the cache is a dict (page, row) -> value."""

    def __init__(self, pages, r):
        self.p, self.r, self.cache, self.want = pages, r, {}, {}

    def copy(self, src, dst, rows):
        rows = [self.p.page_size] * len(src) if rows is None else rows
        assert not set(src) & set(dst) and len(set(dst)) == len(dst)
        for a, b, n in zip(src, dst, rows):
            for i in range(n):
                self.cache[b, i] = self.cache.get((a, i))

    def extend(self, seq, values):
        self.copy(*self.p.extend(seq, len(values)))
        table, lens = self.p.tables([seq])
        at = len(self.want[seq])
        assert lens[0] == at + len(values)
        for i, v in enumerate(values, at):
            page = table[0, i // self.p.page_size]
            assert 0 <= page < self.p.n_pages
            self.cache[page, i % self.p.page_size] = v
        self.want[seq] = self.want[seq] + list(values)

    def check(self):
        used = set()
        for s, want in self.want.items():
            table, lens = self.p.tables([s])
            assert lens[0] == len(want)
            for i, v in enumerate(want):
                page = int(table[0, i // self.p.page_size])
                if page < 0:
                    assert v is None or self.released.get(s, 0) > i
                    continue
                used.add(page)
                assert self.cache[page, i % self.p.page_size] == v
        info = self.p.info()
        assert info["free_pages"] == self.p.n_pages - len(used) and info["n_seqs"] == len(self.want)
        return used

    released: dict = {}


@pytest.mark.parametrize("seed", range(6))
@pytest.mark.parametrize("page", [8, 16])
def test_sequences_keep_what_they_hold(r, seed, page):
    rng, m = random.Random(seed * 31 + page), Model(r.paged.KvPages(60, page), r)
    stamp = iter(range(10 ** 9))
    for _ in range(400):
        seqs = list(m.want)
        act = rng.choice(["new", "extend", "extend", "extend", "fork", "truncate", "free", "compact"])
        if act == "new" and len(seqs) < 8:
            m.want[m.p.new()] = []
        elif act == "extend" and seqs:
            s = rng.choice(seqs)
            before = m.p.info()
            try:
                m.extend(s, [next(stamp) for _ in range(rng.choice([0, 1, 2, page, 3 * page + 1]))])
            except r.RnbError as e:
                assert e.status == 3 and "pages needed" in str(e) and m.p.info() == before
        elif act == "fork" and seqs and len(seqs) < 8:
            s = rng.choice(seqs)
            m.want[m.p.fork(s)] = list(m.want[s])
        elif act == "truncate" and seqs:
            s = rng.choice(seqs)
            n = rng.randint(0, len(m.want[s]))
            m.p.truncate(s, n)
            m.want[s] = m.want[s][:n]
        elif act == "free" and seqs and rng.random() < 0.5:
            s = rng.choice(seqs)
            m.p.free(s)
            del m.want[s]
        elif act == "compact":
            m.copy(*m.p.compact())
            used = m.check()
            assert used == set(range(len(used)))
        m.check()


@pytest.mark.parametrize("window,sinks,n", [(1, 0, 40), (5, 0, 40), (16, 3, 100), (30, 8, 100), (200, 4, 100), (100, 0, 100), (8, 99, 100), (8, 17, 64)])
def test_release_keeps_what_later_tokens_see(r, window, sinks, n):
    p = r.paged.KvPages(20, 8)
    s = p.new()
    p.extend(s, n)
    p.release(s, window, sinks)
    table, _ = p.tables([s])
    for i in range(-(-n // 8)):
        needed = any(j > n - window or j < sinks for j in range(8 * i, 8 * i + 8))   # seen from position n on, or still to be written
        assert (table[0, i] >= 0) == needed
    free = p.info()["free_pages"]
    p.release(s, window, sinks)
    assert p.info()["free_pages"] == free
    # the sequence goes on; its table is longer than what it holds
    p.extend(s, 24)
    assert p.tables([s])[1][0] == n + 24
    if table[0, 0] >= 0 and (table[0] < 0).any():
        first = int(np.argmax(table[0] < 0))
        with pytest.raises(r.RnbError, match="released page"):
            p.truncate(s, 8 * first + 3)
        p.truncate(s, 8 * first)
    p.free(s)
    assert p.info()["free_pages"] == 20


def seen_by_the_next_token(length, window, sinks):
    return [j for j in range(length) if j > length - window or j < sinks]


@pytest.mark.parametrize("window,sinks", [(1, 0), (5, 0), (16, 3), (16, 8), (30, 20), (33, 0)])
def test_truncate_keeps_what_the_next_token_sees(r, window, sinks):
    """Positions that are taken back bring the window back too: where it reaches a released page the sequence could not go on."""
    for n in (40, 100, 104):
        p = r.paged.KvPages(30, 8)
        for keep in range(n, -1, -1):
            s = p.new()
            p.extend(s, n)
            p.release(s, window, sinks)
            table = p.tables([s])[0][0]
            gone = any(table[j // 8] < 0 for j in seen_by_the_next_token(keep, window, sinks)) or (keep % 8 and table[keep // 8] < 0)
            if gone:
                before = p.info(), p.tables([s])[0].tolist()
                with pytest.raises(r.RnbError, match="released page") as e:
                    p.truncate(s, keep)
                assert e.value.status == 2 and (p.info(), p.tables([s])[0].tolist()) == before and p.tables([s])[1][0] == n
            else:
                p.truncate(s, keep)
                assert p.tables([s])[1][0] == keep
                f = p.fork(s)   # and its fork is bound by the same
                p.extend(f, 9)
                p.free(f)
            p.free(s)


def test_a_fork_remembers_what_was_released(r):
    p = r.paged.KvPages(30, 8)
    s = p.new()
    p.extend(s, 100)
    p.release(s, 16)
    f = p.fork(s)
    for x in (s, f):
        with pytest.raises(r.RnbError, match="released page"):
            p.truncate(x, 90)   # sees from 75 on, and 72 .. 79 are gone
        p.truncate(x, 96)
    p.free(s)
    t = p.new()   # the number of a freed sequence, without its past
    assert t == s
    p.extend(t, 100)
    p.truncate(t, 90)


@pytest.mark.parametrize("seed", range(6))
def test_sequences_under_a_window_can_always_go_on(r, seed):
    """Random steps with releases among them: what the next token sees is there, or the step was refused and changed nothing."""
    rng, m, window, sinks, page = random.Random(seed), Model(r.paged.KvPages(60, 8), r), 20 + seed, seed, 8
    stamp, told = iter(range(10 ** 9)), {}
    for _ in range(400):
        seqs = list(m.want)
        act = rng.choice(["new", "extend", "extend", "extend", "fork", "truncate", "release", "release", "free", "compact"])
        s = rng.choice(seqs) if seqs else None
        try:
            if act == "new" and len(seqs) < 8:
                s = m.p.new()
                m.want[s], told[s] = [], False
            elif act == "extend" and seqs:
                m.extend(s, [next(stamp) for _ in range(rng.choice([1, 2, page, 3 * page + 1]))])
            elif act == "fork" and seqs and len(seqs) < 8:
                f = m.p.fork(s)
                m.want[f], told[f] = list(m.want[s]), told[s]
            elif act == "release" and seqs:
                m.p.release(s, window, sinks)
                told[s] = True
            elif act == "truncate" and seqs:
                n = max(0, len(m.want[s]) - rng.choice([0, 1, 3, 9, 30]))
                m.p.truncate(s, n)
                m.want[s] = m.want[s][:n]
            elif act == "free" and seqs and rng.random() < 0.4:
                m.p.free(s)
                del m.want[s], told[s]
            elif act == "compact":
                m.copy(*m.p.compact())
        except r.RnbError as e:
            assert "pages needed" in str(e) or (act == "truncate" and "released page" in str(e))
        for s, want in m.want.items():
            table, lens = m.p.tables([s])
            assert lens[0] == len(want)
            for j in seen_by_the_next_token(len(want), window, sinks) if told[s] else range(len(want)):
                assert table[0, j // page] >= 0 and m.cache[int(table[0, j // page]), j % page] == want[j]


def test_shared_pages_are_freed_once(r):
    p = r.paged.KvPages(4, 8)
    a = p.new()
    p.extend(a, 12)
    b = p.fork(a)
    c = p.fork(b)
    assert p.info() == dict(n_pages=4, page_size=8, free_pages=2, n_seqs=3)
    assert p.extend(a, 1) == ([1], [2], [4])          # the others keep the page
    assert p.extend(b, 1) == ([1], [3], [4])
    assert p.extend(c, 1) == ([], [], [])             # nobody else is left on it
    with pytest.raises(r.RnbError) as e:
        p.extend(c, 9)
    assert e.value.status == 3
    p.free(a)
    p.free(a2 := p.fork(b))
    assert a2 == a and p.info()["free_pages"] == 1
    p.free(b), p.free(c)
    assert p.info()["free_pages"] == 4
    for call in (lambda: p.free(b), lambda: p.fork(7), lambda: p.extend(-1, 1), lambda: p.truncate(9, 0), lambda: p.release(b, 4), lambda: p.tables([b])):
        with pytest.raises(r.RnbError, match="no sequence"):
            call()


def test_book_keeping_refuses(r):
    L = r.load()
    for pages, size in ((0, 16), (-1, 16), (4, 0), (4, 4), (4, 24), (4, 512)):
        with pytest.raises(r.RnbError) as e:
            r.paged.KvPages(pages, size)
        assert e.value.status == 2
    p = r.paged.KvPages(8, 8)
    s = p.new()
    p.extend(s, 20)
    for call, what in ((lambda: p.truncate(s, 21), "cannot keep"), (lambda: p.truncate(s, -1), "cannot keep"), (lambda: p.release(s, 0), "window"),
                       (lambda: p.release(s, 4, -1), "sinks"), (lambda: p.extend(s, -1), "cannot add"), (lambda: p.extend(s, 2 ** 31 - 1), "cannot add"),
                       (lambda: p.tables([s], 2), "3 pages")):
        with pytest.raises(r.RnbError, match=what) as e:
            call()
        assert e.value.status == 2
    t = p.new()
    p.extend(t, 16)
    p.free(s)
    n = C.c_size_t()
    assert L.rnb_b200_kv_pages_compact(p._h, None, None, 0, C.byref(n)) == 2 and n.value == 2   # nothing moved for want of room
    assert p.tables([t])[0].tolist() == [[3, 4]]
    src, dst, _ = p.compact()
    assert (src.tolist(), dst.tolist()) == ([3, 4], [0, 1]) and p.tables([t])[0].tolist() == [[0, 1]]
    assert L.rnb_b200_kv_pages_create(4, 8, None) == 2 and L.rnb_b200_kv_pages_new(None, C.byref(n)) == 2


# ---- calls that are refused on the host: nothing here is read, the addresses are made up --------------------------------
ADDRESS = 0x10000


def cache(r, **kw):
    f = dict(type=1, head_dim=128, kv_heads=2, page_size=16, n_pages=10, page_stride=4096, pos_stride=256, head_stride=128, k=ADDRESS, v=ADDRESS) | kw
    return r._lib.PagedCache(*[f[n] for n, _ in r._lib.PagedCache._fields_])


def batch(r, **kw):
    f = dict(table=ADDRESS, table_stride=4, max_pages=4, n_seq=2, n_tokens=2, kv_len=ADDRESS, q_start=None) | kw
    return r._lib.PagedBatch(*[f[n] for n, _ in r._lib.PagedBatch._fields_])


BAD_CACHE = [
    (dict(type=0), 1, "F16 or BF16"), (dict(type=8), 1, "F16 or BF16"), (dict(head_dim=4), 2, "head_dim"), (dict(head_dim=132), 2, "head_dim"),
    (dict(head_dim=520), 2, "head_dim"), (dict(kv_heads=0), 2, "kv_heads"), (dict(page_size=4), 2, "page_size"), (dict(page_size=24), 2, "page_size"),
    (dict(page_size=512), 2, "page_size"), (dict(n_pages=0), 2, "n_pages"), (dict(k=None), 2, "null"), (dict(v=None), 2, "null"), (dict(k=ADDRESS + 8), 2, "16-byte"),
    (dict(v=ADDRESS + 2), 2, "16-byte"), (dict(pos_stride=260), 2, "strides"), (dict(page_stride=2 ** 40), 2, "strides"), (dict(head_stride=64), 2, "overlap"),
    (dict(pos_stride=128), 2, "overlap"), (dict(page_stride=4088), 2, "overlap"), (dict(pos_stride=0), 2, "overlap"),
]
# strides that are never stepped, of one head or one page, say nothing
FINE_CACHE = [dict(kv_heads=1, head_stride=0), dict(kv_heads=1, head_stride=5), dict(kv_heads=1, head_stride=1 << 40), dict(n_pages=1, page_stride=12), dict(n_pages=1, page_stride=0),
              dict(n_pages=1, page_stride=3, kv_heads=1, head_stride=1)]
BAD_BATCH = [
    (dict(n_seq=-1), 2, "negative"), (dict(n_tokens=-1), 2, "negative"), (dict(n_tokens=3), 2, "one token per sequence"), (dict(table=None), 2, "null"),
    (dict(kv_len=None), 2, "null"), (dict(max_pages=0), 2, "max_pages"), (dict(table_stride=3), 2, "table_stride"), (dict(table=ADDRESS + 2), 2, "4-byte"),
    (dict(kv_len=ADDRESS + 1), 2, "4-byte"), (dict(q_start=ADDRESS + 2, n_tokens=9), 2, "4-byte"),
]


def attend(L, c, b, q_type=0, q=ADDRESS, q_stride=512, heads=4, scale=0.1, window=0, sinks=0, ws=ADDRESS, ws_bytes=None, out=ADDRESS + (1 << 20), out_stride=512, lse=None, prefill=False):
    fn = L.rnb_b200_dev_attention_prefill_paged if prefill else L.rnb_b200_dev_attention_decode_paged
    n = L.rnb_b200_paged_workspace_bytes() if ws_bytes is None else ws_bytes
    return fn(C.byref(c) if c else None, C.byref(b) if b else None, q_type, q, q_stride, heads, scale, window, sinks, ws, n, out, out_stride, lse, None)


def refused(L, rc, status, what):
    assert rc == status and what in L.rnb_b200_last_error().decode(), (rc, L.rnb_b200_last_error())


@pytest.mark.parametrize("kw,status,what", BAD_CACHE)
def test_a_bad_cache_is_refused(r, kw, status, what):
    L, c, b, one = r.load(), cache(r, **kw), batch(r), np.zeros(1, np.int32)
    refused(L, attend(L, c, b), status, what)
    refused(L, attend(L, c, b, prefill=True), status, what)
    refused(L, L.rnb_b200_dev_paged_kv_append(C.byref(c), C.byref(b), 0, ADDRESS, ADDRESS, 256, None), status, what)
    refused(L, L.rnb_b200_dev_paged_kv_copy(C.byref(c), 1, 0, one.ctypes.data, one.ctypes.data, None, 1, None), status, what)


@pytest.mark.parametrize("kw", FINE_CACHE)
def test_strides_that_are_never_stepped_may_be_anything(r, kw):
    """What is let through stops at the next check, the one for a sequence's one token, or of the batch."""
    L, c, one = r.load(), cache(r, **kw), np.zeros(1, np.int32)
    refused(L, attend(L, c, batch(r, q_start=ADDRESS)), 2, "q_start must be null")
    refused(L, L.rnb_b200_dev_paged_kv_append(C.byref(c), C.byref(batch(r, n_seq=-1)), 0, ADDRESS, ADDRESS, 256, None), 2, "negative")
    refused(L, L.rnb_b200_dev_paged_kv_copy(C.byref(c), 1, 0, one.ctypes.data, one.ctypes.data, None, 1, None), 2, "read and written")


@pytest.mark.parametrize("kw,status,what", BAD_BATCH)
def test_a_bad_batch_is_refused(r, kw, status, what):
    L, c, b = r.load(), cache(r), batch(r, **kw)
    refused(L, attend(L, c, b, prefill=b.q_start is not None), status, what)
    refused(L, L.rnb_b200_dev_paged_kv_append(C.byref(c), C.byref(b), 0, ADDRESS, ADDRESS, 256, None), status, what)


@pytest.mark.parametrize("kw,status,what", [
    (dict(q_type=30), 1, "queries"), (dict(q_type=12), 1, "queries"), (dict(q=None), 2, "null"), (dict(out=None), 2, "null"), (dict(heads=0), 2, "multiple of num_kv_heads"),
    (dict(heads=3), 2, "multiple of num_kv_heads"), (dict(heads=65536), 2, "num_heads"), (dict(q=ADDRESS + 8), 2, "16-byte"), (dict(out=ADDRESS + 4), 2, "16-byte"),
    (dict(q_stride=516), 2, "multiples of 8"), (dict(out_stride=516), 2, "multiples of 8"), (dict(q_stride=504), 2, "at least"), (dict(out_stride=256), 2, "at least"),
    (dict(lse=ADDRESS + 2), 2, "lse"), (dict(window=-1), 2, "window"), (dict(sinks=-1), 2, "sinks"), (dict(scale=float("nan")), 2, "scale"),
    (dict(scale=float("inf")), 2, "scale"), (dict(ws=None), 2, "workspace"), (dict(ws=ADDRESS + 64), 2, "workspace"), (dict(ws_bytes=100), 2, "workspace"),
])
def test_attention_refuses(r, kw, status, what):
    L = r.load()
    for prefill in (False, True):
        refused(L, attend(L, cache(r), batch(r), prefill=prefill, **kw), status, what)


@pytest.mark.parametrize("scale,fine", [(3e38, False), (-3e38, False), (2.4e38, False), (2.3e38, True), (-2.3e38, True), (0.0, True), (-float("inf"), False)])
def test_scales_up_to_the_end_of_f32(r, scale, fine):
    """Scores are counted in powers of two: the scale times log2 e has to be a number.  What is let through stops at the check behind it."""
    L = r.load()
    refused(L, attend(L, cache(r), batch(r), scale=scale, ws=None), 2, "workspace" if fine else "scale")


@pytest.mark.parametrize("tokens,q_stride,out_stride,shift,ok", [
    (2, 512, 512, 0, False), (2, 512, 512, 2048, False), (2, 512, 512, 4096, True), (2, 512, 512, -4096, True), (2, 512, 512, -4080, False), (1, 512, 512, 2048, True),
    (1, 512, 512, 2032, False), (5, 1024, 1024, 2048, True), (5, 1024, 1024, -2048, True), (5, 1024, 1024, 2064, False), (5, 1024, 1024, 4096 * 3 + 2048, True),
    (5, 1024, 1024, 2032, False), (5, 1024, 1032, 2048, False), (5, 1536, 1536, 2064, True), (5, 1536, 1536, 4112, False)])
def test_queries_and_outputs_must_not_overlap(r, tokens, q_stride, out_stride, shift, ok):
    """Rows of 4 * 128 f32, side by side in one matrix or apart; what is let through stops at the next check, the one for a sequence's one token."""
    L, base = r.load(), ADDRESS + (1 << 20)
    rc = attend(L, cache(r), batch(r, n_seq=tokens, n_tokens=tokens, q_start=ADDRESS), q=base, out=base + shift, q_stride=q_stride, out_stride=out_stride)
    refused(L, rc, 2, "q_start" if ok else "overlap")


def test_calls_refuse_what_only_they_can_see(r):
    L = r.load()
    refused(L, attend(L, None, batch(r)), 2, "null")
    refused(L, attend(L, cache(r), None), 2, "null")
    refused(L, attend(L, cache(r, head_dim=96, head_stride=96, pos_stride=192, page_stride=192 * 16), batch(r)), 1, "head_dim must be 64 or 128")
    refused(L, attend(L, cache(r, type=30), batch(r), q_type=0), 1, "queries")
    refused(L, attend(L, cache(r), batch(r, q_start=ADDRESS)), 2, "q_start must be null")
    append = lambda *a: L.rnb_b200_dev_paged_kv_append(C.byref(cache(r)), C.byref(batch(r)), *a, None)  # noqa: E731
    refused(L, append(30, ADDRESS, ADDRESS, 256), 1, "F32 or of the cache's type")
    refused(L, append(0, None, ADDRESS, 256), 2, "null")
    refused(L, append(0, ADDRESS, None, 256), 2, "null")
    refused(L, append(0, ADDRESS + 4, ADDRESS, 256), 2, "16-byte")
    refused(L, append(0, ADDRESS, ADDRESS, 252), 2, "multiple of 8")
    refused(L, append(0, ADDRESS, ADDRESS, 128), 2, "smaller than a token")
    refused(L, L.rnb_b200_paged_workspace_init(None, 1 << 30, None), 2, "workspace")
    refused(L, L.rnb_b200_paged_workspace_init(ADDRESS, 8, None), 2, "workspace")


@pytest.mark.parametrize("src,dst,rows,what", [
    ([0], [10], None, "the pool has 10"), ([-1], [2], None, "the pool has 10"), ([0], [0], None, "read and written"), ([0, 1], [2, 2], None, "written twice"),
    ([0, 1], [1, 2], None, "read and written"), ([1, 0], [2, 1], None, "read and written"), ([0], [1], [17], "17 positions"), ([0], [1], [-1], "-1 positions"),
    ([0] * 11, list(range(11)), None, "more copies than pages"),
])
def test_copies_refuse(r, src, dst, rows, what):
    L = r.load()
    a = [np.asarray(x, np.int32) if x is not None else None for x in (src, dst, rows)]
    refused(L, L.rnb_b200_dev_paged_kv_copy(C.byref(cache(r)), 1, 0, a[0].ctypes.data, a[1].ctypes.data, a[2].ctypes.data if rows else None, len(src), None), 2, what)


@pytest.mark.parametrize("bad,error", [
    (np.array([0, 2 ** 32 + 1]), ValueError), (np.array([0, -2 ** 32 + 1]), ValueError), (np.array([0, 2 ** 31], np.uint64), ValueError), ([0, 2 ** 32 + 1], ValueError),
    (np.array([0.0, 1.0]), TypeError), ([0, 1.5], TypeError), (np.array([False, True]), TypeError), ([0, 2 ** 70], TypeError), (["0", "1"], TypeError)])
def test_lists_are_whole_numbers_of_32_bits(r, bad, error):
    """Cut to 32 bits, or to whole numbers, they would be pages and sequences that nobody named."""
    here = r.ops.device_index()
    cache, p = r.paged.PagedCache(OnDevice(here), OnDevice(here)), r.paged.KvPages(8, 8)
    p.extend(p.new(), 5), p.extend(p.new(), 6)
    good = [2, 3]
    for lists in ((bad, good, None), (good, bad, None), ([0, 1], good, bad)):
        with pytest.raises(error, match="src|dst|rows"):
            r.paged.paged_kv_copy(cache, *lists)
    with pytest.raises(error, match="seqs"):
        p.tables(bad)
    import torch
    for fine in ([0, 1], np.array([0, 1]), np.array([0, 1], np.uint8), torch.tensor([0, 1])):
        assert p.tables(fine)[1].tolist() == [5, 6]
    assert p.tables([])[0].shape == (0, 1)


def test_numbers_of_more_than_32_bits_are_refused(r):
    """Cut to 32 bits they would be other ones."""
    p = r.paged.KvPages(8, 8)
    s = p.new()
    p.extend(s, 20)
    far = 2 ** 32
    for call in (lambda: p.extend(s, far + 1), lambda: p.extend(far + s, 1), lambda: p.truncate(s, far + 8), lambda: p.release(s, far + 4), lambda: p.release(s, 4, far),
                 lambda: p.fork(far + s), lambda: p.free(far + s), lambda: r.paged.KvPages(far + 8, 8), lambda: r.paged.KvPages(8, far + 8), lambda: p.tables([s], far + 3)):
        with pytest.raises(ValueError, match="32 bits"):
            call()
    assert p.info() == dict(n_pages=8, page_size=8, free_pages=5, n_seqs=1)
    import torch
    here = r.ops.device_index()
    table, lens, start = (OnDevice(here, shape, torch.int32) for shape in ((2, 4), (2,), (3,)))
    assert r.paged.PagedBatch(table, lens, start, 9).n_tokens == 9
    with pytest.raises(ValueError, match="32 bits"):
        r.paged.PagedBatch(table, lens, start, far + 9)


def test_tables_and_lengths_are_of_one_moment(r, monkeypatch):
    """Another thread may shorten a sequence while its table is asked for."""
    p = r.paged.KvPages(8, 8)
    s = p.new()
    p.extend(s, 40)
    real, calls = r.paged.load(), []

    class Between:
        """Takes positions back behind the first question for tables."""
        def __getattr__(self, name):
            f = getattr(real, name)
            if name != "rnb_b200_kv_pages_tables":
                return f

            def asked(*a):
                rc = f(*a)
                if not calls:
                    calls.append(1)
                    assert real.rnb_b200_kv_pages_truncate(p._h, s, 10) == 0
                return rc
            return asked
    monkeypatch.setattr(r.paged, "load", lambda: Between())
    table, lens = p.tables([s])
    assert calls and lens[0] in (10, 40) and (table[0] >= 0).sum() == -(-lens[0] // 8)


def test_copies_refuse_bad_layers(r):
    L, z = r.load(), np.array([0, 1], np.int32)
    for layers, stride in ((0, 0), (40000, 1 << 20), (2, 0), (2, 12), (2, 1 << 40), (1, (1 << 64) - 8)):
        refused(L, L.rnb_b200_dev_paged_kv_copy(C.byref(cache(r)), layers, stride, z[:1].ctypes.data, z[1:].ctypes.data, None, 1, None), 2, "layer")


class OnDevice:
    """As much of a tensor on a CUDA device as is looked at before anything runs."""
    is_cuda = True

    def __init__(self, index, shape=(4, 16, 2, 64), dtype=None):
        import torch
        self.index, self.like, self.device = index, torch.empty(shape, dtype=dtype or torch.float16), f"cuda:{index}"
        self.shape, self.dtype, self.dim, self.stride = self.like.shape, self.like.dtype, self.like.dim, self.like.stride

    def get_device(self):
        return self.index

    def data_ptr(self):
        return ADDRESS


def test_tensors_on_another_device_than_the_library_s_are_refused(r):
    """The launch goes to the library's device, whatever device the tensors are on."""
    here = r.ops.device_index()
    assert r.paged.PagedCache(OnDevice(here), OnDevice(here)).index == here
    with pytest.raises(ValueError, match=f"runs on cuda:{here}.*cuda:{here + 1}"):
        r.paged.PagedCache(OnDevice(here + 1), OnDevice(here + 1))
    with pytest.raises(ValueError, match="one CUDA device"):
        r.paged.PagedCache(OnDevice(here), OnDevice(here + 1))


def test_calls_of_one_layer_refuse_a_cache_of_several(r):
    """They would take the first one, whichever was meant."""
    import torch
    here = r.ops.device_index()
    at = lambda *shape, t=torch.float16: OnDevice(here, shape, t)  # noqa: E731
    cache = r.paged.PagedCache(at(3, 4, 16, 2, 64), at(3, 4, 16, 2, 64))
    assert cache.n_layers == 3
    batch = r.paged.PagedBatch(at(2, 4, t=torch.int32), at(2, t=torch.int32))
    rows = at(2, 2, 64)
    for call in (lambda: r.paged.attention_decode_paged(cache, batch, rows, 0.1, workspace=None, out=rows), lambda: r.paged.paged_kv_append(cache, batch, rows, rows),
                 lambda: r.paged.attention_prefill_paged(cache, batch, rows, 0.1, workspace=None, out=rows)):
        with pytest.raises(ValueError, match=r"layer\(i\)"):
            call()


def test_a_stream_is_any_object_that_stands_for_one(r):
    class Torch:
        cuda_stream = 77

    class Foreign:
        _as_parameter_ = C.c_void_p(78)
    for stream, handle in ((Torch(), 77), (Foreign(), 78), (79, 79), (C.c_void_p(80), 80), (C.c_void_p(), 0), (0, 0)):
        assert r.paged._stream(0, stream) == handle


def test_the_device_is_the_one_that_would_be_opened(r):
    """Asked for in a process of its own, where nothing is open."""
    import os
    import subprocess
    import sys
    for env, want in ((None, "0"), ("3", "3")):
        e = {k: v for k, v in os.environ.items() if k != "RNB_CUDA_DEVICE"} | ({"RNB_CUDA_DEVICE": env} if env else {})
        got = subprocess.run([sys.executable, "-c", "from runnburn_b200 import ops; print(ops.device_index())"], capture_output=True, text=True, env=e, cwd=r._lib.PKG.parent)
        assert got.stdout.strip() == want, got.stderr


def places(strides, counts, dim):
    """Every element of a pool."""
    import itertools
    return {sum(i * s for i, s in zip(at, strides)) + e for at in itertools.product(*map(range, counts)) for e in range(dim)}


@pytest.mark.parametrize("seed", range(4))
def test_what_is_written_must_not_overlap(r, seed):
    """Layers and the pools of keys and values, wherever they lie: side by side, one in the gaps of the other, or on top of each other in part."""
    import torch
    if torch.cuda.is_available():
        pytest.skip("the addresses are made up, and a call that is let through would run")
    rng, L, n_free, n_met = random.Random(seed), r.load(), 0, 0
    a, b = np.zeros(1, np.int32), np.ones(1, np.int32)
    for _ in range(400):
        counts = [rng.choice([1, 2, 3]), rng.choice([2, 3]), 8, rng.choice([1, 2])]   # layers, pages, positions, heads
        strides, span = [0] * 4, 8
        for i in rng.sample(range(4), 4):
            strides[i] = span + rng.choice([0, 0, 8, 24])
            span = strides[i] * (counts[i] - 1) + span if counts[i] > 1 else span
        if rng.random() < 0.3:
            strides[0] = 8 * rng.randint(1, span // 8)   # layers anywhere
        shift = 8 * rng.choice([0, 1, rng.randint(0, span // 8 + 2), rng.randint(0, 40)]) * rng.choice([-1, 1])
        c = cache(r, head_dim=8, kv_heads=counts[3], page_size=8, n_pages=counts[1], page_stride=strides[1], pos_stride=strides[2], head_stride=strides[3],
                  k=ADDRESS + (1 << 20), v=ADDRESS + (1 << 20) + 2 * shift)
        for layers in {1, counts[0]}:
            n = [layers] + counts[1:]
            keys = places(strides, n, 8)
            met = not keys.isdisjoint(x + shift for x in keys) or len(keys) < 8 * n[0] * n[1] * n[2] * n[3]
            rc = L.rnb_b200_dev_paged_kv_copy(C.byref(c), layers, strides[0], a.ctypes.data, b.ctypes.data, None, 1, None) if counts[1] > 1 else None
            said = L.rnb_b200_last_error().decode()
            if met:
                assert rc == 2 and "overlap" in said, (n, strides, shift, said)
                n_met += 1
            elif "overlap" in said and rc == 2:   # layers that lie between others without a common element, but not one level inside the next
                assert "layers" in said and strides[0] < span, (n, strides, shift, said)
            else:
                assert rc != 2, (n, strides, shift, said)   # without a GPU the call ends behind its checks
                n_free += 1
            if layers == 1:
                rc = L.rnb_b200_dev_paged_kv_append(C.byref(c), C.byref(batch(r)), 0, ADDRESS, ADDRESS, 8 * counts[3], None)
                assert (rc == 2 and "overlap" in L.rnb_b200_last_error().decode()) == met
    assert n_free > 100 and n_met > 100


def test_nothing_to_do_is_no_call(r):
    """No tokens, no sequences, no copies: fine without a GPU."""
    L = r.load()
    assert attend(L, cache(r), batch(r, n_seq=0, n_tokens=0, table=None, kv_len=None), q=None, out=None) == 0
    assert attend(L, cache(r), batch(r, n_tokens=0, q_start=ADDRESS), prefill=True) == 0
    assert L.rnb_b200_dev_paged_kv_append(C.byref(cache(r)), C.byref(batch(r, n_seq=0, n_tokens=0)), 0, None, None, 0, None) == 0
    assert L.rnb_b200_dev_paged_kv_copy(C.byref(cache(r)), 1, 0, None, None, None, 0, None) == 0
