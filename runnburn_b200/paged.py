"""A key-value cache in pages: attention over it, its writes and copies, and the book-keeping of its pages.

The functions take device tensors of PyTorch (anything with its `data_ptr`, `shape`, `stride`, `dtype`, `device` and the like will do)
on the library's device (`ops.device_index()`), whatever device is current, and run on the given stream (a stream of PyTorch or its
handle), else on PyTorch's current one; they do not synchronise and allocate nothing but a missing `out`, so calls with `out` can be
captured into graphs once the library is open (`ops.open()`, or a `Workspace`).  A missing `out` is allocated on the stream that writes
it.  Tensors that the caller brings are used as they are: those of another stream than the call's have to be kept until it is through
(`record_stream`), as ever in PyTorch.  Tables, lengths and starts are read when the work runs.  What they hold is checked on the
device: a page outside the pool, a length that the table cannot hold or a start out of order sets the device error word
(`ops.dev_error_flag()` returns 5) instead of touching memory outside.  The C ABI behind it is declared in include/rnb_b200.h.

    pages = KvPages(n_pages, page_size)                    # host: who holds which page
    cache = PagedCache(k, v)                               # [n_pages, page_size, kv_heads, head_dim] each, any strides
    seq = pages.new()
    pages.extend(seq, n)                                   # room for n tokens (and a copy, where a fork shares the last page)
    table, kv_len = pages.tables([seq])                    # -> device
    batch = PagedBatch(table, kv_len, q_start)
    paged_kv_append(cache, batch, k_new, v_new)
    attention_prefill_paged(cache, batch, q, scale, out=out, workspace=workspace)
"""
from __future__ import annotations

import contextlib
import ctypes as C

import numpy as np

from . import _lib, ops
from ._lib import TYPE_BF16, TYPE_F16, TYPE_F32, check, load

DEVICE_BAD_PAGE, DEVICE_BAD_WORKSPACE = 5, 6   # what ops.dev_error_flag() tells of a call

_types: dict = {}
_I32 = np.dtype(np.int32)


def _type(t) -> int:
    """GGML type id of a tensor's element type."""
    if not _types:
        import torch
        _types.update({torch.float32: TYPE_F32, torch.float16: TYPE_F16, torch.bfloat16: TYPE_BF16})
    try:
        return _types[t.dtype]
    except KeyError:
        raise TypeError(f"expected float32, float16 or bfloat16, got {t.dtype}") from None


def _on_device(index: int, *tensors) -> None:
    for t in tensors:
        if t.get_device() != index:
            raise ValueError(f"tensors have to be on one CUDA device, got {t.device} and cuda:{index}")


def _index(t) -> int:
    if not t.is_cuda:
        raise ValueError(f"tensors have to be on a CUDA device, got {t.device}")
    return t.get_device()


def _library_index(t) -> int:
    """The tensor's device, which has to be the one that the library launches on."""
    index, own = _index(t), ops.device_index()
    if index != own:
        raise ValueError(f"the library runs on cuda:{own} (RNB_CUDA_DEVICE), got a tensor on {t.device}")
    return index


_raw_stream = None


def _stream(index: int, stream) -> int:
    """The stream's handle; None: the current one of PyTorch (asked for by its number alone where that is offered: an object for it takes 2 us)."""
    global _raw_stream
    if stream is not None:
        handle = getattr(stream, "cuda_stream", getattr(stream, "_as_parameter_", stream))
        return getattr(handle, "value", handle) or 0
    if _raw_stream is None:
        import torch
        _raw_stream = getattr(torch._C, "_cuda_getCurrentRawStream", None) or (lambda i: torch.cuda.current_stream(i).cuda_stream)
    return _raw_stream(index)


def _stream_object(index: int, handle: int):
    import torch
    return torch.cuda.ExternalStream(handle, device=index) if handle else torch.cuda.default_stream(index)


def _allocating(index: int, stream):
    """In this context PyTorch allocates memory in the order of `stream`, and takes it back in that order."""
    if stream is None:
        return contextlib.nullcontext()
    import torch
    return torch.cuda.stream(stream if isinstance(stream, torch.cuda.Stream) else _stream_object(index, _stream(index, stream)))


def _int(x, what: str):
    if not -2 ** 31 <= x < 2 ** 31:
        raise ValueError(f"{what}: {x} does not fit 32 bits")
    return x


def _ints(t, what: str, ndim: int):
    if str(t.dtype) != "torch.int32" or t.dim() != ndim or (t.shape[-1] > 1 and t.stride(-1) != 1):
        raise ValueError(f"{what} has to be an int32 tensor of {ndim} dimension(s), its last one contiguous")
    return t


class PagedCache:
    """The pools of a layer's keys and values, [n_pages, page_size, kv_heads, head_dim], or of several layers, [n_layers, ...]; strides are
    the tensors' own (the same for both), so views of one buffer and other orders of the dimensions are taken as they are."""

    def __init__(self, k, v):
        if k.dim() not in (4, 5) or k.shape != v.shape or k.stride() != v.stride() or k.dtype != v.dtype:
            raise ValueError("k and v have to be alike, [n_pages, page_size, kv_heads, head_dim] or with a dimension of layers before these")
        if k.shape[-1] > 1 and k.stride(-1) != 1:
            raise ValueError("the elements of a head's row have to be contiguous")
        self.index = _library_index(k)
        _on_device(self.index, v)
        self.k, self.v = k, v
        self.n_layers, self.layer_stride = (k.shape[0], k.stride(0)) if k.dim() == 5 else (1, 0)
        self.n_pages, self.page_size, self.kv_heads, self.head_dim = k.shape[-4:]
        page, pos, head = k.stride()[-4:-1]
        self._c = _lib.PagedCache(_type(k), self.head_dim, self.kv_heads, self.page_size, self.n_pages, page, pos, head, k.data_ptr(), v.data_ptr())
        self._ref = C.byref(self._c)

    def layer(self, i: int) -> "PagedCache":
        """The cache of one layer, for the calls that take one."""
        return PagedCache(self.k[i], self.v[i])

    def _one(self) -> None:
        if self.n_layers != 1:
            raise ValueError(f"this call takes the cache of one layer, layer(i) of these {self.n_layers}")


class PagedBatch:
    """Sequences of a call: their page tables [n_seq, max_pages], positions in the cache [n_seq] (the call's own tokens included) and, unless
    every sequence has one token, where their tokens start in the token matrices, [n_seq + 1]; all int32 on the device.  n_tokens: rows of
    the token matrices (needed with q_start; more rows than q_start[n_seq] are padding).  The tensors may change in place between calls."""

    def __init__(self, table, kv_len, q_start=None, n_tokens: int | None = None):
        _ints(table, "table", 2), _ints(kv_len, "kv_len", 1)
        n_seq = table.shape[0]
        if kv_len.shape[0] != n_seq:
            raise ValueError(f"table has {n_seq} sequences, kv_len {kv_len.shape[0]}")
        self.index = _index(table)
        _on_device(self.index, kv_len, *(() if q_start is None else (q_start,)))
        if q_start is not None:
            if _ints(q_start, "q_start", 1).shape[0] != n_seq + 1:
                raise ValueError(f"q_start has to have {n_seq + 1} entries, got {q_start.shape[0]}")
            if n_tokens is None:
                raise ValueError("n_tokens is needed with q_start")
        elif n_tokens is None:
            n_tokens = n_seq
        self.table, self.kv_len, self.q_start, self.n_tokens = table, kv_len, q_start, n_tokens
        stride = max(table.stride(0), table.shape[1]) if n_seq < 2 else table.stride(0)
        self._c = _lib.PagedBatch(table.data_ptr(), _int(stride, "table"), _int(table.shape[1], "table"), n_seq, _int(n_tokens, "n_tokens"), kv_len.data_ptr(),
                                  None if q_start is None else q_start.data_ptr())
        self._ref = C.byref(self._c)


class Workspace:
    """Scratch of the attention calls, on the library's device, allocated and initialised on the given stream; other streams wait for that at
    their first call (one that is being captured does not: begin the capture behind it).  Calls that may overlap on the GPU (other streams)
    need one each.  PyTorch's streams that use it are told to the allocator; work on a stream that is given by its handle has to be through
    before the workspace goes."""

    def __init__(self, device=None, stream=None):
        import torch
        device = torch.device("cuda", ops.device_index()) if device is None else torch.device(device)
        n = load().rnb_b200_paged_workspace_bytes()
        self._ready = None
        with torch.cuda.device(device), _allocating(device.index, stream):
            self.buffer = torch.empty(n, dtype=torch.uint8, device=device)
            self.index, self.ptr, self.bytes = _library_index(self.buffer), self.buffer.data_ptr(), n
            on = _stream(self.index, stream)
            check(load().rnb_b200_paged_workspace_init(self.ptr, n, on))
            if not torch.cuda.is_current_stream_capturing():
                self._ready = torch.cuda.current_stream(self.index).record_event()
        self._streams, self._handles = {on}, set()   # that have waited: PyTorch's, and bare handles

    def _used_on(self, handle: int, stream) -> None:
        """Another stream's first call."""
        import torch
        bare = stream is not None and (not isinstance(stream, torch.cuda.Stream) or isinstance(stream, torch.cuda.ExternalStream))
        if bare and handle in self._handles:
            return
        other = _stream_object(self.index, handle)
        with torch.cuda.stream(other):
            if torch.cuda.is_current_stream_capturing():
                return
        if self._ready is not None:
            other.wait_event(self._ready)
        if bare:   # (not told to the allocator: the stream may be gone by the time that it would be asked)
            self._handles.add(handle)
        else:
            self.buffer.record_stream(other)
            self._streams.add(handle)


def _rows(t, what: str, tokens: int, heads: int | None, dim: int):
    """[tokens, heads, dim] with contiguous heads; the stride from one token to the next."""
    shape = t.shape
    if len(shape) != 3 or shape[0] != tokens or shape[2] != dim or (heads is not None and shape[1] != heads):
        raise ValueError(f"{what} has to be [{tokens}, {heads or 'heads'}, {dim}], got {tuple(shape)}")
    a, b, c = t.stride()
    if c != 1 or (b != dim and shape[1] > 1):
        raise ValueError(f"{what}: the heads of a token have to be contiguous")
    return a if tokens > 1 else shape[1] * dim


def _attention(fn, cache, batch, q, scale, out, window, sinks, lse, workspace, stream):
    cache._one()
    n, dim = batch.n_tokens, cache.head_dim
    q_stride = _rows(q, "q", n, None, dim)
    heads = q.shape[1]
    if out is None:
        with _allocating(cache.index, stream):
            out = q.new_empty(q.shape)
    out_stride = _rows(out, "out", n, heads, dim)
    if out.dtype != q.dtype:
        raise ValueError(f"out has to have the queries' type {q.dtype}, got {out.dtype}")
    index = cache.index
    if batch.index != index or workspace.index != index or q.get_device() != index or out.get_device() != index:
        raise ValueError(f"cache, batch, workspace, q and out have to be on one CUDA device, got {index}, {batch.index}, {workspace.index}, {q.device} and {out.device}")
    if lse is not None:
        _on_device(index, lse)
        if str(lse.dtype) != "torch.float32" or tuple(lse.shape) != (n, heads) or not lse.is_contiguous():
            raise ValueError(f"lse has to be a contiguous float32 tensor [{n}, {heads}]")
        lse = lse.data_ptr()
    on = _stream(index, stream)
    if on not in workspace._streams:
        workspace._used_on(on, stream)
    check(fn(cache._ref, batch._ref, _type(q), q.data_ptr(), q_stride, heads, scale, _int(window, "window"), _int(sinks, "sinks"), workspace.ptr, workspace.bytes, out.data_ptr(), out_stride, lse, on))
    return out


def attention_decode_paged(cache: PagedCache, batch: PagedBatch, q, scale: float, *, workspace: Workspace, out=None, window: int = 0, sinks: int = 0, lse=None, stream=None):
    """Attention of one new token per sequence, q [n_seq, heads, head_dim]: softmax(scale q.K^T) V over the sequence's positions, with a
    window over its last `window` positions and its first `sinks`.  Returns `out` (as q); lse, float32 [n_seq, heads], receives the logarithms
    of the sums.  A sequence of length 0 gets zeros and -inf."""
    return _attention(load().rnb_b200_dev_attention_decode_paged, cache, batch, q, scale, out, window, sinks, lse, workspace, stream)


def attention_prefill_paged(cache: PagedCache, batch: PagedBatch, q, scale: float, *, workspace: Workspace, out=None, window: int = 0, sinks: int = 0, lse=None, stream=None):
    """Causal attention of the batch's tokens, q [n_tokens, heads, head_dim]: the last tokens of every sequence's positions are the call's, and
    a token at position p sees positions up to p (with a window, those after p - window and the first `sinks`)."""
    return _attention(load().rnb_b200_dev_attention_prefill_paged, cache, batch, q, scale, out, window, sinks, lse, workspace, stream)


def paged_kv_append(cache: PagedCache, batch: PagedBatch, k_new, v_new, *, stream=None) -> None:
    """Writes the rows of the batch's tokens, [n_tokens, kv_heads, head_dim], to their places in the pages, rounded to the cache's type."""
    cache._one()
    stride = _rows(k_new, "k_new", batch.n_tokens, cache.kv_heads, cache.head_dim)
    if _rows(v_new, "v_new", batch.n_tokens, cache.kv_heads, cache.head_dim) != stride or k_new.dtype != v_new.dtype:
        raise ValueError("k_new and v_new have to be alike")
    index = cache.index
    if batch.index != index or k_new.get_device() != index or v_new.get_device() != index:
        raise ValueError(f"cache, batch and rows have to be on one CUDA device, got {index}, {batch.index}, {k_new.device} and {v_new.device}")
    check(load().rnb_b200_dev_paged_kv_append(cache._ref, batch._ref, _type(k_new), k_new.data_ptr(), v_new.data_ptr(), stride, _stream(index, stream)))


def _host(a, what: str) -> np.ndarray:
    """A list of whole numbers as int32; what would be cut on the way is refused."""
    a = np.asarray(a)
    if a.dtype is _I32:
        return a if a.ndim == 1 and a.flags.c_contiguous else np.ascontiguousarray(a).ravel()
    if a.size:
        if a.dtype.kind not in "iu":
            raise TypeError(f"{what} has to hold whole numbers, got {a.dtype}")
        _int(a.min(), what), _int(a.max(), what)
    return np.ascontiguousarray(a, dtype=np.int32).ravel()


def paged_kv_copy(cache: PagedCache, src, dst, rows=None, *, stream=None) -> None:
    """Copies page src[i] to page dst[i] in all layers, its first rows[i] positions (None: all).  The lists are host integers.  A page may
    be copied to several places; one that is written must be written once and not read."""
    src, dst, rows = _host(src, "src"), _host(dst, "dst"), None if rows is None else _host(rows, "rows")
    if src.size != dst.size or (rows is not None and rows.size != src.size):
        raise ValueError("src, dst and rows have to be equally long")
    check(load().rnb_b200_dev_paged_kv_copy(cache._ref, cache.n_layers, cache.layer_stride, src.ctypes.data, dst.ctypes.data, None if rows is None else rows.ctypes.data,
                                            src.size, _stream(cache.index, stream)))


class KvPages:
    """Who holds which page, on the host.  Sequences are numbers; `extend` and `compact` return the copies, as (src, dst, rows) for
    `paged_kv_copy`, to make before the cache is used again."""

    def __init__(self, n_pages: int, page_size: int):
        h = C.c_void_p()
        check(load().rnb_b200_kv_pages_create(_int(n_pages, "n_pages"), _int(page_size, "page_size"), C.byref(h)))
        self._h, self.n_pages, self.page_size = h, n_pages, page_size

    def close(self) -> None:
        if getattr(self, "_h", None):
            load().rnb_b200_kv_pages_destroy(self._h)
            self._h = None

    __del__ = close

    def info(self) -> dict:
        i = _lib.KvPagesInfo()
        check(load().rnb_b200_kv_pages_get_info(self._h, C.byref(i)))
        return {n: getattr(i, n) for n, _ in i._fields_}

    def new(self) -> int:
        s = C.c_int32()
        check(load().rnb_b200_kv_pages_new(self._h, C.byref(s)))
        return s.value

    def extend(self, seq: int, n_new: int):
        """Room for n_new more positions; ([], [], []) or the one copy that parts a shared last page."""
        n, src, dst, rows = (C.c_int32() for _ in range(4))
        check(load().rnb_b200_kv_pages_extend(self._h, _int(seq, "seq"), _int(n_new, "n_new"), C.byref(n), C.byref(src), C.byref(dst), C.byref(rows)))
        return ([src.value], [dst.value], [rows.value]) if n.value else ([], [], [])

    def fork(self, seq: int) -> int:
        s = C.c_int32()
        check(load().rnb_b200_kv_pages_fork(self._h, _int(seq, "seq"), C.byref(s)))
        return s.value

    def truncate(self, seq: int, length: int) -> None:
        """Keeps the first `length` positions; refused where the next token would see a released page (by the last release's window and sinks)."""
        check(load().rnb_b200_kv_pages_truncate(self._h, _int(seq, "seq"), _int(length, "length")))

    def release(self, seq: int, window: int, sinks: int = 0) -> None:
        """Frees the pages that neither the window of the next token nor the sinks reach."""
        check(load().rnb_b200_kv_pages_release(self._h, _int(seq, "seq"), _int(window, "window"), _int(sinks, "sinks")))

    def free(self, seq: int) -> None:
        check(load().rnb_b200_kv_pages_free(self._h, _int(seq, "seq")))

    def compact(self):
        """Moves the used pages to the front of the pool; (src, dst, None)."""
        src, dst = (np.empty(max(1, self.n_pages // 2), np.int32) for _ in range(2))
        n = C.c_size_t()
        check(load().rnb_b200_kv_pages_compact(self._h, src.ctypes.data, dst.ctypes.data, self.n_pages // 2, C.byref(n)))
        return src[:n.value], dst[:n.value], None

    def tables(self, seqs, max_pages: int | None = None):
        """(int32 [n, max_pages], int32 [n]): page tables and lengths on the host, unused entries -1."""
        seqs = _host(seqs, "seqs")
        lens = np.empty(seqs.size, np.int32)
        check(load().rnb_b200_kv_pages_tables(self._h, seqs.ctypes.data, seqs.size, None, 0, lens.ctypes.data))
        if max_pages is None:
            max_pages = max(1, -(-int(lens.max(initial=0)) // self.page_size))
        _int(max_pages, "max_pages")
        table = np.empty((seqs.size, max_pages), np.int32)
        check(load().rnb_b200_kv_pages_tables(self._h, seqs.ctypes.data, seqs.size, table.ctypes.data, max_pages, lens.ctypes.data))   # both of one moment
        return table, lens
