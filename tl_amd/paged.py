"""A paged KV cache for several sequences, over the C ABI's launchers and page book.

``PageBook`` is the host's book of pages (open / fork / grow / cut / close / compact), ``PagedKV``
a cache that owns its pools, keeps the book in step with them and runs the attention:

    kv = PagedKV(dev, n_pages=256, page_size=64, n_kv_heads=8, head_dim=128)
    a = kv.open()
    kv.append([a], [5], k, v)              # k, v [5, 8, 128]: a prompt of five tokens
    out = kv.prefill([a], [5], q, scale)   # q [5, 32, 128]
    b = kv.fork(a)                         # shares a's pages
    kv.append([a, b], [1, 1], k1, v1)      # the shared tail page is copied first
    out = kv.decode([a, b], q1, scale)

The reference keeps one dense sequence per cache (KVCache, system.rs:387-600) and has no
counterpart.  Row t of every call belongs to the sequences in the order given; a sequence appears
once per call.
"""
import ctypes as C

import numpy as np

from . import _lib
from .device import F16, BackendError, _raise


def _i32(values):
    return np.ascontiguousarray(values, dtype=np.int32)


class PageBook:
    """The host's book: which pages each sequence holds (tl_hip_page_book_*)."""

    def __init__(self, n_pages, page_size):
        self.lib = _lib.load()
        self.page_size = int(page_size)
        self.n_pages = int(n_pages)
        self._h = self.lib.tl_hip_page_book_new(n_pages, page_size)
        if not self._h:
            _raise(self.lib)

    def _check(self, rc):
        if rc:
            _raise(self.lib)

    def _count(self, n):
        if n < 0:
            _raise(self.lib)
        return int(n)

    def open(self):
        return self._count(self.lib.tl_hip_page_book_open(self._h))

    def fork(self, seq):
        return self._count(self.lib.tl_hip_page_book_fork(self._h, seq))

    def close(self, seq):
        self._check(self.lib.tl_hip_page_book_close(self._h, seq))

    def grow(self, seq, n_tokens):
        """Room for n_tokens more positions; the (source, destination) pairs to copy first."""
        src, dst, n = C.c_int32(), C.c_int32(), C.c_int64()
        self._check(self.lib.tl_hip_page_book_grow(self._h, seq, n_tokens, C.byref(src), C.byref(dst), C.byref(n)))
        return [(src.value, dst.value)] if n.value else []

    def cut(self, seq, length):
        self._check(self.lib.tl_hip_page_book_cut(self._h, seq, length))

    def compact(self):
        """The used pages moved down to pages 0 .. used - 1; the pairs to copy."""
        room = self.n_pages - self.free_pages
        src, dst, n = *np.empty((2, max(room, 1)), dtype=np.int32), C.c_int64()
        self._check(self.lib.tl_hip_page_book_compact(self._h, src.ctypes.data_as(_lib.i32p),
                                                      dst.ctypes.data_as(_lib.i32p), room, C.byref(n)))
        return list(zip(src[: n.value].tolist(), dst[: n.value].tolist()))

    def length(self, seq):
        return self._count(self.lib.tl_hip_page_book_length(self._h, seq))

    @property
    def free_pages(self):
        return self._count(self.lib.tl_hip_page_book_free_pages(self._h))

    def row(self, seq, capacity):
        row = np.empty(max(capacity, 1), dtype=np.int32)
        self._check(self.lib.tl_hip_page_book_row(self._h, seq, row.ctypes.data_as(_lib.i32p), capacity))
        return row[:capacity]

    def release(self):
        if self._h:
            self.lib.tl_hip_page_book_release(self._h)
            self._h = None

    def __del__(self):
        try:
            self.release()
        except Exception:
            pass


class PagedKV:
    """Pools of pages on the device, one layer, with their book."""

    def __init__(self, dev, n_pages, page_size, n_kv_heads, head_dim, dtype=F16):
        self.dev, self.lib = dev, dev.lib
        self.book = PageBook(n_pages, page_size)
        self.n_kv_heads, self.head_dim, self.dtype = int(n_kv_heads), int(head_dim), dtype
        shape = (n_pages, n_kv_heads, page_size, head_dim)
        self.k, self.v = dev.tensor_zeros(shape, dtype), dev.tensor_zeros(shape, dtype)

    # -- the book's calls, their copies carried out at once
    def open(self):
        return self.book.open()

    def fork(self, seq):
        return self.book.fork(seq)

    def close(self, seq):
        self.book.close(seq)

    def cut(self, seq, length):
        self.book.cut(seq, length)

    def length(self, seq):
        return self.book.length(seq)

    def compact(self):
        self._copy(self.book.compact())

    def _check(self, rc):
        if rc:
            _raise(self.lib)

    def _copy(self, pairs):
        if pairs:
            src, dst = _i32([p[0] for p in pairs]), _i32([p[1] for p in pairs])
            page = self.n_kv_heads * self.book.page_size * self.head_dim * (2 if self.dtype == F16 else 4)
            self._check(self.lib.tl_hip_launch_kv_copy_pages(
                self.k.data_ptr, self.v.data_ptr, 1, self.book.n_pages, page, src.ctypes.data_as(_lib.i32p),
                dst.ctypes.data_as(_lib.i32p), len(pairs), self.lib.tl_hip_stream()))

    def _tables(self, seqs, counts):
        """The tensor that holds them, device addresses of the page table, cu_seqlens and kv_lens of
        these sequences, and the table's width."""
        if len(set(seqs)) != len(seqs) or len(counts) != len(seqs) or min([0, *counts]) < 0:
            raise BackendError(8, "ArgumentError: a sequence appears once per call, with its number of rows")
        lens = [self.book.length(s) for s in seqs]
        width = max([1] + [-(-n // self.book.page_size) for n in lens])
        rows = [self.book.row(s, width) for s in seqs]
        ints = _i32(np.concatenate([_i32(np.cumsum([0] + list(counts))), _i32(lens)] + rows))
        # a tensor of the library's allocator: its memory is reused in stream order only
        held = self.dev.tensor_new(ints.view(np.float32))
        cu, n = held.data_ptr, len(seqs)
        return held, cu + 4 * (2 * n + 1), cu, cu + 4 * (n + 1), width

    def append(self, seqs, counts, k, v):
        """counts[i] new positions for seqs[i]: k, v [sum(counts), n_kv_heads, head_dim]."""
        total, seqs = int(sum(counts)), list(seqs)
        if len(counts) != len(seqs) or k.shape != (total, self.n_kv_heads, self.head_dim) or v.shape != k.shape:
            raise BackendError(1, f"ShapeMismatch: rows {k.shape}, {v.shape} for {total} positions of {self.n_kv_heads} heads of {self.head_dim}")
        if k.dtype != v.dtype:
            raise BackendError(7, "TypeMismatch: k and v of one dtype")
        if len(set(seqs)) != len(seqs):
            raise BackendError(8, "ArgumentError: a sequence appears once per call")
        before, grown = [self.book.length(s) for s in seqs], 0
        try:
            for s, n in zip(seqs, counts):
                pairs = self.book.grow(s, n)
                grown += 1
                self._copy(pairs)
            held, table, cu, lens, width = self._tables(seqs, counts)
            row = self.n_kv_heads * self.head_dim
            self._check(self.lib.tl_hip_launch_kv_append(
                k.data_ptr, v.data_ptr, k.dtype, row, row, self.k.data_ptr, self.v.data_ptr, self.dtype, self.book.n_pages,
                self.book.page_size, self.n_kv_heads, self.head_dim, table, width, cu, lens, len(seqs), total,
                self.lib.tl_hip_stream()))
        except Exception:
            for s, was in zip(seqs[:grown], before):
                self.book.cut(s, was)
            raise

    def _rows(self, q, total):
        if len(q.shape) != 3 or q.shape[0] != total or q.shape[2] != self.head_dim:
            raise BackendError(1, f"ShapeMismatch: q {q.shape} for {total} rows of head size {self.head_dim}")
        return q.shape[1], self.dev.tensor_zeros(q.shape, q.dtype)

    def decode(self, seqs, q, scale):
        """q [len(seqs), n_heads, head_dim], the newest position of each -> the same shape."""
        seqs = list(seqs)
        heads, out = self._rows(q, len(seqs))
        held, table, _, lens, width = self._tables(seqs, [1] * len(seqs))
        self._check(self.lib.tl_hip_launch_paged_attention_decode(
            q.data_ptr, q.dtype, heads * self.head_dim, self.k.data_ptr, self.v.data_ptr, self.dtype, self.book.n_pages,
            self.book.page_size, heads, self.n_kv_heads, self.head_dim, table, width, lens, len(seqs), out.data_ptr, scale,
            None, 0, self.lib.tl_hip_stream()))
        return out

    def prefill(self, seqs, counts, q, scale):
        """q [sum(counts), n_heads, head_dim]: the last counts[i] positions of seqs[i], causal."""
        total, seqs = int(sum(counts)), list(seqs)
        heads, out = self._rows(q, total)
        held, table, cu, lens, width = self._tables(seqs, counts)
        self._check(self.lib.tl_hip_launch_paged_attention_prefill(
            q.data_ptr, q.dtype, heads * self.head_dim, self.k.data_ptr, self.v.data_ptr, self.dtype, self.book.n_pages,
            self.book.page_size, heads, self.n_kv_heads, self.head_dim, table, width, cu, lens, len(seqs), total,
            out.data_ptr, scale, None, 0, self.lib.tl_hip_stream()))
        return out
