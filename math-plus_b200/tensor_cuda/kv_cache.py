"""The paged key/value cache of a served model: ``PagedKVCache`` holds the pages of one layer,
``BlockTable`` hands pages to sequences and names them to the kernels.

The reference has no counterpart: its ``MultiheadAttention`` recomputes K and V of the whole sequence
(packages/tensor-autograd/src/transformer.ts:173-242). Here a sequence's rows live in pages of
``page_size`` tokens, laid out [page, head, row, dim] so that one head's page is one contiguous block;
``CudaBackend.kv_append`` writes tokens, ``kv_read`` gathers them and ``sdpa_paged`` attends over them.
``dtype="e4m3"`` holds each row in 8 bits with one power-of-two scale byte: a little over half of bf16's
bytes, each value within 2^-4 of itself.
"""
from __future__ import annotations

import ctypes as C

import numpy as np

from . import _ffi as F

#: storage of a cache: the C ABI's dtype code and bytes per value
CACHE_DTYPES = {"f32": (F.F32, 4), "f16": (F.F16, 2), "bf16": (F.BF16, 2), "e4m3": (F.E4M3, 1)}


class PagedKVCache:
    """K and V pages of one layer. ``pools`` takes memory owned elsewhere instead of allocating it: the
    device addresses of (K pages, V pages, K scales, V scales), the scales None unless 8-bit; the caller
    keeps that memory alive."""

    def __init__(self, backend, n_pages: int, page_size: int, n_kv_head: int, head_dim: int, dtype: str = "bf16",
                 head_dim_v: int | None = None, pools=None):
        if dtype not in CACHE_DTYPES:
            raise TypeError(f"tensor-cuda: PagedKVCache: dtype {dtype} (one of {', '.join(CACHE_DTYPES)})")
        head_dim_v = head_dim if head_dim_v is None else head_dim_v
        if n_pages < 0 or min(page_size, n_kv_head, head_dim, head_dim_v) <= 0:
            raise ValueError(f"tensor-cuda: PagedKVCache: {n_pages} pages of {page_size} rows, {n_kv_head} heads of "
                             f"{head_dim} and {head_dim_v}")
        if head_dim > 256 or head_dim_v > 256:
            raise NotImplementedError("tensor-cuda: PagedKVCache: head dims above 256")
        self.backend = backend
        self.n_pages, self.page_size = int(n_pages), int(page_size)
        self.n_kv_head, self.head_dim, self.head_dim_v, self.dtype = int(n_kv_head), int(head_dim), int(head_dim_v), dtype
        code, eb = CACHE_DTYPES[dtype]
        self.desc = F.KvDesc(self.n_pages, self.page_size, self.n_kv_head, self.head_dim, self.head_dim_v, code, 0)
        rows = self.n_pages * self.n_kv_head * self.page_size
        self.nbytes = rows * (self.head_dim + self.head_dim_v) * eb + (2 * rows if dtype == "e4m3" else 0)
        self._bufs = []
        if pools is None:
            sizes = [rows * self.head_dim * eb, rows * self.head_dim_v * eb] + ([rows, rows] if dtype == "e4m3" else [])
            self._bufs = [backend.device.alloc(n) for n in sizes]
            pools = [b.ptr for b in self._bufs] + [None] * (4 - len(self._bufs))
        elif len(pools) != 4 or (dtype == "e4m3" and self.n_pages and None in pools):
            raise ValueError("tensor-cuda: PagedKVCache: pools are four addresses (K, V, K scales, V scales)")
        #: (desc, K pages, V pages, K scales, V scales) as every call of the C ABI takes them
        self.args = (C.byref(self.desc), *(C.c_void_p(p) for p in pools))
        #: element strides (token, head) of dense rows [T, Hk, D]
        self.k_strides = F.I64x2(self.n_kv_head * self.head_dim, self.head_dim)
        self.v_strides = F.I64x2(self.n_kv_head * self.head_dim_v, self.head_dim_v)
        self.disposed = False

    def dispose(self) -> None:
        """Returns the pages to the device allocator (idempotent)."""
        self.disposed = True
        for b in self._bufs:
            b.release()
        self._bufs = []


class BlockTable:
    """The pages of ``n_seq`` sequences, shared by the caches of a model's layers: a free list on the host
    and the i32 [n_seq, max_pages] table on the device. Entries behind a sequence's pages are -1."""

    def __init__(self, backend, n_seq: int, n_pages: int, page_size: int, max_pages: int | None = None):
        if n_seq <= 0 or n_pages <= 0 or page_size <= 0:
            raise ValueError(f"tensor-cuda: BlockTable: {n_seq} sequences, {n_pages} pages of {page_size}")
        self.backend, self.page_size = backend, int(page_size)
        self.n_pages = int(n_pages)
        self.host = np.full((n_seq, n_pages if max_pages is None else max_pages), -1, np.int32)
        self._held = [0] * n_seq
        self._free = list(range(self.n_pages - 1, -1, -1))
        self._device = None

    @property
    def free_pages(self) -> int:
        return len(self._free)

    def reserve(self, lengths) -> None:
        """Gives every sequence the pages that ``lengths`` tokens need (pages it has stay). Nothing is
        taken when the pool or a row of the table is too small: raises MemoryError or ValueError."""
        if len(lengths) != len(self._held):
            raise ValueError(f"tensor-cuda: BlockTable: {len(lengths)} lengths for {len(self._held)} sequences")
        need = [-(-int(n) // self.page_size) for n in lengths]
        for b, n in enumerate(need):
            if n > self.host.shape[1]:
                raise ValueError(f"tensor-cuda: BlockTable: sequence {b} needs {n} pages, a row holds {self.host.shape[1]}")
        more = sum(max(0, n - h) for n, h in zip(need, self._held))
        if more > len(self._free):
            raise MemoryError(f"tensor-cuda: BlockTable: {more} pages needed, {len(self._free)} of {self.n_pages} free")
        for b, n in enumerate(need):
            while self._held[b] < n:
                self.host[b, self._held[b]] = self._free.pop()
                self._held[b] += 1
                self._drop()

    def release(self, b: int) -> None:
        """Returns sequence b's pages to the pool."""
        n = self._held[b]
        if n:
            self._free.extend(int(p) for p in self.host[b, :n][::-1])
            self.host[b, :n] = -1
            self._held[b] = 0
            self._drop()

    def _drop(self) -> None:
        if self._device is not None:
            self.backend.dispose(self._device)
            self._device = None

    @property
    def device(self):
        """The table on the device (uploaded after a change, or where a scope has released it)."""
        if self._device is None or self._device.disposed:
            from .backend import host
            self._device = self.backend.from_host_sync(host("i32", self.host.shape, self.host))
        return self._device

    def dispose(self) -> None:
        self._drop()
