"""Pages of a paged key/value cache, handed out on the GPU.

``PagePool`` keeps, beside a cache's table and lengths, how many table rows hold each page (0: free), and writes all
three on the device from what the requests ask for: nothing is read back, and every call can be captured into a
CUDA graph.

    pool = PagePool.allocate(B, max_len, num_pages, kv_heads, head_dim, device="cuda")
    slots, served = pool.extend(n)                        # room for n tokens more a sequence; lengths count them
    q = kv_append(pool.cache, k, v, q, inv_freq=inv_freq)
    out = kv_attend(pool.cache, q)
    pool.truncate(lengths)                                # rejected drafts: their pages go back
    pool.reorder(parents)                                 # beams: rows take over their parents' pages

``extend`` takes the place of ``PagedKVCache.extend`` in a step (``attention_step`` calls the latter: with a pool, use
the lines above).  The calls of one pool belong on one stream, or in an order that the caller sees to.
"""

from __future__ import annotations

import ctypes as C

import torch
from torch import Tensor

from . import _lib
from ._lib import check, ptr, stream_ptr
from .kv import PagedKVCache, PagedKVCache8, _library, _require


class PagePool:
    """``caches``: a cache (``PagedKVCache`` or ``PagedKVCache8``) or several -- a model's layers -- of the same geometry
    that share one table and one lengths tensor.  ``refs``: int32 ``[pages]``, the table rows that hold each page, kept and
    not copied; without it the pool begins empty: all pages free, lengths 0, table entries -1.  At most 8192
    sequences and 2^22 pages."""

    def __init__(self, caches, refs: Tensor | None = None):
        caches = [caches] if isinstance(caches, PagedKVCache) else list(caches)
        _require(len(caches) >= 1 and all(isinstance(c, PagedKVCache) for c in caches), "a pool needs at least one cache")
        first = caches[0]
        for c in caches[1:]:
            _require(c.table.data_ptr() == first.table.data_ptr() and c.lengths.data_ptr() == first.lengths.data_ptr()
                     and c.table.shape == first.table.shape and c.table.stride() == first.table.stride(),
                     "a pool's caches must share one table and one lengths tensor")
            _require(c.page_size == first.page_size and c.k.shape[0] == first.k.shape[0],
                     "a pool's caches must have pages of one size, equally many")
            _require(c.device == first.device, "a pool's caches must be on one device")
        pages = first.k.shape[0]
        _require(first.batch <= 8192, "a pool serves at most 8192 sequences")
        _require(pages <= 1 << 22, "a pool holds at most 2^22 pages")
        _require(first.table.shape[1] >= 1, "the table has no columns")
        if refs is None:
            refs = torch.zeros(pages, dtype=torch.int32, device=first.device)
            first.table.fill_(-1)
            first.lengths.zero_()
        _require(refs.shape == (pages,) and refs.dtype == torch.int32 and refs.is_contiguous(), f"refs must be contiguous int32 [{pages}]")
        _require(refs.device == first.device, "refs must be on the caches' device")
        self.caches, self.cache, self._refs = caches, first, refs
        descs = [c._desc if c.eight else _lib.KvCache8(pages=c._desc) for c in caches]
        self._descs = (_lib.KvCache8 * len(descs))(*descs)
        self._ref = C.byref(self._descs[0])
        self._copies = torch.empty(first.batch, 4, dtype=torch.int32, device=first.device)  # an extend's, until its last copy

    refs = property(lambda self: self._refs)

    @classmethod
    def allocate(cls, batch: int, max_len: int, num_pages: int, num_kv_heads: int, head_dim: int, page_size: int = 64,
                 dtype: torch.dtype = torch.bfloat16, device=None, eight: bool = False, layers: int = 1) -> "PagePool":
        """An empty pool of ``num_pages`` pages a layer for ``batch`` sequences of up to ``max_len`` keys; ``eight``: caches in
        8 bits."""
        device = device or torch.device("cuda", torch.cuda.current_device())
        table = torch.full((batch, -(-int(max_len) // page_size)), -1, dtype=torch.int32, device=device)
        lengths = torch.zeros(batch, dtype=torch.int32, device=device)
        shape, caches = (num_pages, num_kv_heads, page_size, head_dim), []
        for _ in range(layers):
            if eight:
                k, v = (torch.zeros(shape, dtype=torch.uint8, device=device).view(torch.float8_e4m3fn) for _ in range(2))
                exps = [torch.zeros(shape[:2], dtype=torch.int8, device=device) for _ in range(2)]
                caches.append(PagedKVCache8(k, v, *exps, table, lengths, dtype=dtype))
            else:
                k, v = (torch.zeros(shape, dtype=dtype, device=device) for _ in range(2))
                caches.append(PagedKVCache(k, v, table, lengths))
        return cls(caches)

    def extend(self, n: int | None = None, *, cu: Tensor | None = None, max_new: int | None = None,
               tokens: int | None = None) -> tuple[Tensor, Tensor]:
        """Room for a step's new tokens: ``n`` a sequence, or ``cu`` and ``max_new`` as for ``kv_append``, of ``tokens`` rows
        in all (sequences * ``max_new`` where it is not given).  Lengths count the tokens from here on; new pages
        are the lowest free ones, in order of sequence, then of key.  A partly filled last page that other rows hold too
        is replaced by a copy of the sequence's own, in every cache.

        Returns ``slots``, int64 ``[B, n]`` (``[tokens]`` with ``cu``): page * page_size + slot of every new token, -1 for
        rows of no sequence; and ``served``, bool ``[B]``.  A sequence that does not fit its table row, or for which too few pages are free
        once those before it have theirs, is suspended: its length becomes -1 - length, its slots are -1,
        ``kv_append`` drops its tokens (recording device error 4) and ``kv_attend`` gives zeros for it.  Nothing of it is
        lost: the next ``extend`` or ``truncate`` takes it up again.  A sequence that needs no page is always served."""
        c = self.cache
        if cu is None:
            if n is None or max_new not in (None, n) or tokens not in (None, c.batch * n):
                raise ValueError("extend needs n, or cu and max_new")
            n = int(n)
            shape, tokens = (c.batch, n), c.batch * n
        else:
            if n is not None or max_new is None:
                raise ValueError("extend needs n, or cu and max_new")
            if cu.dtype is not torch.int32 or cu.shape != (c.batch + 1,) or not cu.is_contiguous() or cu.get_device() != c.index:
                raise ValueError(f"cu must be contiguous int32 [{c.batch + 1}] on the cache's device")
            n = int(max_new)
            tokens = c.batch * n if tokens is None else int(tokens)
            if tokens < 0:
                raise ValueError("tokens must not be negative")
            shape = (tokens,)
        if n < 0:
            raise ValueError("the number of new tokens must not be negative")
        lib = _library(c)
        slots = torch.empty(shape, dtype=torch.int64, device=c.device)
        served = torch.empty(c.batch, dtype=torch.bool, device=c.device)
        with _lib.on_device(c.device):
            check(lib.lng_kv_pages_extend(self._ref, len(self.caches), ptr(self._refs), ptr(cu), tokens, n, ptr(slots), ptr(served),
                                          ptr(self._copies), stream_ptr()), "extend")
        return slots, served

    def truncate(self, lengths) -> None:
        """Sequence b keeps its first min(``lengths[b]``, its length) keys (an int, or int32 ``[B]`` on the device); the
        pages behind them are given back, their table entries become -1.  Suspended sequences are taken up again."""
        c = self.cache
        most = 0
        if isinstance(lengths, Tensor):
            if lengths.dtype is not torch.int32 or lengths.shape != (c.batch,) or not lengths.is_contiguous() \
                    or lengths.get_device() != c.index:
                raise ValueError(f"lengths must be an int or contiguous int32 [{c.batch}] on the cache's device")
        else:
            most, lengths = int(lengths), None
            if most < 0:
                raise ValueError("lengths must not be negative")
        lib = _library(c)
        with _lib.on_device(c.device):
            check(lib.lng_kv_pages_truncate(self._ref, ptr(self._refs), ptr(lengths), most, stream_ptr()), "truncate")

    def reorder(self, parents: Tensor) -> None:
        """Beams: row g * beams + k takes over the pages and the length of row g * beams + ``parents[g, k]`` (int64
        ``[groups, beams]``, ``beam_select``'s; ``[1, B]`` for any rows of the batch).  Pages are shared, not copied
        (``extend`` copies one before it is written to); those that no row holds any more become free."""
        c = self.cache
        if parents.dim() != 2 or parents.dtype is not torch.int64 or parents.numel() != c.batch or not parents.is_contiguous() \
                or parents.get_device() != c.index:
            raise ValueError(f"parents must be contiguous int64 [groups, beams] of {c.batch} rows on the cache's device")
        lib = _library(c)
        with _lib.on_device(c.device):
            check(lib.lng_kv_pages_reorder(self._ref, ptr(self._refs), ptr(parents), parents.shape[0],
                                           parents.shape[1], stream_ptr()), "reorder")
