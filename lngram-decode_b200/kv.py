"""A paged cache of keys and values for the attention that runs beside the memory layer in a decode loop.

The reference's ``decode_step`` keeps dense keys and values in its ``DecodeState``
(``ffnmem/infer.py:65-112``); here they lie in pages that a server hands out as sequences grow:

* ``PagedKVCache`` -- the pages, the page table and the sequences' lengths (device tensors; the lengths count
  a step's new tokens from ``extend`` on).
* ``PagedKVCache8`` -- the same in 8 bits: e4m3 values under one exponent for each page and head.  Steps are still
  bf16 or fp16; ``kv_append``, ``kv_attend`` and ``attention_step`` take either cache.
* ``kv_append`` -- a step's keys and values into their slots, keys and queries rotated by position on the way.
* ``kv_attend`` -- causal attention of the step's tokens over the cache: grouped heads, an optional sliding
  window with the first ``sinks`` tokens visible beside it; one token a sequence or whole prompts.
* ``kv_prefix_attend`` -- the same for a batch whose sequences share one prefix, read once for all of them.
* ``attention_step`` -- extend, append and attend in one call, the counterpart of ``seams.memory_step``.

A step's tokens are ``[B, n, heads, head_dim]`` (n new tokens for every sequence) or, for sequences that add
unlike numbers of tokens, ``[tokens, heads, head_dim]`` with ``cu`` (int32 ``[B + 1]`` offsets on the device)
and ``max_new`` (a host bound of one sequence's new tokens).  The inner dimension is contiguous, the others
may be strided (slices of a fused projection).  Everything is asynchronous on the current stream and can be
captured into a CUDA graph: table and lengths are read when the kernels run.

    cache = PagedKVCache.allocate(B, max_len, kv_heads, head_dim, dtype=torch.bfloat16, device="cuda")
    cache.extend(n)                                       # the lengths now count the step's tokens
    q = kv_append(cache, k, v, q, inv_freq=inv_freq)      # rotated queries; keys and values cached
    out = kv_attend(cache, q, window=4096, sinks=4)       # [B, n, heads, head_dim]
"""

from __future__ import annotations

import ctypes as C

import torch
from torch import Tensor
from torch.autograd import forward_ad

from . import _lib
from ._lib import check, ptr, stream_ptr

_DTYPES = (torch.bfloat16, torch.float16)


def _require(cond: bool, msg: str) -> None:
    if not cond:
        raise ValueError(msg)


class PagedKVCache:
    """``k``, ``v``: pages ``[pages, kv_heads, page_size, head_dim]`` (bf16 or fp16; any view whose inner dimension
    is contiguous, so pages laid out ``[pages, page_size, kv_heads, head_dim]`` are passed transposed);
    ``table``: int32 ``[B, max_pages]``, the page of every ``page_size`` keys of a sequence; ``lengths``: int32
    ``[B]``.  The tensors are kept, not copied: write table and lengths in place."""

    def __init__(self, k: Tensor, v: Tensor, table: Tensor, lengths: Tensor):
        _require(k.dim() == 4 and v.shape == k.shape, "k and v must be [pages, kv_heads, page_size, head_dim], alike")
        _require(k.dtype in _DTYPES and v.dtype == k.dtype, "k and v must be bfloat16 or float16, alike")
        pages, heads, size, dim = k.shape
        _require(size >= 8 and size <= 4096 and size & (size - 1) == 0, "page_size must be a power of two in [8, 4096]")
        _require(8 <= dim <= 128 and dim % 8 == 0, "head_dim must be a multiple of 8 up to 128")
        _require(pages >= 1 and heads >= 1, "the cache needs at least one page and one head")
        for t in (k, v):
            _require(t.stride(3) == 1 and all(t.stride(i) > 0 and t.stride(i) % 8 == 0 for i in range(3)),
                     "the head dimension must be contiguous and the other strides positive multiples of 8")
            _require(t.data_ptr() % 16 == 0, "k and v must be 16-byte aligned")
        self._check_table(table, lengths, size)
        _require(k.device == v.device == table.device == lengths.device, "the cache's tensors must be on one device")
        self._k, self._v, self._table, self._lengths = k, v, table, lengths
        self._desc = self._pages_desc(_lib.dtype_code(k.dtype))
        self._set_up(k.dtype)

    eight = False  # whether the pages hold 8 bits (PagedKVCache8)

    @staticmethod
    def _check_table(table: Tensor, lengths: Tensor, size: int) -> None:
        _require(table.dim() == 2 and table.dtype == torch.int32 and (table.shape[1] <= 1 or table.stride(1) == 1),
                 "table must be int32 [B, max_pages] with contiguous rows")
        _require(table.shape[0] <= 1 or table.stride(0) >= table.shape[1], "table: the sequences' rows must not overlap")
        _require(lengths.dim() == 1 and lengths.dtype == torch.int32 and lengths.is_contiguous(),
                 "lengths must be contiguous int32 [B]")
        _require(lengths.shape[0] == table.shape[0], "table and lengths must have one row a sequence")
        _require(table.shape[1] * size < 1 << 30, "max_pages * page_size must be below 2^30")

    def _pages_desc(self, dtype: int) -> _lib.KvCache:
        k, v, table, lengths = self._k, self._v, self._table, self._lengths
        pages, heads, size, dim = k.shape
        return _lib.KvCache(k=k.data_ptr(), v=v.data_ptr(), dtype=dtype, page_size=size, num_pages=pages, num_kv_heads=heads,
                            head_dim=dim, k_page_stride=k.stride(0), k_head_stride=k.stride(1), k_slot_stride=k.stride(2),
                            v_page_stride=v.stride(0), v_head_stride=v.stride(1), v_slot_stride=v.stride(2),
                            table=table.data_ptr(), table_stride=max(table.stride(0), table.shape[1]), max_pages=table.shape[1],
                            lengths=lengths.data_ptr(), batch=table.shape[0])

    def _set_up(self, dtype: torch.dtype) -> None:
        k, table = self._k, self._table
        self._ref = C.byref(self._desc)
        self.device, self.dtype, self.index = k.device, dtype, k.get_device()
        self._sizes: dict = {}
        self.batch, self.page_size, self.num_kv_heads, self.head_dim = table.shape[0], k.shape[2], k.shape[1], k.shape[3]
        self.capacity = table.shape[1] * self.page_size

    k = property(lambda self: self._k)
    v = property(lambda self: self._v)
    table = property(lambda self: self._table)
    lengths = property(lambda self: self._lengths)

    @classmethod
    def allocate(cls, batch: int, max_len: int, num_kv_heads: int, head_dim: int, page_size: int = 64,
                 dtype: torch.dtype = torch.bfloat16, device=None) -> "PagedKVCache":
        """An empty cache in which every sequence owns ceil(max_len / page_size) pages."""
        device = device or torch.device("cuda", torch.cuda.current_device())
        per = -(-int(max_len) // page_size)
        shape = (max(1, batch * per), num_kv_heads, page_size, head_dim)
        return cls(torch.zeros(shape, dtype=dtype, device=device), torch.zeros(shape, dtype=dtype, device=device),
                   torch.arange(batch * per, dtype=torch.int32, device=device).view(batch, per),
                   torch.zeros(batch, dtype=torch.int32, device=device))

    def extend(self, n) -> None:
        """Count n (an int, or int32 [B] on the device) new tokens a sequence.  The lengths are on the device and not
        looked at here: past ``capacity`` ``kv_append`` drops the tokens that do not fit, attention gives zeros for the
        sequence, and device error 4 is recorded (``lng_device_error``)."""
        self._lengths.add_(n)

    def truncate(self, lengths) -> None:
        """Forget the keys behind ``lengths`` (an int, or int32 [B]), e.g. rejected drafts."""
        if isinstance(lengths, Tensor):
            torch.minimum(self._lengths, lengths.to(self._lengths), out=self._lengths)
        else:
            self._lengths.clamp_(max=int(lengths))


class PagedKVCache8(PagedKVCache):
    """A cache in 8 bits.  ``k``, ``v``: float8_e4m3fn pages ``[pages, kv_heads, page_size, head_dim]``; ``k_exp``,
    ``v_exp``: int8 ``[pages, kv_heads]`` exponents; a slot stands for its value times 2^exponent.  ``dtype``: bf16 or
    fp16, of the rows that are appended and attended with.

    ``kv_append`` gives a page and head the least exponent under which its new values fit e4m3, at least -40 and at most
    40 (beyond 448 * 2^40 values saturate; NaN and infinities become NaN); a page that holds earlier keys keeps its
    exponent where that is larger, else the earlier keys are rounded again to the new one.  A power of two as the scale
    costs no precision: e4m3 has an exponent of its own.  Attention rounds its weights to fp16, the values' exponents in
    them: a key's weight keeps its 11 bits while its score (in base 2) + exponent lies up to 21 below the row's largest, and
    from 32 below on its values may count as zero.  The likeliest keys lose nothing while the pages' largest values are
    within 2^21 of one another.  Pages that several sequences name are for reading (``PagePool`` copies a shared page
    before it is written to)."""

    eight = True

    def __init__(self, k: Tensor, v: Tensor, k_exp: Tensor, v_exp: Tensor, table: Tensor, lengths: Tensor,
                 dtype: torch.dtype = torch.bfloat16):
        _require(dtype in _DTYPES, "dtype must be bfloat16 or float16")
        _require(k.dim() == 4 and v.shape == k.shape, "k and v must be [pages, kv_heads, page_size, head_dim], alike")
        _require(k.dtype == torch.float8_e4m3fn and v.dtype == k.dtype, "k and v must be float8_e4m3fn")
        pages, heads, size, dim = k.shape
        _require(size >= 8 and size <= 256 and size & (size - 1) == 0, "page_size must be a power of two in [8, 256]")
        _require(16 <= dim <= 128 and dim % 16 == 0, "head_dim must be a multiple of 16 up to 128")
        _require(pages >= 1 and heads >= 1, "the cache needs at least one page and one head")
        for t in (k, v):
            _require(t.stride(3) == 1 and all(t.stride(i) > 0 and t.stride(i) % 16 == 0 for i in range(3)),
                     "the head dimension must be contiguous and the other strides positive multiples of 16")
            _require(t.data_ptr() % 16 == 0, "k and v must be 16-byte aligned")
        for t in (k_exp, v_exp):
            _require(t.shape == (pages, heads) and t.dtype == torch.int8 and (heads == 1 or t.stride(1) == 1)
                     and (pages == 1 or t.stride(0) >= heads), "k_exp and v_exp must be int8 [pages, kv_heads] with contiguous rows")
        self._check_table(table, lengths, size)
        _require(k.device == v.device == k_exp.device == v_exp.device == table.device == lengths.device,
                 "the cache's tensors must be on one device")
        self._k, self._v, self._k_exp, self._v_exp = k, v, k_exp, v_exp
        self._table, self._lengths = table, lengths
        self._desc = _lib.KvCache8(pages=self._pages_desc(_lib.dtype_code(dtype)), k_exp=k_exp.data_ptr(), v_exp=v_exp.data_ptr(),
                                   k_exp_stride=max(k_exp.stride(0), heads), v_exp_stride=max(v_exp.stride(0), heads))
        self._set_up(dtype)

    k_exp = property(lambda self: self._k_exp)
    v_exp = property(lambda self: self._v_exp)

    @classmethod
    def allocate(cls, batch: int, max_len: int, num_kv_heads: int, head_dim: int, page_size: int = 64,
                 dtype: torch.dtype = torch.bfloat16, device=None) -> "PagedKVCache8":
        """An empty cache in which every sequence owns ceil(max_len / page_size) pages."""
        device = device or torch.device("cuda", torch.cuda.current_device())
        per = -(-int(max_len) // page_size)
        shape = (max(1, batch * per), num_kv_heads, page_size, head_dim)
        k, v = (torch.zeros(shape, dtype=torch.uint8, device=device).view(torch.float8_e4m3fn) for _ in range(2))
        k_exp, v_exp = (torch.zeros(shape[:2], dtype=torch.int8, device=device) for _ in range(2))
        return cls(k, v, k_exp, v_exp, torch.arange(batch * per, dtype=torch.int32, device=device).view(batch, per),
                   torch.zeros(batch, dtype=torch.int32, device=device), dtype=dtype)

    def values(self) -> tuple[Tensor, Tensor]:
        """What the slots of all pages stand for: keys and values, bf16 ``[pages, kv_heads, page_size, head_dim]``
        (every such value is exact in bf16)."""
        lib = _library(self)
        k, v = (torch.empty(self._k.shape, dtype=torch.bfloat16, device=self.device) for _ in range(2))
        with _lib.on_device(self.device):
            check(lib.lng_kv8_values(self._ref, ptr(k), ptr(v), stream_ptr()), "values")
        return k, v


def _strides(t: Tensor, what: str, cache: PagedKVCache) -> tuple[int, int]:
    """(token stride, head stride) of a step's rows whose shape has been checked."""
    st, n = t.stride(), t.shape[-2]
    head = st[-2] if n > 1 else cache.head_dim
    token = st[-3] if t.shape[-3] > 1 else (st[0] if t.dim() == 4 and t.shape[0] > 1 else n * cache.head_dim)
    if t.dim() == 4 and t.shape[0] > 1 and t.shape[1] > 1:
        _require(st[0] == st[1] * t.shape[1], f"{what}: the tokens of all sequences must lie at one stride")
    _require(st[-1] == 1 and head > 0 and head % 8 == 0 and token > 0 and token % 8 == 0,
             f"{what} must be 16-byte aligned with a contiguous head dimension and strides of positive multiples of 8")
    return token, head


def _rows(t: Tensor, what: str, cache: PagedKVCache, shape=None, heads: int | None = None) -> _lib.KvRows:
    """The descriptor of a step's rows; ``shape``: the leading shape they must have."""
    # (messages are only made when they are needed: a decode step's host time is spent in lines like these)
    ts = t.shape
    if t.dtype is not cache.dtype:
        raise ValueError(f"{what} must have the cache's dtype {cache.dtype}")
    if len(ts) not in (3, 4) or ts[-1] != cache.head_dim:
        raise ValueError(f"{what} must be [B, n, heads, {cache.head_dim}] or [tokens, heads, {cache.head_dim}]")
    if shape is not None and ts[:-2] != shape:
        raise ValueError(f"{what} must have the step's leading shape {tuple(shape)}")
    n = ts[-2]
    if heads is not None and n != heads:
        raise ValueError(f"{what} must have {heads} heads")
    if t.is_contiguous():
        token, head = max(n, 1) * cache.head_dim, cache.head_dim
    else:
        token, head = _strides(t, what, cache)
    p = t.data_ptr()
    if p % 16:
        raise ValueError(f"{what} must be 16-byte aligned with a contiguous head dimension and strides of positive multiples of 8")
    if t.get_device() != cache.index:
        raise ValueError(f"{what} must be on the cache's device")
    return _lib.KvRows(p, token, head, n)


def _step(cache: PagedKVCache, t: Tensor, cu: Tensor | None, max_new: int | None):
    """(tokens, max_new) of a step whose rows are shaped like t."""
    ts = t.shape
    if cu is None:
        if len(ts) != 4 or ts[0] != cache.batch:
            raise ValueError(f"without cu the step's rows must be [B = {cache.batch}, n, heads, {cache.head_dim}]")
        if max_new is not None and max_new != ts[1]:
            raise ValueError("max_new must be the step's n when there is no cu")
        return ts[0] * ts[1], ts[1]
    if len(ts) != 3:
        raise ValueError("with cu the step's rows must be [tokens, heads, head_dim]")
    if cu.dtype is not torch.int32 or cu.shape != (cache.batch + 1,) or not cu.is_contiguous() or cu.get_device() != cache.index:
        raise ValueError(f"cu must be contiguous int32 [{cache.batch + 1}] on the cache's device")
    if max_new is None or max_new < 0:
        raise ValueError("a step with cu needs max_new")
    return ts[0], int(max_new)


def _no_grad(cache: PagedKVCache, *tensors: Tensor | None) -> None:
    if torch.is_grad_enabled() and (cache._k.requires_grad or cache._v.requires_grad
                                    or any(t is not None and t.requires_grad for t in tensors)):
        raise RuntimeError("the paged cache's operators have no backward: call them under torch.no_grad()")
    if getattr(forward_ad, "_current_level", 0) >= 0 and any(
            t is not None and forward_ad.unpack_dual(t).tangent is not None for t in (cache._k, cache._v) + tensors):
        raise RuntimeError("the paged cache's operators carry no tangent: give them the primal values")


def _library(cache: PagedKVCache):
    if cache.index < 0:
        raise RuntimeError("the cache must be on a CUDA device: lngram_b200 has no CPU path")
    return _lib._LIB if cache.index in _lib._DEVICE_OK else _lib.library()


def kv_append(cache: PagedKVCache, k: Tensor, v: Tensor, q: Tensor | None = None, *, cu: Tensor | None = None,
              max_new: int | None = None, positions: Tensor | None = None, inv_freq: Tensor | None = None,
              interleaved: bool = False, q_out: Tensor | None = None) -> Tensor | None:
    """Write a step's keys and values to the cache: token i of the n new ones of a sequence becomes key
    ``lengths - n + i`` (``extend`` first).  With ``inv_freq`` (fp32 ``[rotary_dim / 2]``) the first rotary_dim
    values of keys and queries are rotated by the token's position -- ``positions`` (int64, the step's leading
    shape; needed behind a shared prefix) or its place in the sequence -- in pairs (j, j + rotary_dim / 2), or (2j, 2j + 1) if ``interleaved``.
    Returns the rotated queries (``q_out`` if given; it may be ``q``) or None without ``q``.  Pages that several
    sequences name are for reading: no two tokens of a step may go to one slot.  No gradients."""
    _no_grad(cache, k, v, q, inv_freq, q_out)
    tokens, max_new = _step(cache, k, cu, max_new)
    lead = k.shape[:-2]
    kr = _rows(k, "k", cache, lead, cache.num_kv_heads)
    vr = _rows(v, "v", cache, lead, cache.num_kv_heads)
    qr = qo = None
    if q is not None:
        qr = C.byref(_rows(q, "q", cache, lead))
        if q_out is None:
            q_out = torch.empty_like(q, memory_format=torch.contiguous_format)
        qo = C.byref(_rows(q_out, "q_out", cache, lead, q.shape[-2]))
    elif q_out is not None:
        raise ValueError("q_out without q")
    rotary = 0
    if inv_freq is not None:
        if inv_freq.dtype is not torch.float32 or inv_freq.dim() != 1 or not inv_freq.is_contiguous() \
                or inv_freq.get_device() != cache.index:
            raise ValueError("inv_freq must be contiguous fp32 [rotary_dim / 2] on the cache's device")
        rotary = 2 * inv_freq.shape[0]
        if rotary > cache.head_dim:
            raise ValueError("inv_freq has more pairs than the head")
    if positions is not None and (positions.dtype is not torch.int64 or positions.shape != lead or not positions.is_contiguous()
                                  or positions.get_device() != cache.index):
        raise ValueError("positions must be contiguous int64 of the step's leading shape")
    lib = _library(cache)
    with _lib.on_device(cache.device):
        append = lib.lng_kv8_append if cache.eight else lib.lng_kv_append
        check(append(cache._ref, ptr(cu), tokens, max_new, C.byref(kr), C.byref(vr), qr, qo, ptr(positions),
                     ptr(inv_freq) if rotary else None, rotary, 1 if interleaved else 0, stream_ptr()), "kv_append")
    return q_out


def _attend_args(cache, q, cu, max_new, max_len, scale, out):
    _no_grad(cache, q, out)
    tokens, max_new = _step(cache, q, cu, max_new)
    qr = _rows(q, "q", cache)
    heads = qr.heads
    if heads % cache.num_kv_heads or not 1 <= heads // cache.num_kv_heads <= 128:
        raise ValueError("query heads must be a multiple of the key heads, at most 128 a key head")
    if out is None:
        out = torch.empty_like(q, memory_format=torch.contiguous_format)
    orow = _rows(out, "out", cache, q.shape[:-2], heads)
    if tokens and orow.ptr == qr.ptr:
        raise ValueError("out must not overlap q")
    max_len = cache.capacity if max_len is None else int(max_len)
    if max_len < 0:
        raise ValueError("max_len must not be negative")
    scale = cache.head_dim ** -0.5 if scale is None else float(scale)
    if not 0.0 < scale < 2.35e38:  # (scores are kept in base 2: scale * log2(e) must be finite in fp32)
        raise ValueError("scale must be positive and below 2.35e38")
    return tokens, max_new, max_len, qr, heads, scale, out, orow


def _workspace(cache: PagedKVCache, key: tuple, size) -> Tensor | None:
    """A workspace of its own for this call, of the size that ``size()`` gives (kept by the call's arguments)."""
    need = cache._sizes.get(key)
    if need is None:
        if len(cache._sizes) > 256:
            cache._sizes.clear()
        need = cache._sizes[key] = size()
    return torch.empty(need, dtype=torch.uint8, device=cache.device) if need else None


def kv_attend(cache: PagedKVCache, q: Tensor, *, cu: Tensor | None = None, max_new: int | None = None,
              max_len: int | None = None, window: int = 0, sinks: int = 0, scale: float | None = None,
              out: Tensor | None = None) -> Tensor:
    """Causal attention of a step's tokens over the cache, whose lengths count them (``kv_append`` first): the
    token at position p sees keys j <= p; with ``window`` > 0 only its last ``window`` keys and the first
    ``sinks`` of the sequence.  softmax(scale q . k) v with ``scale`` = head_dim^-1/2 by default; a token
    that sees no key gets zeros, one with a score of NaN or +inf NaN.  Values that any token of the step sees must be
    finite.  ``max_len`` (a host bound of the lengths) only guides how the work is split.
    Rows of ``q`` that belong to no sequence are skipped: their rows of ``out`` stay as they are.  No gradients."""
    tokens, max_new, max_len, qr, heads, scale, out, orow = _attend_args(cache, q, cu, max_new, max_len, scale, out)
    window, sinks = int(window), int(sinks)
    if window < 0 or sinks < 0:
        raise ValueError("window and sinks must not be negative")
    window, sinks = min(window, 1 << 30), min(sinks, 1 << 30)
    lib = _library(cache)
    with _lib.on_device(cache.device):
        attend, need = (lib.lng_kv8_attend, lib.lng_kv8_attend_workspace_bytes) if cache.eight else \
            (lib.lng_kv_attend, lib.lng_kv_attend_workspace_bytes)
        ws = _workspace(cache, (tokens, max_new, max_len, heads, window, sinks), lambda: need(
            cache._ref, tokens, max_new, max_len, heads, window, sinks))
        check(attend(cache._ref, ptr(cu), tokens, max_new, max_len, C.byref(qr), scale, window, sinks,
                     C.byref(orow), ptr(ws), 0 if ws is None else ws.numel(), stream_ptr()), "kv_attend")
    return out


def kv_prefix_attend(cache: PagedKVCache, q: Tensor, prefix_table: Tensor, prefix_len: int, *, cu: Tensor | None = None,
                     max_new: int | None = None, max_len: int | None = None, scale: float | None = None,
                     out: Tensor | None = None) -> Tensor:
    """``kv_attend`` (without a window) for a batch whose sequences all begin with the ``prefix_len`` keys in the
    pages ``prefix_table`` (int32 ``[>= ceil(prefix_len / page_size)]``) of the same cache; ``table`` and
    ``lengths`` hold what each sequence adds to it.  The prefix is read once for the whole batch.  ``kv_append``'s own
    positions count a sequence's own keys only: behind a prefix give it ``positions`` that count the prefix too
    (prefix_len + the key's place).  The prefix itself is appended once, through a cache of one sequence over the same
    pages whose table is ``prefix_table``.  Not for a cache in 8 bits (a ``PagePool`` shares its pages).  No gradients."""
    if cache.eight:
        raise ValueError("kv_prefix_attend takes a cache in 16 bits")
    tokens, max_new, max_len, qr, heads, scale, out, orow = _attend_args(cache, q, cu, max_new, max_len, scale, out)
    prefix_len = int(prefix_len)
    if not 0 <= prefix_len < 1 << 30:
        raise ValueError("prefix_len must be in [0, 2^30)")
    if prefix_table.dtype is not torch.int32 or prefix_table.dim() != 1 or not prefix_table.is_contiguous() \
            or prefix_table.get_device() != cache.index:
        raise ValueError("prefix_table must be contiguous int32 on the cache's device")
    if prefix_table.shape[0] * cache.page_size < prefix_len:
        raise ValueError("prefix_table has too few pages for prefix_len")
    lib = _library(cache)
    with _lib.on_device(cache.device):
        ws = _workspace(cache, (prefix_len, tokens, max_new, max_len, heads), lambda: lib.lng_kv_prefix_workspace_bytes(
            cache._ref, prefix_len, tokens, max_new, max_len, heads))
        check(lib.lng_kv_prefix_attend(cache._ref, ptr(prefix_table) if prefix_len else None, prefix_len, ptr(cu), tokens,
                                       max_new, max_len, C.byref(qr), scale, C.byref(orow), ptr(ws),
                                       0 if ws is None else ws.numel(), stream_ptr()), "kv_prefix_attend")
    return out


def attention_step(cache: PagedKVCache, q: Tensor, k: Tensor, v: Tensor, *, cu: Tensor | None = None,
                   max_new: int | None = None, positions: Tensor | None = None, inv_freq: Tensor | None = None,
                   interleaved: bool = False, max_len: int | None = None, window: int = 0, sinks: int = 0,
                   scale: float | None = None, out: Tensor | None = None) -> Tensor:
    """The attention part of a decode step, beside ``seams.memory_step``: the lengths count the step's tokens,
    keys and values are appended, and the rotated queries attend.  A refused step leaves the lengths as they were."""
    _step(cache, q, cu, max_new)
    n = q.shape[1] if cu is None else cu[1:] - cu[:-1]
    cache.extend(n)
    try:
        q = kv_append(cache, k, v, q, cu=cu, max_new=max_new, positions=positions, inv_freq=inv_freq, interleaved=interleaved)
        return kv_attend(cache, q, cu=cu, max_new=max_new, max_len=max_len, window=window, sinks=sinks, scale=scale, out=out)
    except BaseException:
        cache.extend(-n)
        raise
