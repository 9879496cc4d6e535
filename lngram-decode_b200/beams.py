"""Beam search beside the memory layer: the choice of continuations, and the states that follow it.

* ``beam_select`` -- the best continuations over a request's beams and the vocabulary.
* ``beam_reorder`` -- rows of dense states take over their parents', in place (``MemoryCache.reorder`` and
  ``PagePool.reorder`` are the caches' own; the reference's incremental state has ``index_select`` for it,
  ``ffnmem/memory/lngram_v2.py:187-204``).

    scores, tokens, parents = beam_select(logits, scores)     # logits [groups, beams, vocab]
    memory_cache.reorder(parents)
    pool.reorder(parents)
"""

from __future__ import annotations

import torch
from torch import Tensor
from torch.autograd import forward_ad

from . import _lib
from ._lib import check, ptr, stream_ptr

_DTYPES = (torch.float32, torch.bfloat16, torch.float16)
_SIZES: dict = {}  # workspace bytes by a call's shape and device


def _no_grad(*tensors: Tensor | None) -> None:
    if torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in tensors):
        raise RuntimeError("beam search's operators have no backward: call them under torch.no_grad()")
    if getattr(forward_ad, "_current_level", 0) >= 0 and any(
            t is not None and t.is_floating_point() and forward_ad.unpack_dual(t).tangent is not None for t in tensors):
        raise RuntimeError("beam search's operators carry no tangent: give them the primal values")


def _library(index: int):
    if index < 0:
        raise RuntimeError("beam search's tensors must be on a CUDA device: lngram_b200 has no CPU path")
    return _lib._LIB if index in _lib._DEVICE_OK else _lib.library()


def beam_select(logits: Tensor, scores: Tensor, *, width: int | None = None, done: Tensor | None = None,
                eos: int | None = None) -> tuple[Tensor, Tensor, Tensor]:
    """One step of beam search.  ``logits`` ``[groups, beams, vocab]`` (fp32, bf16 or fp16; the vocabulary contiguous,
    rows at one stride), ``scores`` fp32 ``[groups, beams]``: of a group's candidates scores[k] + log_softmax(logits[k])[v]
    the ``width`` largest (default: as many as beams), in falling order, ties to the lowest beam, then token.  ``done``
    (bool ``[groups, beams]``): a beam that has ended offers only ``eos``, at its own score, and -inf for the rest.  A row
    that holds a NaN, +inf or nothing but -inf offers -inf throughout, and so does a beam (ended or not) whose score is -inf
    or NaN; scores must be below +inf.

    Returns ``scores`` fp32, ``tokens`` int64 and ``parents`` int64, ``[groups, width]``.  Sums are fp32, their joins and
    the ranking 64 bits; finite candidates of one beam rank as their logits do, whatever the score rounds away.  At most 32
    beams, and a width of 32.  No gradients."""
    _no_grad(logits, scores)
    if logits.dim() != 3 or logits.dtype not in _DTYPES:
        raise ValueError("logits must be [groups, beams, vocab] in float32, bfloat16 or float16")
    groups, beams, vocab = logits.shape
    if not 1 <= beams <= 32:
        raise ValueError("there must be 1 to 32 beams")
    if not 1 <= vocab < 1 << 30:
        raise ValueError("vocab must be in [1, 2^30)")
    if groups >= 1 << 24:
        raise ValueError("there must be fewer than 2^24 groups")
    width = beams if width is None else int(width)
    if not 1 <= width <= 32 or width > beams * vocab:
        raise ValueError("width must be in [1, 32] and at most beams * vocab")
    if scores.dtype is not torch.float32 or scores.shape != (groups, beams) or not scores.is_contiguous():
        raise ValueError(f"scores must be contiguous float32 [{groups}, {beams}]")
    stride = logits.stride(1) if beams > 1 else logits.stride(0) if groups > 1 else vocab
    if (vocab > 1 and logits.stride(2) != 1) or (groups * beams > 1 and stride < vocab) or \
            (groups > 1 and logits.stride(0) != beams * stride):
        raise ValueError("logits: the vocabulary must be contiguous and all rows at one stride")
    if done is not None:
        if done.dtype is not torch.bool or done.shape != (groups, beams) or not done.is_contiguous():
            raise ValueError(f"done must be contiguous bool [{groups}, {beams}]")
        if eos is None or not 0 <= int(eos) < vocab:
            raise ValueError("done needs eos, a token of the vocabulary")
    index = logits.get_device()
    if scores.get_device() != index or (done is not None and done.get_device() != index):
        raise ValueError("logits, scores and done must be on one device")
    lib = _library(index)
    device = logits.device
    out = torch.empty(groups, width, dtype=torch.float32, device=device)
    tokens, parents = (torch.empty(groups, width, dtype=torch.int64, device=device) for _ in range(2))
    with _lib.on_device(device):
        need = _SIZES.get((index, groups, beams, vocab, width))
        if need is None:
            if len(_SIZES) > 256:
                _SIZES.clear()
            need = _SIZES[index, groups, beams, vocab, width] = lib.lng_beam_workspace_bytes(groups, beams, vocab, width)
        ws = torch.empty(need, dtype=torch.uint8, device=device)
        check(lib.lng_beam_select(ptr(logits), _lib.dtype_code(logits.dtype), stride, groups, beams, vocab, ptr(scores), ptr(done),
                                  0 if done is None else int(eos), width, ptr(out), ptr(tokens), ptr(parents), ptr(ws), need,
                                  stream_ptr()), "beam_select")
    return out, tokens, parents


def _meet(a: _lib.BeamState, b: _lib.BeamState, rows: int) -> bool:
    """Whether what moves of two states has bytes in common."""
    if a.bytes == 0 or b.bytes == 0:
        return False
    if b.ptr < a.ptr:
        a, b = b, a
    if a.ptr + (rows - 1) * a.stride + a.bytes <= b.ptr:
        return False
    if a.stride == b.stride:
        inside = (b.ptr - a.ptr) % a.stride  # where b's rows begin in a's
        return inside < a.bytes or a.stride - inside < b.bytes
    # of each of a's rows: the first of b's that ends behind its beginning
    for at in range(a.ptr, a.ptr + rows * a.stride, a.stride):
        j = max(0, (at - b.ptr - b.bytes) // b.stride + 1)
        if j < rows and b.ptr + j * b.stride < at + a.bytes:
            return True
    return False


def beam_reorder(parents: Tensor, *states: Tensor, length: int | None = None) -> None:
    """Rows of ``states``, in place: row g * beams + k becomes what row g * beams + ``parents[g, k]`` was (int64 ``[groups,
    beams]``, on the device).  A state is ``[groups * beams, ...]`` of any type, each row contiguous, rows at any stride
    that keeps them apart; with ``length`` only the first ``length`` entries of its next dimension move.  States that
    overlap in what moves are refused.  A parent out of range records device error 4 and leaves its row as it is.  At most 32 beams.  No
    gradients."""
    _no_grad(*states)
    if parents.dim() != 2 or parents.dtype is not torch.int64 or not parents.is_contiguous():
        raise ValueError("parents must be contiguous int64 [groups, beams]")
    groups, beams = parents.shape
    if not 1 <= beams <= 32:
        raise ValueError("there must be 1 to 32 beams")
    if groups > 65535:
        raise ValueError("there must be at most 65535 groups")
    index, descs = parents.get_device(), []
    for x in states:
        if x.dim() < 1 or x.shape[0] != groups * beams:
            raise ValueError(f"a state must have {groups * beams} rows")
        if x.get_device() != index:
            raise ValueError("parents and states must be on one device")
        inner = x.shape[1:]
        if length is not None:
            if x.dim() < 2 or not 0 <= int(length) <= inner[0]:
                raise ValueError("length must be within every state's second dimension")
            inner = (int(length),) + tuple(inner[1:])
        expected = 1
        for n in x.shape[1:]:
            expected *= n
        if not x.is_contiguous():
            inside = 1
            for n, stride in zip(reversed(x.shape[1:]), reversed(x.stride()[1:])):
                if n != 1 and stride != inside:
                    raise ValueError("a state's rows must be contiguous")
                inside *= n
            if x.shape[0] > 1 and x.stride(0) < expected:
                raise ValueError("a state's rows must not overlap")
        size = x.element_size()
        count = 1
        for s in inner:
            count *= s
        desc = _lib.BeamState(x.data_ptr(), max(x.stride(0), expected) * size, count * size)
        if any(_meet(desc, other, groups * beams) for other in descs):
            raise ValueError("states must not overlap")
        descs.append(desc)
    lib = _library(index)
    with _lib.on_device(parents.device):
        for i in range(0, len(descs), 8):
            some = descs[i:i + 8]
            check(lib.lng_beam_reorder(ptr(parents), groups, beams, (_lib.BeamState * len(some))(*some), len(some), stream_ptr()),
                  "beam_reorder")
