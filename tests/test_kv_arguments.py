"""Arguments of the paged cache's calls at the edges of what they take, without a GPU."""

from __future__ import annotations

import ctypes as C

import pytest
import torch

from tests.test_kv_refusals import make

BF = dict(dtype=torch.bfloat16)


def test_scales_whose_base_2_form_overflows(lngram):
    """Scores are kept in base 2: scale * log2(e) has to be finite in fp32, 2.35e38 at most for the scale."""
    c, q = make(lngram), torch.zeros(2, 3, 4, 64, **BF)
    for scale in (2.4e38, 2.9e38, 3.3e38, 1e300):
        with pytest.raises(ValueError, match="scale"):
            lngram.kv_attend(c, q, scale=scale)
    with pytest.raises(RuntimeError, match="no CPU path"):
        lngram.kv_attend(c, q, scale=2.3e38)
    _lib = lngram._lib
    if not _lib.LIB_PATH.exists():
        pytest.skip("library not built")
    lib = _lib.library(require_device=False)
    cache = _lib.KvCache(k=4096, v=8192, dtype=_lib.BF16, page_size=16, num_pages=4, num_kv_heads=2, head_dim=64,
                         k_page_stride=2048, k_head_stride=1024, k_slot_stride=64, v_page_stride=2048, v_head_stride=1024,
                         v_slot_stride=64, table=256, table_stride=2, max_pages=2, lengths=512, batch=2)
    rows = [_lib.KvRows(ptr=1 << p, token_stride=256, head_stride=64, heads=4) for p in (20, 21)]
    # (addresses that are never read: the scale is judged before anything is launched)
    for scale in (2.4e38, 2.9e38):
        assert lib.lng_kv_attend(C.byref(cache), None, 6, 3, 0, C.byref(rows[0]), scale, 0, 0, C.byref(rows[1]), None, 0,
                                 None) == _lib.ERR_ARGUMENT
        assert b"scale" in lib.lng_last_error()


@pytest.mark.parametrize("kw, error", [(dict(window=None), TypeError), (dict(sinks="x"), ValueError), (dict(scale=[]), TypeError),
                                       (dict(max_len=float("inf")), OverflowError), (dict(out=3), AttributeError)])
def test_a_step_refused_after_the_append_leaves_lengths(lngram, monkeypatch, kw, error):
    """Whatever ends the step behind ``extend``; the append is a stand-in that takes everything."""
    import sys
    monkeypatch.setattr(sys.modules[lngram.kv_append.__module__], "kv_append", lambda cache, k, v, q, **_: q)
    c, q, k = make(lngram), torch.zeros(2, 3, 4, 64, **BF), torch.zeros(2, 3, 2, 64, **BF)
    c.lengths.copy_(torch.tensor([5, 7], dtype=torch.int32))
    with pytest.raises(error):
        lngram.attention_step(c, q, k, k, **kw)
    cu = torch.tensor([0, 1, 6], dtype=torch.int32)
    with pytest.raises(error):
        lngram.attention_step(c, q.view(6, 4, 64), k.view(6, 2, 64), k.view(6, 2, 64), cu=cu, max_new=5, **kw)
    assert c.lengths.tolist() == [5, 7]


def test_no_gradients_of_anything(lngram):
    """Not of the frequencies, the pages, the outputs or a tangent either: nothing is lost without a word."""
    import torch.autograd.forward_ad as fwd
    q, k = torch.zeros(2, 3, 4, 64, **BF), torch.zeros(2, 3, 2, 64, **BF)
    freq, table = torch.ones(32), torch.zeros(1, dtype=torch.int32)
    c, cg = make(lngram), make(lngram, k=torch.zeros(4, 2, 16, 64, **BF).requires_grad_())
    qg, freqg = q.clone().requires_grad_(), freq.clone().requires_grad_()
    calls = [lambda: lngram.kv_append(c, k, k, q, inv_freq=freqg), lambda: lngram.kv_append(c, k, k, q, q_out=qg),
             lambda: lngram.kv_append(cg, k, k), lambda: lngram.kv_attend(cg, q), lambda: lngram.kv_attend(c, q, out=qg),
             lambda: lngram.kv_prefix_attend(cg, q, table, 3), lambda: lngram.kv_prefix_attend(c, q, table, 3, out=qg),
             lambda: lngram.attention_step(c, q, k, k, inv_freq=freqg)]
    for call in calls:
        with pytest.raises(RuntimeError, match="no backward"):
            call()
        with torch.no_grad(), pytest.raises(RuntimeError, match="no CPU path"):
            call()
    with fwd.dual_level():
        qd, kd, fd = (fwd.make_dual(x, torch.ones_like(x)) for x in (q, k, freq))
        for call in (lambda: lngram.kv_attend(c, qd), lambda: lngram.kv_append(c, kd, k), lambda: lngram.kv_append(c, k, kd),
                     lambda: lngram.kv_append(c, k, k, q, inv_freq=fd), lambda: lngram.kv_prefix_attend(c, qd, table, 3)):
            for mode in (torch.no_grad(), torch.enable_grad()):
                with mode, pytest.raises(RuntimeError, match="tangent"):
                    call()
        with pytest.raises(RuntimeError, match="no CPU path"):
            lngram.kv_attend(c, q)
    assert c.lengths.tolist() == [0, 0]
