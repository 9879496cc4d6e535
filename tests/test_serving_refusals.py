"""What the 8-bit cache, the page pool and beam search refuse, without a GPU: the Python checks on CPU tensors, and the C
entries' own, which come before any CUDA call."""

from __future__ import annotations

import ctypes as C

import pytest
import torch
import torch.autograd.forward_ad as fwd

BF = dict(dtype=torch.bfloat16)
E4M3 = torch.float8_e4m3fn


def pages8(*shape):
    return torch.zeros(*shape, dtype=torch.uint8).view(E4M3)


def make8(lngram, batch=2, pages=4, heads=2, size=16, dim=64, per=2, dtype=torch.bfloat16, **kw):
    args = dict(k=pages8(pages, heads, size, dim), v=pages8(pages, heads, size, dim), k_exp=torch.zeros(pages, heads, dtype=torch.int8),
                v_exp=torch.zeros(pages, heads, dtype=torch.int8), table=torch.zeros(batch, per, dtype=torch.int32),
                lengths=torch.zeros(batch, dtype=torch.int32))
    return lngram.PagedKVCache8(*{**args, **kw}.values(), dtype=dtype)


@pytest.mark.parametrize("kw, match", [
    (dict(dtype=torch.float32), "bfloat16 or float16"),
    (dict(k=torch.zeros(4, 2, 16, 64, **BF)), "float8_e4m3fn"),
    (dict(v=pages8(4, 2, 16, 32)), "alike"),
    (dict(size=12), "power of two"), (dict(size=512), "power of two"), (dict(size=4), "power of two"),
    (dict(dim=24), "head_dim"), (dict(dim=144), "head_dim"), (dict(dim=8), "head_dim"),
    (dict(k=pages8(4, 2, 16, 72)[..., :64]), "multiples of 16"),
    (dict(k=pages8(1, 2, 16, 64).expand(4, 2, 16, 64)), "positive"),
    (dict(k=pages8(4, 2, 16, 80)[..., 8:72]), "16-byte"),
    (dict(k_exp=torch.zeros(4, 2, dtype=torch.int32)), "int8"),
    (dict(v_exp=torch.zeros(4, 3, dtype=torch.int8)), "int8"),
    (dict(v_exp=torch.zeros(2, 4, dtype=torch.int8).t()), "contiguous rows"),
    (dict(k_exp=torch.zeros(1, 2, dtype=torch.int8).expand(4, 2)), "contiguous rows"),
    (dict(table=torch.zeros(2, 2, dtype=torch.int64)), "int32"),
    (dict(lengths=torch.zeros(3, dtype=torch.int32)), "one row a sequence"),
])
def test_cache8_refusals(lngram, kw, match):
    with pytest.raises(ValueError, match=match):
        make8(lngram, **kw)


def test_steps_of_an_8_bit_cache(lngram):
    c = make8(lngram)
    q, k = torch.zeros(2, 3, 4, 64, **BF), torch.zeros(2, 3, 2, 64, **BF)
    for call, match in [
        (lambda: lngram.kv_attend(c, q.half()), "dtype"),
        (lambda: lngram.kv_append(c, pages8(2, 3, 2, 64), k), "dtype"),
        (lambda: lngram.kv_attend(c, torch.zeros(2, 3, 3, 64, **BF)), "multiple of the key heads"),
        (lambda: lngram.kv_attend(c, q, out=q), "overlap"),
        (lambda: lngram.kv_prefix_attend(c, q, torch.zeros(1, dtype=torch.int32), 3), "16 bits"),
        (lambda: lngram.kv_append(c, k, k, inv_freq=torch.ones(33)), "more pairs"),
    ]:
        with pytest.raises(ValueError, match=match):
            call()
    for call in (lambda: lngram.kv_append(c, k, k), lambda: lngram.kv_attend(c, q), lambda: c.values(),
                 lambda: lngram.attention_step(c, q, k, k)):
        with pytest.raises(RuntimeError, match="no CPU path"):
            call()
    assert c.lengths.tolist() == [0, 0]
    with pytest.raises(RuntimeError, match="no backward"):
        lngram.kv_attend(c, q.clone().requires_grad_())
    with fwd.dual_level(), pytest.raises(RuntimeError, match="tangent"):
        lngram.kv_append(c, fwd.make_dual(k, torch.ones_like(k)), k)


def cache16(lngram, batch=2, pages=6, heads=1, size=8, dim=16, per=2, table=None, lengths=None):
    k, v = (torch.zeros(pages, heads, size, dim, **BF) for _ in range(2))
    return lngram.PagedKVCache(k, v, torch.zeros(batch, per, dtype=torch.int32) if table is None else table,
                               torch.zeros(batch, dtype=torch.int32) if lengths is None else lengths)


def test_pool_refusals(lngram):
    a = cache16(lngram)
    for call, match in [
        (lambda: lngram.PagePool([]), "at least one"),
        (lambda: lngram.PagePool([a, cache16(lngram)]), "share one table"),
        (lambda: lngram.PagePool([a, cache16(lngram, size=16, table=a.table, lengths=a.lengths)]), "one size"),
        (lambda: lngram.PagePool([a, cache16(lngram, pages=7, table=a.table, lengths=a.lengths)]), "equally many"),
        (lambda: lngram.PagePool(a, torch.zeros(5, dtype=torch.int32)), "refs must be"),
        (lambda: lngram.PagePool(a, torch.zeros(6, dtype=torch.int64)), "refs must be"),
        (lambda: lngram.PagePool(a, torch.zeros(12, dtype=torch.int32)[::2]), "refs must be"),
        (lambda: lngram.PagePool(cache16(lngram, per=0)), "no columns"),
        (lambda: lngram.PagePool(cache16(lngram, batch=8193)), "8192"),
    ]:
        with pytest.raises(ValueError, match=match):
            call()
    pool = lngram.PagePool(a, torch.ones(6, dtype=torch.int32))
    cu = torch.tensor([0, 1, 2], dtype=torch.int32)
    for call, match in [
        (lambda: pool.extend(), "needs n"), (lambda: pool.extend(3, cu=cu, max_new=3), "needs n"), (lambda: pool.extend(cu=cu), "needs n"),
        (lambda: pool.extend(3, max_new=4), "needs n"), (lambda: pool.extend(3, tokens=5), "needs n"), (lambda: pool.extend(-1), "negative"),
        (lambda: pool.extend(cu=cu, max_new=1, tokens=-2), "negative"),
        (lambda: pool.extend(cu=cu.long(), max_new=3), "int32"), (lambda: pool.extend(cu=cu[:2], max_new=3), "int32"),
        (lambda: pool.truncate(-1), "negative"), (lambda: pool.truncate(torch.zeros(2)), "int32"),
        (lambda: pool.truncate(torch.zeros(3, dtype=torch.int32)), "int32"),
        (lambda: pool.reorder(torch.zeros(2, dtype=torch.int64)), "groups, beams"),
        (lambda: pool.reorder(torch.zeros(1, 2, dtype=torch.int32)), "int64"),
        (lambda: pool.reorder(torch.zeros(1, 3, dtype=torch.int64)), "2 rows"),
    ]:
        with pytest.raises(ValueError, match=match):
            call()
    for call in (lambda: pool.extend(1), lambda: pool.truncate(0), lambda: pool.reorder(torch.zeros(1, 2, dtype=torch.int64))):
        with pytest.raises(RuntimeError, match="no CPU path"):
            call()


def test_beam_refusals(lngram):
    x, s = torch.zeros(2, 3, 10), torch.zeros(2, 3)
    done = torch.zeros(2, 3, dtype=torch.bool)
    for call, match in [
        (lambda: lngram.beam_select(x.double(), s), "float32, bfloat16"), (lambda: lngram.beam_select(x[0], s), "groups, beams, vocab"),
        (lambda: lngram.beam_select(torch.zeros(1, 33, 4), torch.zeros(1, 33)), "32 beams"),
        (lambda: lngram.beam_select(torch.zeros(1, 3, 0), torch.zeros(1, 3)), "vocab"),
        (lambda: lngram.beam_select(x, s, width=0), "width"), (lambda: lngram.beam_select(x, s, width=33), "width"),
        (lambda: lngram.beam_select(x[..., :1], s, width=4), "width"),
        (lambda: lngram.beam_select(x, s.half()), "scores"), (lambda: lngram.beam_select(x, s[:1]), "scores"),
        (lambda: lngram.beam_select(x, s.t().contiguous().t()), "scores"),
        (lambda: lngram.beam_select(x.transpose(1, 2).contiguous().transpose(1, 2), s), "one stride"),
        (lambda: lngram.beam_select(torch.zeros(2, 4, 10)[:, :3], s), "one stride"),
        (lambda: lngram.beam_select(x[:, :1].expand(2, 3, 10), s), "one stride"),
        (lambda: lngram.beam_select(x, s, done=done), "eos"), (lambda: lngram.beam_select(x, s, done=done, eos=10), "eos"),
        (lambda: lngram.beam_select(x, s, done=done.int(), eos=1), "bool"), (lambda: lngram.beam_select(x, s, done=done[:1], eos=1), "bool"),
    ]:
        with pytest.raises(ValueError, match=match):
            call()
    parents = torch.zeros(2, 3, dtype=torch.int64)
    for call, match in [
        (lambda: lngram.beam_reorder(parents.int(), x), "int64"), (lambda: lngram.beam_reorder(parents[0], x), "groups, beams"),
        (lambda: lngram.beam_reorder(torch.zeros(1, 33, dtype=torch.int64)), "32 beams"),
        (lambda: lngram.beam_reorder(parents, torch.zeros(5, 4)), "6 rows"),
        (lambda: lngram.beam_reorder(parents, torch.zeros(6, 4, 4).transpose(1, 2)[:, ::2]), "contiguous"),
        (lambda: lngram.beam_reorder(parents, torch.zeros(1, 4).expand(6, 4)), "overlap"),
        (lambda: lngram.beam_reorder(parents, torch.zeros(6, 4), length=5), "length"),
        (lambda: lngram.beam_reorder(parents, torch.zeros(6), length=1), "length"),
        (lambda: lngram.beam_reorder(parents, torch.zeros(6, 4), length=-1), "length"),
    ]:
        with pytest.raises(ValueError, match=match):
            call()
    for call in (lambda: lngram.beam_select(x, s), lambda: lngram.beam_reorder(parents, torch.zeros(6, 4))):
        with pytest.raises(RuntimeError, match="no CPU path"):
            call()
    for call in (lambda: lngram.beam_select(x.clone().requires_grad_(), s), lambda: lngram.beam_select(x, s.clone().requires_grad_()),
                 lambda: lngram.beam_reorder(parents, torch.zeros(6, 4, requires_grad=True))):
        with pytest.raises(RuntimeError, match="no backward"):
            call()
    with fwd.dual_level(), pytest.raises(RuntimeError, match="tangent"):
        lngram.beam_select(fwd.make_dual(x, x), s)


def test_c_entries_refuse_before_any_launch(lngram):
    """Addresses that are never read: every call here returns LNG_ERR_ARGUMENT (or has nothing to do)."""
    _lib = lngram._lib
    if not _lib.LIB_PATH.exists():
        pytest.skip("library not built")
    lib = _lib.library(require_device=False)
    pages = dict(k=4096, v=8192, dtype=_lib.BF16, page_size=16, num_pages=4, num_kv_heads=2, head_dim=64, k_page_stride=2048,
                 k_head_stride=1024, k_slot_stride=64, v_page_stride=2048, v_head_stride=1024, v_slot_stride=64, table=256,
                 table_stride=2, max_pages=2, lengths=512, batch=2)
    rows = dict(ptr=1 << 20, token_stride=256, head_stride=64, heads=4)
    bad_arg = _lib.ERR_ARGUMENT

    def cache(over=None, **kw):
        exps = dict(k_exp=64, v_exp=128, k_exp_stride=2, v_exp_stride=2)
        return C.byref(_lib.KvCache8(pages=_lib.KvCache(**{**pages, **(over or {})}), **{**exps, **kw}))

    def attend(c, r=None, o=None, tokens=6, scale=0.125, window=0, max_len=0):
        q, out = _lib.KvRows(**{**rows, **(r or {})}), _lib.KvRows(**{**rows, "ptr": 1 << 21, **(o or {})})
        return lib.lng_kv8_attend(c, None, tokens, 3, max_len, C.byref(q), scale, window, 0, C.byref(out), 1 << 22, 1 << 40, None)

    def append(c, k=None, rotary=64, freq=64):
        kr = _lib.KvRows(**{**rows, "heads": 2, **(k or {})})
        return lib.lng_kv8_append(c, None, 6, 3, C.byref(kr), C.byref(kr), None, None, None, freq, rotary, 0, None)

    for c in (cache(dict(head_dim=72)), cache(dict(page_size=512)), cache(dict(k_slot_stride=72)), cache(dict(v_page_stride=2056)),
              cache(dict(dtype=_lib.F32)), cache(k_exp=None), cache(v_exp=None), cache(k_exp_stride=1), cache(dict(k=None)),
              cache(dict(lengths=None))):
        assert attend(c) == bad_arg and append(c) == bad_arg
    for kw in (dict(r=dict(heads=3)), dict(r=dict(ptr=8)), dict(o=dict(ptr=1 << 20)), dict(tokens=5), dict(scale=-1.0),
               dict(scale=2.4e38), dict(window=-1), dict(max_len=-1), dict(r=dict(heads=258))):
        assert attend(cache(), **kw) == bad_arg, kw
    for kw in (dict(k=dict(heads=3)), dict(rotary=65), dict(rotary=66), dict(freq=None), dict(k=dict(token_stride=4))):
        assert append(cache(), **kw) == bad_arg, kw
    assert lib.lng_kv8_values(cache(), 8, None, None) == bad_arg and lib.lng_kv8_values(cache(k_exp=None), 16, None, None) == bad_arg

    extend = lambda c, refs=64, tokens=6, slots=64, served=64, copies=64, count=1: lib.lng_kv_pages_extend(  # noqa: E731
        c, count, refs, None, tokens, 3, slots, served, copies, None)
    for c in (cache(k_exp=None), cache(dict(batch=8193)), cache(dict(num_pages=(1 << 22) + 1)), cache(dict(max_pages=0))):
        assert extend(c) == bad_arg
    for kw in (dict(refs=None), dict(slots=None), dict(served=None), dict(copies=None), dict(copies=72), dict(tokens=4), dict(count=0)):
        assert extend(cache(), **kw) == bad_arg, kw
    assert lib.lng_kv_pages_truncate(cache(), None, None, 3, None) == bad_arg
    assert lib.lng_kv_pages_truncate(cache(), 64, None, -1, None) == bad_arg
    assert lib.lng_kv_pages_reorder(cache(), 64, 64, 1, 3, None) == bad_arg
    assert lib.lng_kv_pages_reorder(cache(), 64, None, 1, 2, None) == bad_arg
    assert extend(cache(dict(batch=0)), tokens=0) == _lib.OK

    def select(dtype=_lib.F32, stride=10, groups=2, beams=3, vocab=10, logits=4096, eos=0, width=3, done=None, ws=1 << 20, need=1 << 30):
        return lib.lng_beam_select(logits, dtype, stride, groups, beams, vocab, 64, done, eos, width, 64, 64, 64, ws, need, None)

    for kw in (dict(dtype=_lib.I32), dict(stride=9), dict(groups=-1), dict(beams=0), dict(beams=33), dict(vocab=0), dict(width=0),
               dict(width=33), dict(width=31), dict(logits=None), dict(logits=4098), dict(done=64, eos=10), dict(ws=None), dict(ws=128), dict(need=0)):
        assert select(**kw) == bad_arg, kw
    assert select(groups=0) == _lib.OK
    one = (_lib.BeamState * 1)(_lib.BeamState(4096, 16, 32))
    assert lib.lng_beam_reorder(64, 2, 3, one, 1, None) == bad_arg
    one[0] = _lib.BeamState(4096, 32, 32)
    for args in ((64, 2, 0, one, 1), (64, 2, 33, one, 1), (64, 65536, 3, one, 1), (None, 2, 3, one, 1), (64, 2, 3, one, 9), (64, 2, 3, one, -1)):
        assert lib.lng_beam_reorder(*args, None) == bad_arg, args
    assert lib.lng_beam_reorder(64, 2, 3, one, 0, None) == _lib.OK
