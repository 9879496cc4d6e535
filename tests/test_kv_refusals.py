"""What the paged cache's calls refuse, without a GPU: the Python checks on CPU tensors and the C entries'
own argument checks, which all come before any CUDA call."""

from __future__ import annotations

import ctypes as C

import pytest
import torch


def make(lngram, batch=2, pages=4, heads=2, size=16, dim=64, per=2, dtype=torch.bfloat16, **kw):
    k = kw.get("k", torch.zeros(pages, heads, size, dim, dtype=dtype))
    v = kw.get("v", torch.zeros(pages, heads, size, dim, dtype=dtype))
    table = kw.get("table", torch.zeros(batch, per, dtype=torch.int32))
    lengths = kw.get("lengths", torch.zeros(batch, dtype=torch.int32))
    return lngram.PagedKVCache(k, v, table, lengths)


@pytest.mark.parametrize("kw, match", [
    (dict(dtype=torch.float32), "bfloat16 or float16"),
    (dict(size=12), "power of two"),
    (dict(size=4), "power of two"),
    (dict(dim=136), "head_dim"),
    (dict(dim=12), "head_dim"),
    (dict(v=torch.zeros(4, 2, 16, 32, dtype=torch.bfloat16)), "alike"),
    (dict(k=torch.zeros(4, 2, 16, 128, dtype=torch.bfloat16)[..., ::2]), "contiguous"),
    (dict(k=torch.zeros(4, 2, 16, 68, dtype=torch.bfloat16)[..., :64]), "multiples of 8"),
    (dict(k=torch.zeros(1, 2, 16, 64, dtype=torch.bfloat16).expand(4, 2, 16, 64)), "positive"),
    (dict(table=torch.zeros(2, 2, dtype=torch.int64)), "int32"),
    (dict(table=torch.zeros(2, 1 << 26, dtype=torch.int32)), "2\\^30"),
    (dict(lengths=torch.zeros(3, dtype=torch.int32)), "one row a sequence"),
    (dict(lengths=torch.zeros(2)), "int32"),
])
def test_cache_refusals(lngram, kw, match):
    with pytest.raises(ValueError, match=match):
        make(lngram, **kw)


def test_step_refusals(lngram):
    c = make(lngram)
    bf = dict(dtype=torch.bfloat16)
    q, k = torch.zeros(2, 3, 4, 64, **bf), torch.zeros(2, 3, 2, 64, **bf)
    cu = torch.tensor([0, 3, 6], dtype=torch.int32)
    freq = torch.ones(32)
    for call, match in [
        (lambda: lngram.kv_attend(c, q.half()), "dtype"),
        (lambda: lngram.kv_attend(c, torch.zeros(2, 3, 4, 32, **bf)), "must be"),
        (lambda: lngram.kv_attend(c, torch.zeros(3, 3, 4, 64, **bf)), "without cu"),
        (lambda: lngram.kv_attend(c, torch.zeros(6, 4, 64, **bf)), "without cu"),
        (lambda: lngram.kv_attend(c, q, max_new=4), "max_new"),
        (lambda: lngram.kv_attend(c, q, cu=cu, max_new=3), "with cu"),
        (lambda: lngram.kv_attend(c, q.view(6, 4, 64), cu=cu), "max_new"),
        (lambda: lngram.kv_attend(c, q.view(6, 4, 64), cu=cu.long(), max_new=3), "int32"),
        (lambda: lngram.kv_attend(c, q.view(6, 4, 64), cu=cu[:2], max_new=3), "cu must be"),
        (lambda: lngram.kv_attend(c, torch.zeros(2, 3, 3, 64, **bf)), "multiple of the key heads"),
        (lambda: lngram.kv_attend(c, torch.zeros(2, 3, 258, 64, **bf)), "128"),
        (lambda: lngram.kv_attend(c, q, window=-1), "negative"),
        (lambda: lngram.kv_attend(c, q, sinks=-1), "negative"),
        (lambda: lngram.kv_attend(c, q, scale=0.0), "scale"),
        (lambda: lngram.kv_attend(c, q, scale=float("nan")), "scale"),
        (lambda: lngram.kv_attend(c, q, max_len=-1), "max_len"),
        (lambda: lngram.kv_attend(c, q, out=q), "overlap"),
        (lambda: lngram.kv_attend(c, q, out=torch.zeros(2, 3, 6, 64, **bf)), "heads"),
        (lambda: lngram.kv_attend(c, torch.zeros(2, 3, 4, 65, **bf)[..., 1:]), "16-byte"),
        (lambda: lngram.kv_attend(c, torch.zeros(2, 4, 4, 64, **bf)[:, :3]), "one stride"),
        (lambda: lngram.kv_prefix_attend(c, q, torch.zeros(1, dtype=torch.int32), 17), "too few pages"),
        (lambda: lngram.kv_prefix_attend(c, q, torch.zeros(1, dtype=torch.int64), 3), "int32"),
        (lambda: lngram.kv_prefix_attend(c, q, torch.zeros(1, dtype=torch.int32), -1), "prefix_len"),
        (lambda: lngram.kv_append(c, k, k[:, :2]), "leading shape"),
        (lambda: lngram.kv_append(c, q, q), "heads"),
        (lambda: lngram.kv_append(c, k, k, q[:, :2]), "leading shape"),
        (lambda: lngram.kv_append(c, k, k, q_out=q), "without q"),
        (lambda: lngram.kv_append(c, k, k, inv_freq=freq.double()), "fp32"),
        (lambda: lngram.kv_append(c, k, k, inv_freq=torch.ones(33)), "more pairs"),
        (lambda: lngram.kv_append(c, k, k, inv_freq=freq, positions=torch.zeros(2, 3)), "int64"),
        (lambda: lngram.kv_append(c, k, k, inv_freq=freq, positions=torch.zeros(6, dtype=torch.int64)), "leading shape"),
    ]:
        with pytest.raises(ValueError, match=match):
            call()


def test_cpu_tensors_are_refused(lngram):
    c = make(lngram)
    q, k = torch.zeros(2, 1, 4, 64, dtype=torch.bfloat16), torch.zeros(2, 1, 2, 64, dtype=torch.bfloat16)
    for call in (lambda: lngram.kv_append(c, k, k), lambda: lngram.kv_attend(c, q),
                 lambda: lngram.kv_prefix_attend(c, q, torch.zeros(1, dtype=torch.int32), 4)):
        with pytest.raises(RuntimeError, match="CUDA"):
            call()


def test_c_entries_refuse_before_any_launch(lngram):
    """Addresses that are never read: every call here returns LNG_ERR_ARGUMENT (or has nothing to do)."""
    _lib = lngram._lib
    if not _lib.LIB_PATH.exists():
        pytest.skip("library not built")
    lib = _lib.library(require_device=False)
    good = dict(k=4096, v=8192, dtype=_lib.BF16, page_size=16, num_pages=4, num_kv_heads=2, head_dim=64, k_page_stride=2048,
                k_head_stride=1024, k_slot_stride=64, v_page_stride=2048, v_head_stride=1024, v_slot_stride=64, table=256,
                table_stride=2, max_pages=2, lengths=512, batch=2)
    rows = dict(ptr=1 << 20, token_stride=256, head_stride=64, heads=4)

    def attend(cache=None, r=None, o=None, cu=None, tokens=6, max_new=3, max_len=0, scale=0.125, window=0, sinks=0, ws=1 << 22,
               need=1 << 40, prefix=None, prefix_len=0):
        c = C.byref(_lib.KvCache(**{**good, **(cache or {})}))
        q, out = _lib.KvRows(**{**rows, **(r or {})}), _lib.KvRows(**{**rows, "ptr": 1 << 21, **(o or {})})
        if prefix_len:
            return lib.lng_kv_prefix_attend(c, prefix, prefix_len, cu, tokens, max_new, max_len, C.byref(q), scale,
                                            C.byref(out), ws, need, None)
        return lib.lng_kv_attend(c, cu, tokens, max_new, max_len, C.byref(q), scale, window, sinks, C.byref(out), ws, need, None)

    for bad in (dict(dtype=_lib.F32), dict(page_size=24), dict(page_size=8192), dict(num_pages=0), dict(head_dim=132),
                dict(head_dim=0), dict(num_kv_heads=0), dict(max_pages=1 << 26, table_stride=1 << 26), dict(table_stride=1),
                dict(k=None), dict(lengths=None), dict(table=None), dict(k=4104), dict(k_slot_stride=60), dict(v_page_stride=0),
                dict(batch=-1)):
        assert attend(cache=bad) == _lib.ERR_ARGUMENT, bad
    for bad in (dict(ptr=None), dict(ptr=8), dict(token_stride=4), dict(head_stride=-64), dict(heads=3), dict(heads=0),
                dict(heads=258)):
        assert attend(r=bad) == _lib.ERR_ARGUMENT, bad
    for bad in (dict(o=dict(heads=2)), dict(o=dict(ptr=1 << 20)), dict(tokens=5), dict(max_new=0, tokens=0, cu=64, scale=-1.0),
                dict(scale=float("inf")), dict(scale=float("nan")), dict(window=-1), dict(sinks=-2), dict(max_len=-1),
                dict(prefix_len=9), dict(prefix_len=-1, prefix=64)):
        assert attend(**bad) == _lib.ERR_ARGUMENT, bad
    assert attend(cache=dict(batch=0), tokens=0) == _lib.OK and attend(tokens=0, max_new=0) == _lib.OK

    def append(cache=None, k=None, v=None, q=None, qo=None, positions=None, freq=64, rotary=64, tokens=6, max_new=3):
        kr, vr = _lib.KvRows(**{**rows, "heads": 2, **(k or {})}), _lib.KvRows(**{**rows, "heads": 2, **(v or {})})
        return lib.lng_kv_append(C.byref(_lib.KvCache(**{**good, **(cache or {})})), None, tokens, max_new, C.byref(kr),
                                 C.byref(vr), q and C.byref(_lib.KvRows(**{**rows, **q})),
                                 qo and C.byref(_lib.KvRows(**{**rows, **qo})), positions, freq, rotary, 0, None)

    for bad in (dict(rotary=63), dict(rotary=66), dict(rotary=-2), dict(freq=None), dict(q=dict(heads=4)), dict(qo=dict(heads=4)),
                dict(q=dict(heads=4), qo=dict(heads=2)), dict(k=dict(heads=4)), dict(v=dict(ptr=None)), dict(k=dict(ptr=24)),
                dict(q=dict(heads=4), qo=dict(heads=4, token_stride=512))):
        assert append(**bad) == _lib.ERR_ARGUMENT, bad
    assert append(tokens=0, max_new=0) == _lib.OK


def test_overlapping_table_rows(lngram):
    # one row expanded over the batch, and rows that overlap: the kernels would walk past the row's end
    with pytest.raises(ValueError, match="overlap"):
        make(lngram, table=torch.zeros(1, 2, dtype=torch.int32).expand(2, 2))
    with pytest.raises(ValueError, match="overlap"):
        make(lngram, table=torch.zeros(4, dtype=torch.int32).as_strided((2, 3), (1, 1)))
    make(lngram, batch=1, table=torch.zeros(3, dtype=torch.int32).as_strided((1, 3), (1, 1)), lengths=torch.zeros(1, dtype=torch.int32))


def test_no_gradients(lngram):
    c = make(lngram)
    bf = dict(dtype=torch.bfloat16)
    q, k = torch.zeros(2, 3, 4, 64, **bf), torch.zeros(2, 3, 2, 64, **bf)
    qg, kg = q.clone().requires_grad_(), k.clone().requires_grad_()
    for call in (lambda: lngram.kv_attend(c, qg), lambda: lngram.kv_append(c, k, kg), lambda: lngram.kv_append(c, k, k, qg),
                 lambda: lngram.kv_prefix_attend(c, qg, torch.zeros(1, dtype=torch.int32), 3),
                 lambda: lngram.attention_step(c, q, kg, k)):
        with pytest.raises(RuntimeError, match="no backward"):
            call()
        with torch.no_grad(), pytest.raises(RuntimeError, match="no CPU path"):
            call()


def test_refused_step_leaves_lengths(lngram):
    c = make(lngram)
    bf = dict(dtype=torch.bfloat16)
    q, k = torch.zeros(2, 3, 4, 64, **bf), torch.zeros(2, 3, 2, 64, **bf)
    c.lengths.copy_(torch.tensor([5, 7], dtype=torch.int32))
    with pytest.raises(ValueError, match="dtype"):
        lngram.attention_step(c, q, k.half(), k)
    cu = torch.tensor([0, 1, 6], dtype=torch.int32)
    with pytest.raises(ValueError, match="dtype"):
        lngram.attention_step(c, q.view(6, 4, 64), k.view(6, 2, 64), k.view(6, 2, 64).half(), cu=cu, max_new=5)
    assert c.lengths.tolist() == [5, 7]
