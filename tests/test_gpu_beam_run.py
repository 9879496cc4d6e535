"""A beam search with everything it needs -- pages from lengths, append, attention, the memory layer's cache, selection,
reordering -- against the same steps on caches of which every beam owns a copy, moved by ``index_select``."""

from __future__ import annotations

import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("eight", [False, True])
@pytest.mark.parametrize("groups, beams, page", [(1, 4, 8), (3, 5, 16)])
def test_beam_search(lngram, eight, groups, beams, page):
    g = torch.Generator(device="cuda").manual_seed(groups)
    heads, kv, dim, vocab, routes, hidden, steps, prompt = 8, 2, 32, 500, 6, 24, 30, 21
    batch, longest = groups * beams, prompt + steps
    bf = torch.bfloat16

    def weights(*shape):
        return (torch.randn(*shape, generator=g, device="cuda") / shape[0] ** 0.5).to(bf)

    embed, wq, wk, wv = weights(vocab, 64) * 20, weights(64, heads * dim), weights(64, kv * dim), weights(64, kv * dim)
    head = weights(heads * dim, vocab) * 3
    freq = (1000.0 ** (-torch.arange(dim // 2, device="cuda", dtype=torch.float64) / (dim // 2))).float()
    # one beam's worth of pages is shared by all beams of a group to begin with
    pool = lngram.PagePool.allocate(batch, longest, batch * (longest // page + 3), kv, dim, page_size=page, device="cuda", eight=eight, layers=2)
    kind = lngram.PagedKVCache8 if eight else lngram.PagedKVCache
    own = [kind.allocate(batch, longest, kv, dim, page_size=page, dtype=bf, device="cuda") for _ in range(2)]
    memory, memory_own = (type("Cache", (lngram.MemoryCache,), {"__init__": lambda self: None})() for _ in range(2))
    for m in (memory, memory_own):
        m.batch, m.max_len, m.length = batch, longest, 0
        m.codes = torch.zeros(batch, longest, routes, dtype=torch.uint8, device="cuda")
        m.conv_in = torch.zeros(batch, longest, hidden, dtype=bf, device="cuda")

    def layers(caches, x):
        out = 0
        for i, cache in enumerate(caches):
            y = torch.roll(x, i, -1)
            q, k, v = (y @ wq).view(*x.shape[:2], heads, dim), (y @ wk).view(*x.shape[:2], kv, dim), (y @ wv).view(*x.shape[:2], kv, dim)
            q = lngram.kv_append(cache, k, v, q, inv_freq=freq)
            out = out + lngram.kv_attend(cache, q)
        return out.flatten(2)

    def remember(m, tokens):
        n = tokens.shape[1]
        m.codes[:, m.length:m.length + n] = (tokens[..., None] + torch.arange(routes, device="cuda")) % 16
        m.conv_in[:, m.length:m.length + n] = embed[tokens][..., :hidden]
        m.length += n

    tokens = torch.randint(0, vocab, (groups, prompt), generator=g, device="cuda").repeat_interleave(beams, 0)
    scores = torch.full((groups, beams), -float("inf"), device="cuda")
    scores[:, 0] = 0
    done = torch.zeros(groups, beams, dtype=torch.bool, device="cuda")
    texts = tokens
    for step in range(steps):
        n = tokens.shape[1]
        if step == 0:
            # the prompt once a group; the other beams take it over
            first = torch.arange(batch, device="cuda") % beams == 0
            cu = torch.cat((torch.zeros(1, dtype=torch.int32, device="cuda"), (first * n).cumsum(0).to(torch.int32)))
            _, served = pool.extend(cu=cu, max_new=n, tokens=groups * n)
            x = embed[tokens[first]]
            for i, cache in enumerate(pool.caches):
                y = torch.roll(x, i, -1).flatten(0, 1)
                lngram.kv_append(cache, (y @ wk).view(-1, kv, dim), (y @ wv).view(-1, kv, dim), inv_freq=freq, cu=cu, max_new=n)
            pool.reorder(torch.zeros(groups, beams, dtype=torch.int64, device="cuda"))
            assert int(pool.refs.max()) == beams
            used = groups * -(-n // page)
            assert int((pool.refs > 0).sum()) == used
            for c in own:
                c.extend(n)
            got = layers(own, embed[tokens])[:, -1]
            # (the pool's own attention to the last token of the prompt)
            q0 = 0
            for i, cache in enumerate(pool.caches):
                y = torch.roll(embed[tokens[:, -1:]], i, -1)
                q = (y @ wq).view(batch, 1, heads, dim)
                spare = torch.empty(batch, 1, kv, dim, dtype=bf, device="cuda")
                scratch = kind.allocate(batch, 1, kv, dim, page_size=page, dtype=bf, device="cuda")
                scratch.extend(1)
                q = lngram.kv_append(scratch, spare.zero_(), spare, q, inv_freq=freq,
                                     positions=torch.full((batch, 1), n - 1, dtype=torch.int64, device="cuda"))
                q0 = q0 + lngram.kv_attend(cache, q)
            h = q0.flatten(2)[:, 0]
            assert (h.float() - got.float()).abs().max() <= 2.0 ** -5 * got.float().abs().max()
            h = got
        else:
            _, served = pool.extend(n)
            for c in own:
                c.extend(n)
            h, want = layers(pool.caches, embed[tokens])[:, -1], layers(own, embed[tokens])[:, -1]
            assert torch.equal(h, want)
        assert served.all()
        for m in (memory, memory_own):
            remember(m, tokens)
        logits = (h @ head).view(groups, beams, vocab)
        scores, chosen, parents = lngram.beam_select(logits, scores, done=done if step else None, eos=7)
        rows = (parents + torch.arange(groups, device="cuda")[:, None] * beams).flatten()
        pool.reorder(parents)
        memory.reorder(parents)
        memory_own.codes, memory_own.conv_in = memory_own.codes[rows], memory_own.conv_in[rows]
        for c in own:
            per = c.table.shape[1]
            for t in ((c.k.view(torch.uint8), c.v.view(torch.uint8), c.k_exp, c.v_exp) if eight else (c.k, c.v)):
                t.copy_(t.view(batch, per, *t.shape[1:])[rows].reshape(t.shape))
        done = done.gather(1, parents) | (chosen == 7)
        tokens = chosen.view(batch, 1)
        texts = torch.cat((texts[rows], tokens), 1)
        assert torch.equal(memory.codes[:, :memory.length], memory_own.codes[:, :memory.length])
        assert torch.equal(memory.conv_in[:, :memory.length], memory_own.conv_in[:, :memory.length])
        assert (scores[:, :-1] >= scores[:, 1:]).all()
    # the codes of a beam's cache are those of its text
    want = (texts[:, :memory.length, None] + torch.arange(routes, device="cuda")) % 16
    assert torch.equal(memory.codes[:, :memory.length].long(), want)
    pool.truncate(0)
    assert (pool.refs == 0).all() and (pool.cache.table == -1).all() and (pool.cache.lengths == 0).all()
    assert lngram._lib.device_error() == 0
