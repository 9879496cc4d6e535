"""Operators of a beam or decode step around a paged cache that is held in 8 bits, as they are measured.

* ``append``: a step's new keys and values go to their slots of the cache, rounded to 8 bits (e4m3) under
  one exponent for each page and head, keys and queries rotated by their position on the way.
* ``attend``: causal attention of the newest tokens over that cache.
* ``pages``: the cache's page table and the new tokens' slots, made on the GPU from the requests' lengths: the
  pages of rejected drafts go back, the lowest free ones are handed out; sequences that beams have forked share their
  pages, and a page that is written to while others hold it is copied first.
* ``select``: the best continuations over a request's beams and the vocabulary.
* ``reorder``: the memory layer's cached codes and conv inputs follow the beams that were chosen.

An 8-bit cache is pages ``[pages, kv heads, page size, head size]`` of e4m3 for keys and for values with exponents
``[pages, kv heads]`` (a slot stands for its e4m3 value times 2^exponent), a table ``[batch, pages per
sequence]`` of page numbers and the sequences' lengths, the newest tokens counted.
"""

import math

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}
E4M3 = torch.float8_e4m3fn
LEAST, MOST = -40, 40  # the exponents that a page may have


# ---------------------------------------------------------------------------------------- the cases
def _cache_case(name, op, batch, new, ctx, heads, kv, dim, page, dtype, window=0, sinks=0, rotary=0, interleaved=False,
                shift=0):
    """``new`` and ``ctx`` are (smallest, largest) over the batch: tokens of this step, and tokens held before."""
    case = {"op": op, "batch": batch, "new_lo": new[0], "new_hi": new[1], "ctx_lo": ctx[0], "ctx_hi": ctx[1],
            "heads": heads, "kv": kv, "dim": dim, "page": page, "dtype": dtype, "window": window, "sinks": sinks,
            "rotary": rotary, "interleaved": interleaved, "shift": shift}
    return {"name": name, **case} if name else case


def _pages_case(name, groups, beams, new, ctx, kv, dim, page, spare):
    """``groups`` requests of ``beams`` sequences each (1: no beams) add ``new`` tokens; ``spare``: free pages."""
    case = {"op": "pages", "groups": groups, "beams": beams, "new": new, "ctx_lo": ctx[0], "ctx_hi": ctx[1], "kv": kv,
            "dim": dim, "page": page, "spare": spare}
    return {"name": name, **case} if name else case


def _select_case(name, groups, beams, vocab, dtype, done):
    """``done``: one of how many beams has ended (0: none)."""
    case = {"op": "select", "groups": groups, "beams": beams, "vocab": vocab, "dtype": dtype, "done": done}
    return {"name": name, **case} if name else case


def _reorder_case(name, groups, beams, length, routes, hidden, dtype):
    case = {"op": "reorder", "groups": groups, "beams": beams, "length": length, "routes": routes, "hidden": hidden,
            "dtype": dtype}
    return {"name": name, **case} if name else case


def listed():
    return [
        # one decode step of 64 sequences (the memory layer's heads: 16 query, 4 key, 64 wide)
        _cache_case("append_step", "append", 64, (1, 1), (100, 900), 16, 4, 64, 64, "bf16", rotary=64),
        # a batch of prompts as the memory layer's prefill takes them: 32 x 2048 positions
        _cache_case("append_prompt", "append", 32, (2048, 2048), (0, 0), 16, 4, 64, 64, "bf16", rotary=64),
        # one user, one token: nothing but latency
        _cache_case("attend_one", "attend", 1, (1, 1), (4095, 4095), 16, 4, 64, 64, "bf16"),
        # a decode step of a full batch whose sequences are of all lengths
        _cache_case("attend_step", "attend", 64, (1, 1), (500, 16000), 32, 8, 128, 64, "bf16"),
        # 16 drafted tokens a sequence verified after a context of 1024
        _cache_case("attend_verify", "attend", 64, (16, 16), (1024, 1024), 16, 4, 64, 64, "bf16"),
        # two long prompts of unlike lengths, 7 query heads a key head, small pages, a window and sinks
        _cache_case("attend_long", "attend", 2, (5001, 8000), (0, 999), 28, 4, 128, 16, "f16", window=4096, sinks=4),
        # 64 sequences give back the pages of the drafts that were rejected and make room for the next 16
        _pages_case("pages_drafts", 64, 1, 16, (100, 4000), 4, 64, 64, 1500),
        # 64 requests of 8 beams go one token on after a choice that has dropped some beams and forked others
        _pages_case("pages_beams", 64, 8, 1, (30, 2000), 4, 64, 64, 4000),
        # one request, four beams, a vocabulary of 32000
        _select_case("select_one", 1, 4, 32000, "f32", 0),
        # a batch of requests of eight beams over a large vocabulary, some beams ended
        _select_case("select_batch", 64, 8, 128000, "bf16", 9),
        # four beams of one request after a short text: the memory layer's 184 codes and 1024 conv inputs a position
        _reorder_case("reorder_one", 1, 4, 300, 184, 1024, "bf16"),
        # 16 requests of four beams after 2048 positions
        _reorder_case("reorder_batch", 16, 4, 2048, 184, 1024, "bf16"),
    ]


def _log(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    most = {}
    for case in listed():
        w = work(case)
        most[case["op"]] = {k: max(v, most.get(case["op"], {}).get(k, 0)) for k, v in w.items()}
    while True:
        op = rng.choice(["append", "attend", "attend", "pages", "select", "reorder"])
        kv, dim = rng.choice([1, 2, 3, 4, 8]), rng.choice([16, 32, 64, 64, 80, 96, 128, 128])
        heads = kv * rng.choice([1, 2, 3, 4, 4, 5, 7, 8, 8, 16])
        page, dtype = rng.choice([8, 16, 32, 64, 64, 128, 256]), rng.choice(["bf16", "bf16", "f16"])
        if op == "append":
            batch, hi = _log(rng, 1, 128), _log(rng, 1, 4096)
            case = _cache_case(None, op, batch, (_log(rng, 1, hi), hi), (0, _log(rng, 1, 2000)), heads, kv, dim, page, dtype,
                               rotary=rng.choice([dim, dim, dim // 2, 0]), interleaved=rng.random() < 0.5,
                               shift=rng.choice([0, 0, 131072, 1000000]))
        elif op == "attend":
            # tokens at a time (decoding and verification), or prompts and chunks of prompts
            few = rng.random() < 0.6
            batch = _log(rng, 1, 128 if few else 16)
            hi = rng.choice([1, 1, 1, 2, 5, 8, 16]) if few else _log(rng, 17, 8000)
            ctx = _log(rng, 16, 30000) if few else _log(rng, 1, 4000)
            lo = (hi if rng.random() < 0.7 else 1) if few else _log(rng, 1, hi)
            windowed = rng.random() < 0.4
            case = _cache_case(None, op, batch, (lo, hi), (0 if not few else _log(rng, 1, ctx), ctx), heads, kv, dim, page, dtype,
                               window=_log(rng, 16, 8192) if windowed else 0, sinks=rng.choice([0, 1, 4, 70]) if windowed else 0)
        elif op == "pages":
            hi = _log(rng, 8, 6000)
            case = _pages_case(None, _log(rng, 1, 256), rng.choice([1, 1, 2, 4, 5, 8]), rng.choice([1, 1, 2, 5, 16, 100]),
                               (_log(rng, 1, hi), hi), rng.choice([1, 2, 4]), rng.choice([16, 32, 64]), page, _log(rng, 1, 20000))
        elif op == "select":
            case = _select_case(None, _log(rng, 1, 128), rng.choice([1, 2, 3, 4, 5, 8, 16]), _log(rng, 40, 160000),
                                rng.choice(["bf16", "f16", "f32"]), rng.choice([0, 0, 2, 5, 9]))
        else:
            case = _reorder_case(None, _log(rng, 1, 64), rng.choice([2, 3, 4, 5, 8, 16]), _log(rng, 1, 3000),
                                 rng.choice([5, 32, 184, 200]), rng.choice([32, 100, 256, 1024]), rng.choice(["bf16", "f16", "f32"]))
        w = work(case)
        if any(w[k] > most[op][k] for k in w):
            continue
        if op in ("append", "attend"):
            news, ctxs = _sizes(case)
            longest = max(c + n for c, n in zip(ctxs, news))
            if len(news) * max(news) * longest * heads > 5e9 or len(news) * longest * kv * dim > 1.2e9:
                continue
        if op == "pages":
            held = sum(-(-(c + case["new"]) // page) for c in _contexts(case)) * case["beams"] + case["spare"]
            if held > 400000 or held * page * case["kv"] * case["dim"] > 1 << 30:
                continue
        return case


def _spread(lo, hi, count, step):
    """`count` numbers over their range in a mixed order."""
    return [hi - (hi - lo) * ((i * step) % 1009) // 1008 for i in range(count)]


def _sizes(case):
    """The batch's (new tokens, tokens held before them)."""
    return _spread(case["new_lo"], case["new_hi"], case["batch"], 389), _spread(case["ctx_lo"], case["ctx_hi"], case["batch"], 617)


def _contexts(case):
    return _spread(case["ctx_lo"], case["ctx_hi"], case["groups"], 617)


def work(case):
    op = case["op"]
    if op == "append":
        news, ctxs = _sizes(case)
        tokens, heads, kv, dim, page = sum(news), case["heads"], case["kv"], case["dim"], case["page"]
        blocks = sum(-(-(c + n) // page) - c // page for c, n in zip(ctxs, news))
        # each row in, keys and values out in a byte, queries in two, exponents
        return {"bytes": tokens * dim * (2 * (heads + 2 * kv) + 2 * heads + 2 * kv) + 2 * blocks * kv,
                "flops": 3 * tokens * case["rotary"] * (heads + kv) + 2 * tokens * dim * kv}
    if op == "attend":
        news, ctxs = _sizes(case)
        heads, kv, dim, tokens = case["heads"], case["kv"], case["dim"], sum(news)
        window, sinks, held, pairs = case["window"], case["sinks"], 0, 0
        for n, c in zip(news, ctxs):
            if window:
                first = max(0, c + 1 - window)  # of the keys that the first new token's window holds
                held += c + n - first + min(sinks, first)
                for p in range(c, c + n):
                    below = max(0, p + 1 - window)
                    pairs += p + 1 - below + min(sinks, below)
            else:
                held += c + n
                pairs += n * c + n * (n + 1) // 2
        return {"bytes": 4 * dim * heads * tokens + 2 * kv * dim * held, "flops": 4 * dim * heads * pairs}
    if op == "pages":
        beams, new, page, ctxs = case["beams"], case["new"], case["page"], _contexts(case)
        pages = sum(-(-(c + new) // page) for c in ctxs) * beams + case["spare"]
        # the pages' counts are read; the rows of the table that change, the new slots (and forked tails) are written
        bytes_ = 4 * pages + sum(beams * (8 * new + 4 * (-(-(c + new) // page) - c // page) + 8) for c in ctxs)
        if beams > 1:
            copied = sum(2 * (beams // 2) * (c % page) * case["kv"] * case["dim"] * 2 for c in ctxs)  # half the beams, K and V, 2 bytes
            bytes_ += 2 * copied + sum(beams * 8 * -(-c // page) for c in ctxs)
        return {"bytes": bytes_, "flops": pages}
    size = {"bf16": 2, "f16": 2, "f32": 4}[case["dtype"]]
    rows = case["groups"] * case["beams"]
    if op == "select":
        return {"bytes": rows * (case["vocab"] * size + 4 + 20), "flops": 3 * rows * case["vocab"]}
    # about half of the beams change, and are copied from one of the others
    return {"bytes": 2 * case["groups"] * (case["beams"] // 2) * case["length"] * (case["routes"] + size * case["hidden"]),
            "flops": rows}


# --------------------------------------------------------------------------------------- the inputs
def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    return {"append": _prepare_cache, "attend": _prepare_cache, "pages": _prepare_pages, "select": _prepare_select,
            "reorder": _prepare_reorder}[case["op"]](case, gen)


def _prepare_cache(case, gen):
    dtype, page, kv, dim, heads = DTYPES[case["dtype"]], case["page"], case["kv"], case["dim"], case["heads"]
    news, ctxs = _sizes(case)
    lengths = [n + c for n, c in zip(news, ctxs)]
    ragged, tokens = min(news) != max(news), sum(news)
    per = max(-(-n // page) for n in lengths)
    pages = sum(-(-n // page) for n in lengths) + 1

    def normal(*shape):
        return torch.randn(*shape, generator=gen, device="cuda", dtype=dtype)

    # pages are handed out in no order, as after hours of serving
    order = torch.randperm(pages, generator=gen, device="cuda").to(torch.int32)
    lens = torch.tensor(lengths, device="cuda", dtype=torch.int32)
    counts = (lens + page - 1) // page
    ends = torch.cumsum(counts, 0)
    column = torch.arange(per, device="cuda")
    index = (ends - counts)[:, None] + column
    table = torch.where(column < counts[:, None], order[index.clamp_max(pages - 1)], 0).to(torch.int32)
    state = {"op": case["op"], "page": page, "window": case["window"], "sinks": case["sinks"], "dim": dim, "dtype": dtype,
             "interleaved": case["interleaved"], "max_new": max(news), "max_len": max(lengths), "table": table,
             "lengths": lens, "cu": None}
    for x in "kv":
        # values of about the size of one, under exponents that differ a little from page to page
        state[x + "_exp"] = torch.randint(-7, -5, (pages, kv), generator=gen, device="cuda").to(torch.int8)
        state[x + "_pages"] = (normal(pages, kv, page, dim) * 64).to(E4M3)
    starts = torch.cumsum(torch.tensor([0] + news, device="cuda"), 0)
    if ragged:
        state["cu"] = starts.to(torch.int32)
    shape = (tokens,) if ragged else (case["batch"], news[0])
    state["q"] = normal(*shape, heads, dim)
    if case["op"] == "append":
        state["k"], state["v"] = normal(*shape, kv, dim), normal(*shape, kv, dim)
        half = case["rotary"] // 2
        state["inv_freq"] = (10000.0 ** (-torch.arange(half, device="cuda", dtype=torch.float64) / half)).float() if half else None
        state["positions"] = None
        if case["shift"]:
            n = starts[1:] - starts[:-1]
            at = torch.arange(tokens, device="cuda") - torch.repeat_interleave(starts[:-1] + n - lens, n)
            state["positions"] = (at + case["shift"]).view(shape)
    return state


def _survivors(groups, beams, gen):
    """Parents [groups, beams] of a choice that keeps about half of the beams where they are and puts copies of them in
    the places of the others."""
    lots = torch.rand(groups, beams, generator=gen, device="cuda")
    kept = lots.argsort(1)[:, :beams - beams // 2]
    pick = torch.randint(0, kept.shape[1], (groups, beams), generator=gen, device="cuda")
    parents = kept.gather(1, pick)
    return parents.scatter(1, kept, kept)


def _prepare_pages(case, gen):
    groups, beams, page, new, ctxs = case["groups"], case["beams"], case["page"], case["new"], _contexts(case)
    batch = groups * beams
    per = -(-(max(ctxs) + new) // page)
    pages = sum(-(-(c + new) // page) for c in ctxs) * beams + case["spare"]
    order = torch.randperm(pages, generator=gen, device="cuda").to(torch.int32)
    before = torch.tensor(ctxs, device="cuda").repeat_interleave(beams)
    lens = before + new if beams == 1 else before  # (without beams: the last step's drafts, all rejected, are still counted)
    # beams of a request share their pages but for the last eighth of its text
    shared = (lens * 7 // 8 // page if beams > 1 else lens * 0)[:, None]
    count = ((lens + page - 1) // page)[:, None]
    column = torch.arange(per, device="cuda")[None]
    first = torch.arange(batch, device="cuda")[:, None] % beams == 0
    taken = (column < count) & (first | (column >= shared))  # pages of the sequence's own
    number = taken.flatten().cumsum(0).view(taken.shape) - 1
    table = order[number.clamp(0, pages - 1)]
    lead = table.view(groups, beams, per)[:, :1].expand(groups, beams, per).reshape(batch, per)
    table = torch.where(column < shared, lead, table)
    table = torch.where(column < count, table, -1)
    refs = torch.bincount(table[table >= 0].flatten(), minlength=pages)
    # table, lengths and counts in one buffer: what a pass begins with
    start = torch.cat((table.flatten(), lens, refs)).to(torch.int32)
    live = start.clone()
    cells = batch * per
    state = {"op": "pages", "page": page, "new": new, "beams": beams, "start": start, "live": live,
             "table": live[:cells].view(batch, per), "lengths": live[cells:cells + batch], "refs": live[cells + batch:],
             "before": before.to(torch.int32)}
    shape = (pages, case["kv"], page, case["dim"])
    state["k_pages"] = torch.randn(shape, generator=gen, device="cuda", dtype=torch.bfloat16)
    state["v_pages"] = torch.randn(shape, generator=gen, device="cuda", dtype=torch.bfloat16)
    state["parents"] = _survivors(groups, beams, gen) if beams > 1 else None
    return state


def _prepare_select(case, gen):
    shape = (case["groups"], case["beams"])
    logits = torch.randn(*shape, case["vocab"], generator=gen, device="cuda") * 2.5
    scores = -torch.rand(shape, generator=gen, device="cuda") * 6 - 20
    done = torch.arange(shape[0] * shape[1], device="cuda").view(shape) % case["done"] == case["done"] - 1 if case["done"] else None
    return {"op": "select", "logits": logits.to(DTYPES[case["dtype"]]), "scores": scores, "done": done, "eos": 2}


def _prepare_reorder(case, gen):
    rows, length = case["groups"] * case["beams"], case["length"]
    codes = torch.randint(0, 16, (rows, length, case["routes"]), generator=gen, device="cuda", dtype=torch.uint8)
    conv = torch.randn(rows, length, case["hidden"], generator=gen, device="cuda", dtype=DTYPES[case["dtype"]])
    return {"op": "reorder", "codes": codes, "conv": conv, "parents": _survivors(case["groups"], case["beams"], gen)}


# ---------------------------------------------------------------------------------- the plain forms
def _padded(state):
    """(which token [B, n], which of them there are [B, n], its place in the sequence [B, n])."""
    lens = state["lengths"].long()
    cu = state["cu"]
    if cu is None:
        cu = torch.arange(lens.numel() + 1, device=lens.device) * state["max_new"]
    cu = cu.long()
    n = cu[1:] - cu[:-1]
    j = torch.arange(state["max_new"], device=lens.device)
    there = j < n[:, None]
    return torch.where(there, cu[:-1, None] + j, 0), there, (lens - n)[:, None] + j


def _rotate(x, cos, sin, interleaved):
    """x [N, H, D] in 32 bits, its first 2 * cos.shape[-1] values rotated in pairs."""
    half = cos.shape[-1]
    turned, rest = x[..., :2 * half], x[..., 2 * half:]
    if interleaved:
        a, b = turned[..., 0::2], turned[..., 1::2]
        both = torch.stack((a * cos - b * sin, b * cos + a * sin), -1).flatten(-2)
    else:
        a, b = turned[..., :half], turned[..., half:]
        both = torch.cat((a * cos - b * sin, b * cos + a * sin), -1)
    return torch.cat((both, rest), -1)


def _exponent(most):
    """The least exponent under which values up to `most` stay within e4m3's 448."""
    m, e = torch.frexp(most)  # most = m 2^e, m in [1/2, 1); 448 = 7/8 2^9
    e = torch.where(m > 0.875, e - 8, e - 9)
    return torch.where(most > 0, e, LEAST).clamp(LEAST, MOST)


def _power(e):
    return ((e.int() + 127) << 23).view(torch.float32)


def _round8(x, e):
    """x in 32 bits to e4m3 under exponents e."""
    return (x * _power(-e.int())).clamp(-448, 448).to(E4M3)


def _values(pages, exp):
    """What the slots of a cache stand for."""
    return (pages.float() * _power(exp)[..., None, None]).to(torch.bfloat16)


def _store(pages, exp, x, page, slot, first):
    """Rows x [N, KV, D] in 32 bits to (page, slot); `first`: the lowest slot that is written in each row's page."""
    most = torch.zeros(exp.shape, device=x.device)
    most.index_reduce_(0, page, x.abs().amax(-1), "amax")
    lowest = torch.full((exp.shape[0],), pages.shape[2], device=x.device, dtype=torch.long)
    lowest.index_reduce_(0, page, first, "amin")
    used = torch.unique(page)
    old, need = exp[used].int(), _exponent(most[used])
    kept = lowest[used] > 0  # pages that hold earlier keys
    now = torch.where(kept[:, None], torch.maximum(old, need), need)
    # the earlier slots, under the new exponent
    held = used[kept]
    again = _round8(pages[held].float() * _power(old[kept])[..., None, None], now[kept][..., None, None])
    earlier = torch.arange(pages.shape[2], device=x.device)[None] < lowest[held][:, None]
    pages[held] = torch.where(earlier[:, None, :, None], again.float(), pages[held].float()).to(E4M3)
    exp[used] = now.to(torch.int8)
    pages.view(torch.uint8)[page, :, slot] = _round8(x, exp[page][..., None]).view(torch.uint8)


def _append(state):
    token, there, place = _padded(state)
    token, place = token[there], place[there]
    row = torch.arange(there.shape[0], device=there.device)[:, None].expand(there.shape)[there]
    q, k, v = state["q"], state["k"].flatten(0, -3)[token].float(), state["v"].flatten(0, -3)[token].float()
    if state["inv_freq"] is not None:
        position = place if state["positions"] is None else state["positions"].reshape(-1)[token]
        angle = position.double()[:, None] * state["inv_freq"].double()  # a far position's angle needs 64 bits
        cos, sin = angle.cos().float()[:, None], angle.sin().float()[:, None]
        k = _rotate(k, cos, sin, state["interleaved"])
        q = _rotate(q.flatten(0, -3).float(), cos, sin, state["interleaved"]).to(q.dtype).view(q.shape)
    page, slot = state["table"][row, place // state["page"]].long(), place % state["page"]
    _store(state["k_pages"], state["k_exp"], k, page, slot, slot)
    _store(state["v_pages"], state["v_exp"], v, page, slot, slot)
    return {"k": _values(state["k_pages"], state["k_exp"]), "v": _values(state["v_pages"], state["v_exp"]), "q": q}


def _own_keys(state, x):
    """Keys or values of every sequence [B, KV, L, D] in 32 bits."""
    place = torch.arange(state["max_len"], device="cuda")
    page = state["table"][:, place // state["page"]].long()
    slot = (place % state["page"]).expand(page.shape)
    rows = state[x + "_pages"].view(torch.uint8)[page, :, slot].view(E4M3).float()
    return rows.mul_(_power(state[x + "_exp"])[page][..., None]).transpose(1, 2)


def _visible(state, place):
    """[B, n, L]: which keys of its own sequence each token sees."""
    key = torch.arange(state["max_len"], device="cuda")
    p = place[..., None]
    seen = key <= p
    if state["window"]:
        seen &= (key > p - state["window"]) | (key < state["sinks"])
    return seen


def _attend(state):
    token, there, place = _padded(state)
    k, v = _own_keys(state, "k"), _own_keys(state, "v")
    kv, d = k.shape[1], k.shape[3]
    q = state["q"].flatten(0, -3)[token].float() * state["dim"] ** -0.5
    b, n, heads, _ = q.shape
    group = heads // kv
    q = q.view(b, n, kv, group, d).transpose(1, 2).reshape(b, kv, n * group, d)
    s = q @ k.transpose(-1, -2)
    s.masked_fill_(~_visible(state, place).repeat_interleave(group, 1)[:, None], -math.inf)
    s.sub_(s.amax(-1, keepdim=True).clamp_min(-1e30)).exp_()
    out = (s @ v) / s.sum(-1, keepdim=True).clamp_min(1e-30)
    out = out.view(b, kv, n, group, d).transpose(1, 2).reshape(b, n, heads, d)[there]
    return out.to(state["q"].dtype).view(state["q"].shape)


def _truncate(state, lengths):
    table, lens, refs, page = state["table"], state["lengths"], state["refs"], state["page"]
    now = torch.minimum(lens, lengths)
    column = torch.arange(table.shape[1], device="cuda")[None]
    gone = (column >= -(-now // page)[:, None]) & (column < -(-lens // page)[:, None])
    refs.index_add_(0, table[gone].long(), torch.full_like(table[gone], -1))
    table[gone] = -1
    lens.copy_(now)


def _fork(state, parents):
    table, lens, refs, page = state["table"], state["lengths"], state["refs"], state["page"]
    beams = parents.shape[1]
    rows = (parents + torch.arange(parents.shape[0], device="cuda")[:, None] * beams).flatten()
    column = torch.arange(table.shape[1], device="cuda")[None]
    held = column < -(-lens // page)[:, None]
    change = (torch.bincount(rows, minlength=rows.numel()) - 1).to(torch.int32)[:, None].expand(table.shape)
    refs.index_add_(0, table[held].long(), change[held])
    table.copy_(torch.where(held, table, -1)[rows])
    lens.copy_(lens[rows])


def _extend(state, new):
    table, lens, refs, page = state["table"], state["lengths"], state["refs"], state["page"]
    batch, per = table.shape
    column = torch.arange(per, device="cuda")[None]
    have, want = -(-lens // page).long(), -(-(lens + new) // page).long()
    last = table.gather(1, (have - 1).clamp_min(0)[:, None])[:, 0].long()
    used = lens % page
    copied = (used > 0) & (refs[last.clamp_min(0)] > 1)  # a page that others hold too: its keys move to one of the sequence's own
    fits = want <= per
    need = torch.where(fits, want - have + copied, 0)
    ends = need.cumsum(0)
    free = (refs == 0).nonzero()[:, 0]
    ok = fits & ((need == 0) | (ends <= free.numel()))
    begin = have - copied.long()  # the first column that gets a page
    fresh = ok[:, None] & (column >= begin[:, None]) & (column < want[:, None])
    at = (ends - need - begin)[:, None] + column
    pages = free[at[fresh]]
    moved = ok & copied
    source = last[moved]
    table[fresh] = pages.to(torch.int32)
    refs[pages] = 1
    refs.index_add_(0, source, torch.full_like(source, -1, dtype=torch.int32))
    target = table.gather(1, begin.clamp_max(per - 1)[:, None])[:, 0].long()[moved]
    slots = torch.arange(page, device="cuda")[None] < used[moved][:, None]
    for x in (state["k_pages"], state["v_pages"]):
        x[target] = torch.where(slots[:, None, :, None], x[source], x[target])
    place = lens.long()[:, None] + torch.arange(new, device="cuda")
    slot = table.gather(1, (place // page).clamp_max(per - 1)).long() * page + place % page
    lens.copy_(torch.where(ok, lens + new, -1 - lens))
    return torch.where(ok[:, None], slot, -1), ok


def _pages(state):
    state["live"].copy_(state["start"])
    if state["parents"] is not None:
        _fork(state, state["parents"])
    else:
        _truncate(state, state["before"])
    slots, ok = _extend(state, state["new"])
    out = {"slots": slots, "ok": ok, "table": state["table"], "lengths": state["lengths"], "refs": state["refs"]}
    if state["parents"] is not None:
        out["k"], out["v"] = state["k_pages"], state["v_pages"]
    return out


def _select(state):
    x, scores, done = state["logits"].float(), state["scores"], state["done"]
    groups, beams, vocab = x.shape
    top = x.amax(-1, keepdim=True)
    norm = (x - top).exp().double().sum(-1, keepdim=True).log() + top.double()
    best = scores.double()[..., None] + (x.double() - norm)  # candidates a few ulp of 32 bits apart must not change places
    if done is not None:
        ended = torch.full((vocab,), -math.inf, device="cuda", dtype=torch.float64)
        ended[state["eos"]] = 0
        best = torch.where(done[..., None], scores.double()[..., None] + ended, best)
    best = best.flatten(1)
    values, index = [], []
    for _ in range(beams):
        at = best.argmax(1, keepdim=True)
        values.append(best.gather(1, at))
        index.append(at)
        best.scatter_(1, at, -math.inf)
    index = torch.cat(index, 1)
    return {"scores": torch.cat(values, 1).float(), "tokens": index % vocab, "parents": index // vocab}


def _reorder(state):
    parents = state["parents"]
    rows = (parents + torch.arange(parents.shape[0], device="cuda")[:, None] * parents.shape[1]).flatten()
    for x in (state["codes"], state["conv"]):
        x.copy_(x[rows])
    return {"codes": state["codes"], "conv": state["conv"]}


# ------------------------------------------------------------------------------------- one pass
def _handle(state):
    """The framework's handles of the state: made once, as a server makes them."""
    if "framework" not in state:
        from __graft_entry__ import load_package
        kv = state["framework"] = load_package()
        if state["op"] in ("append", "attend"):
            state["cache"] = kv.PagedKVCache8(state["k_pages"], state["v_pages"], state["k_exp"], state["v_exp"], state["table"],
                                              state["lengths"], dtype=state["dtype"])
        if state["op"] == "pages":
            cache = kv.PagedKVCache(state["k_pages"], state["v_pages"], state["table"], state["lengths"])
            state["pool"] = kv.PagePool(cache, state["refs"])
    return state["framework"]


def run(state):
    op = state["op"]
    if own:
        kv = _handle(state)
        if op == "append":
            q = kv.kv_append(state["cache"], state["k"], state["v"], state["q"], cu=state["cu"], max_new=state["max_new"],
                             positions=state["positions"], inv_freq=state["inv_freq"], interleaved=state["interleaved"])
            k, v = state["cache"].values()
            return {"k": k, "v": v, "q": q}
        if op == "attend":
            return kv.kv_attend(state["cache"], state["q"], cu=state["cu"], max_new=state["max_new"], max_len=state["max_len"],
                                window=state["window"], sinks=state["sinks"])
        if op == "pages":
            pool = state["pool"]
            state["live"].copy_(state["start"])
            if state["parents"] is not None:
                pool.reorder(state["parents"])
            else:
                pool.truncate(state["before"])
            slots, ok = pool.extend(state["new"])
            out = {"slots": slots, "ok": ok, "table": state["table"], "lengths": state["lengths"], "refs": state["refs"]}
            if state["parents"] is not None:
                out["k"], out["v"] = state["k_pages"], state["v_pages"]
            return out
        if op == "select":
            scores, tokens, parents = kv.beam_select(state["logits"], state["scores"], done=state["done"], eos=state["eos"])
            return {"scores": scores, "tokens": tokens, "parents": parents}
        kv.beam_reorder(state["parents"], state["codes"], state["conv"])
        return {"codes": state["codes"], "conv": state["conv"]}
    return {"append": _append, "attend": _attend, "pages": _pages, "select": _select, "reorder": _reorder}[op](state)


# ------------------------------------------------------------------------- the definition in 64 bits
def exact(case, seed):
    if case["op"] in ("pages", "reorder"):
        return None  # whole numbers, and values that only move
    state = prepare(case, seed)
    if case["op"] == "select":
        return _exact_select(state)
    return _exact_append(case, state) if case["op"] == "append" else _exact_attend(case, state)


def _exact_select(state):
    scores, tokens, parents = [], [], []
    for i in range(state["scores"].shape[0]):
        offers = torch.log_softmax(state["logits"][i].double(), -1)
        if state["done"] is not None:
            for beam in state["done"][i].nonzero()[:, 0].tolist():
                offers[beam] = -math.inf
                offers[beam, state["eos"]] = 0
        offers += state["scores"][i].double()[:, None]
        values, order = torch.sort(offers.flatten(), descending=True, stable=True)
        count = offers.shape[0]
        scores.append(values[:count])
        tokens.append(order[:count] % offers.shape[1])
        parents.append(torch.div(order[:count], offers.shape[1], rounding_mode="floor"))
    return {"scores": torch.stack(scores), "tokens": torch.stack(tokens), "parents": torch.stack(parents)}


def _exact_append(case, state):
    news, ctxs = _sizes(case)
    page, dim = case["page"], case["dim"]
    q, k, v = (state[x].double().flatten(0, -3).clone() for x in "qkv")
    place = torch.cat([torch.arange(c, c + n) for n, c in zip(news, ctxs)]).cuda()
    if state["inv_freq"] is not None:
        freq = state["inv_freq"].double()
        for x in (q, k):
            for i in range(freq.numel()):
                a, b = (2 * i, 2 * i + 1) if case["interleaved"] else (i, i + freq.numel())
                turn = torch.polar(torch.ones_like(place, dtype=torch.float64), (place + case["shift"]) * freq[i])
                z = torch.complex(x[..., a], x[..., b]) * turn[:, None]
                x[..., a], x[..., b] = z.real, z.imag
    # the steps of e4m3 by magnitude: 2^-9 below 2^-6, then an eighth of each power of two
    grid = torch.tensor([i / 512 for i in range(8)] + [(1 + i / 8) * 2.0 ** e for e in range(-6, 9) for i in range(8)],
                        dtype=torch.float64, device="cuda")[:-1]

    def nearest(x):
        """Each value's nearest step, the even one between two."""
        y = x.abs().clamp_max(448.0)
        hi = torch.searchsorted(grid, y.contiguous()).clamp(1, grid.numel() - 1)
        lo = hi - 1
        up, down = grid[hi] - y, y - grid[lo]
        pick = torch.where((up < down) | ((up == down) & (hi % 2 == 0)), hi, lo)
        return torch.copysign(grid[pick], x)

    done = {}
    for name, rows in (("k", k), ("v", v)):
        pages, exps = state[name + "_pages"].double(), state[name + "_exp"].double()
        out = pages * 2.0 ** exps[..., None, None]
        tables, at = state["table"].tolist(), 0
        # the pages of all sequences side by side: [page, heads, slots, dim], NaN where a slot is not among the new ones
        first, where, cells = [], [], []
        for i, (n, c) in enumerate(zip(news, ctxs)):
            for j in range(c // page, -(-(c + n) // page)):
                begin, end = max(c, j * page), min(c + n, (j + 1) * page)
                where.append(tables[i][j])
                first.append(begin - j * page)
                cells.append((at + begin - c, end - begin))
            at += n
        # (page by page would be too many steps for a long prompt)
        index = torch.full((len(where), page), -1, dtype=torch.long)
        for r, (begin, count) in enumerate(cells):
            index[r, first[r]:first[r] + count] = torch.arange(begin, begin + count)
        index = index.cuda()
        fresh = (index >= 0)[:, None, :, None]
        new = rows[index.clamp_min(0)].transpose(1, 2)
        where, first = torch.tensor(where, device="cuda"), torch.tensor(first, device="cuda")
        most = torch.where(fresh, new.abs(), 0.0).amax((-1, -2))
        need = torch.ceil(torch.log2((most / 448).clamp_min(2.0 ** LEAST))).clamp(LEAST, MOST)
        need = torch.where((need > LEAST) & (most <= 448 * 2.0 ** (need - 1)), need - 1, need)
        need = torch.where((need < MOST) & (most > 448 * 2.0 ** need), need + 1, need)
        exp = torch.where((first > 0)[:, None], torch.maximum(need, exps[where]), need)
        step = 2.0 ** exp[..., None, None]
        slots = torch.arange(page, device="cuda")
        held = (slots[None] < first[:, None])[:, None, :, None]
        rest = pages[where] * step  # behind the new ones: whatever the slots hold, under the new exponent
        out[where] = torch.where(fresh, nearest(new / step) * step, torch.where(held, nearest(out[where] / step) * step, rest))
        done[name] = out
    return {"k": done["k"], "v": done["v"], "q": q.view(state["q"].shape)}


def _exact_attend(case, state):
    news, ctxs = _sizes(case)
    page, kv, heads, dim = case["page"], case["kv"], case["heads"], case["dim"]
    group = heads // kv
    q = state["q"].double().flatten(0, -3)
    out = torch.empty_like(q)
    begin = 0
    for i, (n, c) in enumerate(zip(news, ctxs)):
        used = state["table"][i, :-(-(n + c) // page)].long()
        keys, values = ((state[x + "_pages"][used].double() * 2.0 ** state[x + "_exp"][used].double()[..., None, None])
                        .permute(1, 0, 2, 3).reshape(kv, -1, dim)[:, :n + c] for x in "kv")
        p = c + torch.arange(n, device="cuda")[:, None]
        j = torch.arange(n + c, device="cuda")[None]
        hidden = j > p
        if case["window"]:
            hidden |= (j <= p - case["window"]) & (j >= case["sinks"])
        for h in range(heads):
            s = (q[begin:begin + n, h] @ keys[h // group].T) / math.sqrt(dim)
            out[begin:begin + n, h] = torch.softmax(s.masked_fill(hidden, -math.inf), -1) @ values[h // group]
        begin += n
    return out.view(state["q"].shape)
