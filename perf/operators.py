"""The operators around a paged cache of keys and values, as they are measured.

* ``append``: a step's new keys and values go to their slots of the paged cache, keys (and the step's
  queries) rotated by their position on the way.
* ``attend``: causal attention of the newest tokens over that cache, with grouped heads, optionally
  through a sliding window beside which the first few tokens (the sinks) stay visible.
* ``prefix``: the same attention for a batch whose sequences all begin with one long prefix, whose
  keys and values are stored once.

A cache is pages ``[pages, kv heads, page size, head size]`` for keys and for values, a table
``[batch, pages per sequence]`` of page numbers and the sequences' lengths, the newest tokens counted.
"""

import math

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "f16": torch.float16}


# ---------------------------------------------------------------------------------------- the cases
def _case(name, op, batch, new, ctx, heads, kv, dim, page, dtype, window=0, sinks=0, rotary=0, interleaved=False,
          shift=0, prefix=0):
    """``new`` and ``ctx`` are (smallest, largest) over the batch: tokens of this step, and tokens that a
    sequence holds already (after the prefix, where there is one)."""
    case = {"op": op, "batch": batch, "new_lo": new[0], "new_hi": new[1], "ctx_lo": ctx[0], "ctx_hi": ctx[1],
            "heads": heads, "kv": kv, "dim": dim, "page": page, "dtype": dtype, "window": window, "sinks": sinks,
            "rotary": rotary, "interleaved": interleaved, "shift": shift, "prefix": prefix}
    return {"name": name, **case} if name else case


def listed():
    return [
        # one decode step of 64 sequences (the memory layer's heads: 16 query, 4 key, 64 wide)
        _case("append_step", "append", 64, (1, 1), (900, 2000), 16, 4, 64, 64, "bf16", rotary=64),
        # a batch of prompts as the memory layer's prefill takes them: 32 x 2048 positions
        _case("append_prompt", "append", 32, (2048, 2048), (0, 0), 16, 4, 64, 64, "bf16", rotary=64),
        # a continuous batch: prompts, chunks of prompts and single tokens, far positions, half of each head rotated
        _case("append_ragged", "append", 37, (1, 1500), (0, 2500), 28, 4, 128, 16, "f16", rotary=64, interleaved=True,
              shift=1000000),
        # one user, one token: nothing but latency
        _case("attend_one", "attend", 1, (1, 1), (4095, 4095), 16, 4, 64, 64, "bf16"),
        # a decode step of a full batch whose sequences are of all lengths
        _case("attend_step", "attend", 64, (1, 1), (500, 16000), 32, 8, 128, 64, "bf16"),
        # the same through a window with sinks, on small pages
        _case("attend_window", "attend", 24, (1, 1), (6000, 20000), 32, 8, 128, 16, "f16", window=4096, sinks=4),
        # 16 drafted tokens a sequence verified after a context of 1024
        _case("attend_verify", "attend", 64, (16, 16), (1024, 1024), 16, 4, 64, 64, "bf16"),
        # the batch of prompts of append_prompt
        _case("attend_prompt", "attend", 32, (2048, 2048), (0, 0), 16, 4, 64, 64, "bf16"),
        # two long prompts of unlike lengths, 7 query heads a key head, a window and sinks
        _case("attend_long", "attend", 2, (5001, 8000), (0, 999), 28, 4, 128, 16, "f16", window=4096, sinks=4),
        # a few continuations of one short text
        _case("prefix_few", "prefix", 5, (3, 3), (0, 87), 16, 4, 64, 16, "f16", prefix=1000),
        # a decode step of 64 conversations under one system prompt
        _case("prefix_step", "prefix", 64, (1, 1), (20, 600), 32, 8, 128, 64, "bf16", prefix=8192),
        # many short answers about one long document
        _case("prefix_many", "prefix", 256, (1, 1), (64, 1500), 64, 8, 128, 64, "bf16", prefix=32768),
    ]


def _log(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    most = {}
    for case in listed():
        w = work(case)
        most[case["op"]] = {k: max(v, most.get(case["op"], {}).get(k, 0)) for k, v in w.items()}
    while True:
        op = rng.choice(["append", "attend", "attend", "prefix"])
        kv, dim = rng.choice([1, 2, 3, 4, 8]), rng.choice([32, 64, 64, 80, 96, 128, 128])
        heads = kv * rng.choice([1, 2, 3, 4, 4, 5, 7, 8, 8, 16])
        page, dtype = rng.choice([16, 32, 64, 128]), rng.choice(["bf16", "bf16", "f16"])
        if op == "append":
            batch, hi = _log(rng, 1, 128), _log(rng, 1, 4096)
            rotary = rng.choice([dim, dim, dim // 2])
            case = _case(None, op, batch, (_log(rng, 1, hi), hi), (0, _log(rng, 1, 4000)), heads, kv, dim, page, dtype,
                         rotary=rotary, interleaved=rng.random() < 0.5, shift=rng.choice([0, 0, 131072, 1000000]))
        elif op == "attend" and rng.random() < 0.6:
            # tokens at a time: decoding and verification
            batch, ctx, hi = _log(rng, 1, 128), _log(rng, 16, 30000), rng.choice([1, 1, 1, 2, 5, 8, 16])
            windowed = rng.random() < 0.4
            case = _case(None, op, batch, (hi if rng.random() < 0.7 else 1, hi), (_log(rng, 1, ctx), ctx), heads, kv, dim, page, dtype,
                         window=_log(rng, 16, 8192) if windowed else 0, sinks=rng.choice([0, 1, 4, 70]) if windowed else 0)
        elif op == "attend":
            # prompts and chunks of prompts
            batch, hi = _log(rng, 1, 16), _log(rng, 33, 8000)
            windowed = rng.random() < 0.4
            case = _case(None, op, batch, (_log(rng, 1, hi), hi), (0, _log(rng, 1, 4000)), heads, kv, dim, page, dtype,
                         window=_log(rng, 16, 8192) if windowed else 0, sinks=rng.choice([0, 1, 4, 70]) if windowed else 0)
        else:
            batch, hi = _log(rng, 2, 256), rng.choice([1, 1, 1, 2, 4, 9])
            case = _case(None, op, batch, (hi, hi), (0, _log(rng, 1, 1500)), heads, kv, dim, page, dtype,
                         prefix=_log(rng, 100, 32768))
        w = work(case)
        news, ctxs = _sizes(case)
        padded = len(news) * max(news) * (max(c + n for c, n in zip(ctxs, news)) + (case["prefix"])) * heads
        held = len(news) * max(c + n for c, n in zip(ctxs, news)) * kv * dim
        if all(w[k] <= most[op][k] for k in w) and padded <= 5e9 and held <= 1.2e9:
            return case


def _sizes(case):
    """The batch's (new tokens, tokens held before them), spread over their ranges in a mixed order."""
    def spread(lo, hi, step):
        return [hi - (hi - lo) * ((i * step) % 1009) // 1008 for i in range(case["batch"])]
    return spread(case["new_lo"], case["new_hi"], 389), spread(case["ctx_lo"], case["ctx_hi"], 617)


def work(case):
    news, ctxs = _sizes(case)
    heads, kv, dim, size = case["heads"], case["kv"], case["dim"], 2
    tokens = sum(news)
    if case["op"] == "append":
        return {"bytes": 2 * size * tokens * dim * (heads + 2 * kv), "flops": 3 * tokens * case["rotary"] * (heads + kv)}
    window, sinks, held, pairs = case["window"], case["sinks"], case["prefix"], case["prefix"] * tokens
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
    return {"bytes": size * dim * (2 * heads * tokens + 2 * kv * held), "flops": 4 * dim * heads * pairs}


# --------------------------------------------------------------------------------------- the inputs
def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    dtype, page, kv, dim, heads = DTYPES[case["dtype"]], case["page"], case["kv"], case["dim"], case["heads"]
    news, ctxs = _sizes(case)
    lengths = [n + c for n, c in zip(news, ctxs)]
    ragged, tokens = min(news) != max(news), sum(news)
    per = max(-(-n // page) for n in lengths)
    shared = -(-case["prefix"] // page)
    pages = shared + sum(-(-n // page) for n in lengths) + 1

    def normal(*shape):
        return torch.randn(*shape, generator=gen, device="cuda", dtype=dtype)

    # pages are handed out in no order, as after hours of serving
    order = torch.randperm(pages, generator=gen, device="cuda").to(torch.int32)
    lens = torch.tensor(lengths, device="cuda", dtype=torch.int32)
    counts = (lens + page - 1) // page
    ends = torch.cumsum(counts, 0)
    column = torch.arange(per, device="cuda")
    index = (shared + ends - counts)[:, None] + column
    table = torch.where(column < counts[:, None], order[index.clamp_max(pages - 1)], 0).to(torch.int32)
    state = {"op": case["op"], "page": page, "window": case["window"], "sinks": case["sinks"], "dim": dim,
             "prefix": case["prefix"], "interleaved": case["interleaved"], "max_new": max(news), "max_len": max(lengths),
             "k_pages": normal(pages, kv, page, dim), "v_pages": normal(pages, kv, page, dim), "table": table,
             "lengths": lens, "prefix_table": order[:shared].contiguous(), "cu": None}
    starts = torch.cumsum(torch.tensor([0] + news, device="cuda"), 0)
    if ragged:
        state["cu"] = starts.to(torch.int32)
    shape = (tokens,) if ragged else (case["batch"], news[0])
    state["q"] = normal(*shape, heads, dim)
    if case["op"] == "append":
        state["k"], state["v"] = normal(*shape, kv, dim), normal(*shape, kv, dim)
        half = case["rotary"] // 2
        state["inv_freq"] = (10000.0 ** (-torch.arange(half, device="cuda", dtype=torch.float64) / half)).float()
        state["positions"] = None
        if case["shift"]:
            n = starts[1:] - starts[:-1]
            at = torch.arange(tokens, device="cuda") - torch.repeat_interleave(starts[:-1] + n - lens, n)
            state["positions"] = (at + case["shift"]).view(shape)
    return state


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


def _append(state):
    token, there, place = _padded(state)
    token, place = token[there], place[there]
    row = torch.arange(there.shape[0], device=there.device)[:, None].expand(there.shape)[there]
    position = place if state["positions"] is None else state["positions"].reshape(-1)[token]
    angle = position.double()[:, None] * state["inv_freq"].double()  # a far position's angle needs 64 bits
    cos, sin = angle.cos().float()[:, None], angle.sin().float()[:, None]
    q, k, v = state["q"], state["k"].flatten(0, -3)[token], state["v"].flatten(0, -3)[token]
    page, slot = state["table"][row, place // state["page"]].long(), place % state["page"]
    state["k_pages"][page, :, slot] = _rotate(k.float(), cos, sin, state["interleaved"]).to(k.dtype)
    state["v_pages"][page, :, slot] = v
    turned = _rotate(q.flatten(0, -3).float(), cos, sin, state["interleaved"]).to(q.dtype).view(q.shape)
    return {"k_pages": state["k_pages"], "v_pages": state["v_pages"], "q": turned}


def _own_keys(state):
    """Keys and values of every sequence [B, KV, L, D] in 32 bits."""
    place = torch.arange(state["max_len"], device="cuda")
    page = state["table"][:, place // state["page"]].long()
    slot = (place % state["page"]).expand(page.shape)
    return (state["k_pages"][page, :, slot].transpose(1, 2).float(), state["v_pages"][page, :, slot].transpose(1, 2).float())


def _queries(state, token, kv):
    """[B, KV, n * G, D] in 32 bits, scaled."""
    q = state["q"].flatten(0, -3)[token].float() * state["dim"] ** -0.5
    b, n, heads, d = q.shape
    return q.view(b, n, kv, heads // kv, d).transpose(1, 2).reshape(b, kv, n * (heads // kv), d)


def _visible(state, place):
    """[B, n, L]: which keys of its own sequence each token sees."""
    key = torch.arange(state["max_len"], device="cuda")
    p = place[..., None]
    seen = key <= p
    if state["window"]:
        seen &= (key > p - state["window"]) | (key < state["sinks"])
    return seen


def _back(state, out, there):
    """[B, KV, n * G, D] as the queries lie, the tokens that are not there left out."""
    b, kv, rows, d = out.shape
    n = there.shape[1]
    out = out.view(b, kv, n, rows // n, d).transpose(1, 2).reshape(b, n, -1, d)[there]
    return out.to(state["q"].dtype).view(state["q"].shape)


def _attend(state):
    token, there, place = _padded(state)
    k, v = _own_keys(state)
    q = _queries(state, token, k.shape[1])
    group = q.shape[2] // token.shape[1]
    s = q @ k.transpose(-1, -2)
    seen = _visible(state, place).repeat_interleave(group, 1)[:, None]
    s.masked_fill_(~seen, -math.inf)
    top = s.amax(-1, keepdim=True).clamp_min(-1e30)
    s.sub_(top).exp_()
    out = (s @ v) / s.sum(-1, keepdim=True).clamp_min(1e-30)
    return _back(state, out, there)


def _prefix(state):
    token, there, place = _padded(state)
    k, v = _own_keys(state)
    b, kv, _, d = k.shape
    q = _queries(state, token, kv)
    group = q.shape[2] // token.shape[1]
    at = torch.arange(state["prefix"], device="cuda")
    page, slot = state["prefix_table"][at // state["page"]].long(), at % state["page"]
    pk, pv = state["k_pages"][page, :, slot].transpose(0, 1).float(), state["v_pages"][page, :, slot].transpose(0, 1).float()
    flat = q.transpose(0, 1).reshape(kv, -1, d)  # all rows of the batch against the one prefix
    ps = (flat @ pk.transpose(-1, -2)).view(kv, b, -1, at.numel())
    s = q @ k.transpose(-1, -2)
    seen = _visible(state, place).repeat_interleave(group, 1)[:, None]
    s.masked_fill_(~seen, -math.inf)
    top = torch.maximum(ps.amax(-1, keepdim=True).transpose(0, 1), s.amax(-1, keepdim=True))
    s.sub_(top).exp_()
    ps.sub_(top.transpose(0, 1)).exp_()
    total = s.sum(-1, keepdim=True) + ps.sum(-1, keepdim=True).transpose(0, 1)
    both = s @ v + (ps.view(kv, -1, at.numel()) @ pv).view(kv, b, -1, d).transpose(0, 1)
    return _back(state, both / total, there)


# ------------------------------------------------------------------------------------- one pass
def _cache(state):
    """The framework's handle of the state's cache: made once, as a server makes it."""
    if "cache" not in state:
        from __graft_entry__ import load_package
        state["kv"] = load_package()
        state["cache"] = state["kv"].PagedKVCache(state["k_pages"], state["v_pages"], state["table"], state["lengths"])
    return state["kv"], state["cache"]


def run(state):
    if own:
        kv, cache = _cache(state)
        if state["op"] == "append":
            q = kv.kv_append(cache, state["k"], state["v"], state["q"], cu=state["cu"], max_new=state["max_new"],
                             positions=state["positions"], inv_freq=state["inv_freq"], interleaved=state["interleaved"])
            return {"k_pages": state["k_pages"], "v_pages": state["v_pages"], "q": q}
        if state["op"] == "attend":
            return kv.kv_attend(cache, state["q"], cu=state["cu"], max_new=state["max_new"], max_len=state["max_len"],
                                window=state["window"], sinks=state["sinks"])
        return kv.kv_prefix_attend(cache, state["q"], state["prefix_table"], state["prefix"], cu=state["cu"],
                                   max_new=state["max_new"], max_len=state["max_len"])
    return {"append": _append, "attend": _attend, "prefix": _prefix}[state["op"]](state)


# ------------------------------------------------------------------------- the definition in 64 bits
def exact(case, seed):
    state = prepare(case, seed)
    news, ctxs = _sizes(case)
    page, kv, heads, dim = case["page"], case["kv"], case["heads"], case["dim"]
    group = heads // kv
    begin = [sum(news[:i]) for i in range(len(news))]
    if case["op"] == "append":
        k_pages, v_pages = state["k_pages"].double(), state["v_pages"].double()
        q, k, v = (state[x].double().flatten(0, -3).clone() for x in "qkv")
        place = torch.cat([torch.arange(c, c + n) for n, c in zip(news, ctxs)]).cuda()
        freq = state["inv_freq"].double()
        for x in (q, k):
            for i in range(freq.numel()):
                a, b = (2 * i, 2 * i + 1) if case["interleaved"] else (i, i + freq.numel())
                turn = torch.polar(torch.ones_like(place, dtype=torch.float64), (place + case["shift"]) * freq[i])
                z = torch.complex(x[..., a], x[..., b]) * turn[:, None]
                x[..., a], x[..., b] = z.real, z.imag
        for i, (n, c) in enumerate(zip(news, ctxs)):
            at = torch.arange(c, c + n, device="cuda")
            where = state["table"][i].long()[torch.div(at, page, rounding_mode="floor")]
            for pages, x in ((k_pages, k), (v_pages, v)):
                pages.permute(0, 2, 1, 3)[where, at % page] = x[begin[i]:begin[i] + n]
        return {"k_pages": k_pages, "v_pages": v_pages, "q": q.view(state["q"].shape)}
    q = state["q"].double().flatten(0, -3)
    out = torch.empty_like(q)

    def lay(pages, rows, count):
        return pages[rows.long()].permute(1, 0, 2, 3).reshape(kv, -1, dim)[:, :count].double()

    shared = [lay(state[x], state["prefix_table"], case["prefix"]) for x in ("k_pages", "v_pages")]
    for i, (n, c) in enumerate(zip(news, ctxs)):
        used = state["table"][i, :-(-(n + c) // page)]
        keys = torch.cat((shared[0], lay(state["k_pages"], used, n + c)), 1)
        values = torch.cat((shared[1], lay(state["v_pages"], used, n + c)), 1)
        p = case["prefix"] + c + torch.arange(n, device="cuda")[:, None]
        j = torch.arange(keys.shape[1], device="cuda")[None]
        hidden = j > p
        if case["window"]:
            hidden |= (j <= p - case["window"]) & (j >= case["sinks"])
        for h in range(heads):
            s = (q[begin[i]:begin[i] + n, h] @ keys[h // group].T) / math.sqrt(dim)
            out[begin[i]:begin[i] + n, h] = torch.softmax(s.masked_fill(hidden, -math.inf), -1) @ values[h // group]
    return out.view(state["q"].shape)
