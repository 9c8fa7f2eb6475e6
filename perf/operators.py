"""Performance cases of the paged key/value cache and the attention that reads it.

Every case is a plain dict; `op` says which entry point of
flashgann_amd.attention a pass goes through:

  plan       cache_plan: block tables and slot maps from request lengths
  append     cache_append: new keys and values into their slots
  attend     attend: a chunk of new tokens over the paged cache (one token a
             request is a chunk of one), with or without a sliding window and
             first tokens that stay visible
  retrieved  attend_retrieved: one token a request over the first tokens, the
             last ones and the ids that a search by inner product returned

`own` picks between those entry points and the plain form of each: elementary
torch operations in 32 bits on padded batches, rounded once at the end.
A request's lengths come from the case alone; the seed draws the values, the
pages and so the ids.
"""
from __future__ import annotations

import math
import random

import torch

DEV = "cuda"
own = False
TYPES = {"bf16": torch.bfloat16, "fp16": torch.float16}


# ------------------------------------------------------------------ the cases

def _plan(requests, new, cached, page):
    return dict(op="plan", requests=requests, new_lo=new[0], new_hi=new[1], cached_lo=cached[0], cached_hi=cached[1],
                page=page)


def _append(tokens, padding, heads_kv, dim, page, dtype, layout):
    return dict(op="append", tokens=tokens, padding=padding, heads_kv=heads_kv, dim=dim, page=page, dtype=dtype,
                layout=layout)


def _attend(requests, new, cached, heads, heads_kv, dim, page, dtype, layout, window=0, sinks=0):
    return dict(op="attend", requests=requests, new_lo=new[0], new_hi=new[1], cached_lo=cached[0], cached_hi=cached[1],
                heads=heads, heads_kv=heads_kv, dim=dim, page=page, dtype=dtype, layout=layout, window=window,
                sinks=sinks)


def _retrieved(requests, cached, heads, heads_kv, lists, ids, dim, page, dtype, layout, window, sinks):
    return dict(op="retrieved", requests=requests, new_lo=1, new_hi=1, cached_lo=cached[0], cached_hi=cached[1],
                heads=heads, heads_kv=heads_kv, lists=lists, ids=ids, dim=dim, page=page, dtype=dtype, layout=layout,
                window=window, sinks=sinks)


def listed():
    named = {
        # a decode step's bookkeeping: one new token for each of 48 running requests
        "plan_decode": _plan(48, (1, 1), (1, 4000), 16),
        # a large admission step: 700 requests of ragged length, about 105k tokens
        "plan_prefill": _plan(700, (1, 300), (0, 900), 64),
        # the keys and values of one decode step
        "append_decode": _append(64, 0, 8, 128, 16, "bf16", "nhd"),
        # those of a large prefill step, a padded batch, pages laid out head by head
        "append_chunk": _append(30000, 700, 8, 128, 64, "fp16", "hnd"),
        # the smallest attention call: a few short conversations, one token each
        "decode_small": _attend(4, (1, 1), (200, 1500), 32, 8, 128, 16, "bf16", "nhd"),
        # a serving batch of single tokens, contexts of very different length
        "decode_batch": _attend(64, (1, 1), (500, 16000), 32, 8, 128, 16, "bf16", "nhd"),
        # one user with one very long document
        "decode_long": _attend(1, (1, 1), (131070, 131070), 16, 2, 128, 64, "fp16", "hnd"),
        # a chunk of a long prompt, half of it cached: the largest call
        "chunk_8k": _attend(1, (8192, 8192), (8192, 8192), 32, 8, 128, 64, "bf16", "nhd"),
        # chunks and single tokens in one batch; no size is a power of two
        "chunk_mixed": _attend(24, (1, 400), (0, 4000), 12, 4, 96, 24, "fp16", "nhd"),
        # a long prompt through a layer with a sliding window and four first tokens
        "chunk_window": _attend(1, (12000, 12000), (4001, 4001), 16, 8, 64, 32, "bf16", "hnd", window=1000, sinks=4),
        # one token over what a search for each query head found in 100k keys
        "retrieved_one": _retrieved(1, (100000, 100000), 32, 8, 32, 100, 128, 16, "bf16", "nhd", 64, 4),
        # a batch of them, one search for each group of heads, K 256
        "retrieved_batch": _retrieved(32, (4000, 24000), 32, 8, 8, 256, 128, 32, "fp16", "nhd", 512, 16),
    }
    return [dict(name=n, **c) for n, c in named.items()]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choices(("plan", "append", "attend", "retrieved"), (12, 12, 52, 24))[0]
    page = rng.choice((16, 16, 32, 64, 128, 8, 24, 1))
    if op == "plan":
        requests = _log_int(rng, 1, 2000)
        new = _log_int(rng, 1, max(1, min(8192, 200_000 // requests)))
        return _plan(requests, rng.choice(((1, 1), (0, new), (new, new))), (0, _log_int(rng, 1, 20_000)), page)
    heads_kv, group = rng.choice(((8, 4), (8, 8), (2, 8), (4, 3), (4, 7), (1, 16), (12, 1), (8, 2), (16, 1)))
    dim = rng.choice((64, 96, 128, 128, 128, 256))
    dtype, layout = rng.choice(("bf16", "bf16", "fp16")), rng.choice(("nhd", "nhd", "hnd"))
    if op == "append":
        tokens = _log_int(rng, 1, 30_000)
        return _append(tokens, rng.choice((0, 0, tokens // 3)), heads_kv, dim, page, dtype, layout)
    heads = heads_kv * group
    window = _log_int(rng, 1, 4096)
    sinks = rng.choice((0, 1, 4, 4, 16, 100))
    if op == "retrieved":
        # at most the tokens of a large batch; the ids no more than a beam holds
        requests = _log_int(rng, 1, 64)
        cached = _log_int(rng, 300, max(301, min(120_000, 600_000 // requests)))
        ids = _log_int(rng, 1, 500)
        return _retrieved(requests, (cached // 2, cached), heads, heads_kv, rng.choice((heads, heads_kv)), ids, dim,
                          page, dtype, layout, rng.choice((0, 1, 64, min(window, 1024))), sinks)
    window, sinks = (window, sinks) if rng.random() < 0.4 else (0, 0)
    if rng.random() < 0.45:  # one token each, or the few of a draft that is being checked
        requests = _log_int(rng, 1, 128)
        cached = _log_int(rng, 1, max(2, min(130_000, int(1.2e9 / (requests * heads_kv * dim)))))
        new = rng.choice((1, 1, 1, 3, 5))
        return _attend(requests, (new, new), (rng.choice((0, cached // 4, cached)), cached), heads, heads_kv, dim, page,
                       dtype, layout, window, sinks)
    # chunks: the padded scores stay below those of the largest listed case
    most = 2e9
    cached = rng.choice((0, _log_int(rng, 16, 20_000)))
    new = _log_int(rng, 2, 8192)
    while new * (new + cached) * heads > most:
        new, cached = max(2, int(new * 0.8)), int(cached * 0.8)
    requests = max(1, min(_log_int(rng, 1, 32), int(most / (new * (new + cached) * heads))))
    return _attend(requests, (rng.choice((0, 1, new)), new), (cached // 3, cached), heads, heads_kv, dim, page, dtype,
                   layout, window, sinks)


# ------------------------------------------------------------------ inputs

def _lengths(c):
    """(new tokens, cached tokens) of each request, the same for every seed."""
    rng = random.Random("lengths %s" % sorted((k, v) for k, v in c.items() if k not in ("name", "dtype", "layout")))
    new = [rng.randint(c["new_lo"], c["new_hi"]) for _ in range(c["requests"])]
    new[0] = max(new[0], 1, c["new_hi"] if c["requests"] == 1 else 0)
    cached = [rng.randint(c["cached_lo"], c["cached_hi"]) for _ in range(c["requests"])]
    return new, cached


def _ints(v):
    return torch.tensor(v, dtype=torch.int32, device=DEV)


def _cache(c, pages, g):
    """A cache of (pages, page, heads_kv, dim), whatever the order in memory.  Page 0 is never handed out."""
    shape = (pages, c["heads_kv"], c["page"], c["dim"]) if c["layout"] == "hnd" else (pages, c["page"], c["heads_kv"], c["dim"])
    out = torch.randn(shape, generator=g, device=DEV, dtype=TYPES[c["dtype"]])
    return out.permute(0, 2, 1, 3) if c["layout"] == "hnd" else out


def prepare(case, seed):
    c = case
    g = torch.Generator(device=DEV)
    g.manual_seed(seed)
    s = dict(case=c, op=c["op"])
    page = c["page"]
    if c["op"] == "append":
        T, pages = c["tokens"], -(-2 * c["tokens"] // page) + 2
        s["k"] = torch.randn((T, c["heads_kv"], c["dim"]), generator=g, device=DEV, dtype=TYPES[c["dtype"]])
        s["v"] = torch.randn((T, c["heads_kv"], c["dim"]), generator=g, device=DEV, dtype=TYPES[c["dtype"]])
        s["k_cache"], s["v_cache"] = _cache(c, pages, g), _cache(c, pages, g)
        # requests write runs of tokens into pages that lie anywhere: whole pages, in random order
        order = torch.randperm(pages - 1, generator=g, device=DEV) + 1
        t = torch.arange(T, device=DEV)
        s["slots"] = order[t // page] * page + t % page
        if c["padding"]:
            s["slots"][T - c["padding"]:] = -1
        return s
    new, cached = _lengths(c)
    total = [n + m for n, m in zip(new, cached)]
    width = max(1, max(-(-t // page) for t in total)) + 2
    b = torch.arange(width, device=DEV)
    s["lens"], s["new"], s["kv_lens"] = _ints(cached), _ints(new), _ints(total)
    s["q_starts"] = _ints([sum(new[:r]) for r in range(len(new) + 1)])
    s["tokens"], s["max_new"], s["max_kv"] = sum(new), max(new), max(total)
    need = -(-(s["lens"] if c["op"] == "plan" else s["kv_lens"]) // page)  # pages that each request holds
    pages = sum(-(-t // page) for t in total) + 3
    order = torch.randperm(pages - 1, generator=g, device=DEV).to(torch.int32) + 1
    first = torch.cumsum(need, 0) - need
    held = b < need[:, None]
    s["table"] = torch.where(held, order[(first[:, None] + b).clamp(max=pages - 2)], -1).to(torch.int32)
    if c["op"] == "plan":
        s["free"] = order[sum(-(-m // page) for m in cached):].contiguous()
        return s
    s["k_cache"], s["v_cache"] = _cache(c, pages, g), _cache(c, pages, g)
    # a few channels of the keys lie off zero, as trained keys' do
    s["k_cache"].add_(torch.randn((c["heads_kv"], c["dim"]), generator=g, device=DEV).mul_(0.5).to(s["k_cache"].dtype))
    s["q"] = (torch.randn((s["tokens"], c["heads"], c["dim"]), generator=g, device=DEV) * 1.5).to(TYPES[c["dtype"]])
    s["scale"] = c["dim"] ** -0.5
    if c["op"] == "retrieved":
        s["ids"] = _found(s, c)
    return s


def _found(s, c):
    """What an exact search by inner product returns for each list: best first.  A search whose beam is
    shorter than K repeats its last id: so do the odd lists here."""
    k = _rows(s["k_cache"], s["table"], s["max_kv"], c["page"])
    B, L, n, K = c["requests"], c["lists"], s["max_kv"], c["ids"]
    q = s["q"].float().view(B, L, c["heads"] // L, c["dim"]).mean(2)
    score = torch.matmul(q.view(B, c["heads_kv"], L // c["heads_kv"], c["dim"]), k.permute(0, 2, 3, 1).contiguous())
    score.masked_fill_((torch.arange(n, device=DEV) >= s["kv_lens"][:, None])[:, None, None], -math.inf)
    ids = score.view(B, L, n).topk(min(K, n), -1).indices.to(torch.int32)
    ids = torch.cat([ids, ids[..., -1:].expand(B, L, K - ids.shape[-1])], -1).contiguous()
    beam = max(1, (3 * K) // 4)
    ids[:, 1::2, beam:] = ids[:, 1::2, beam - 1:beam]
    return ids


# ------------------------------------------------------------------ plain forms

def _rows(cache, table, n, page):
    """Tokens 0 .. n-1 of each request in 32 bits: (requests, n, heads_kv, dim)."""
    t = torch.arange(n, device=DEV)
    return cache[table[:, t // page].clamp(min=0).long(), t % page].float()


def _softmax_times(scores, v):
    """(softmax(scores) v, log of the sum of exponentials); a row of -inf alone gives 0 and -inf."""
    m = scores.amax(-1, keepdim=True)
    p = torch.exp(scores - torch.where(m == -math.inf, 0.0, m))
    l = p.sum(-1, keepdim=True)
    return torch.matmul(p, v) / torch.where(l > 0, l, 1.0), (m + torch.log(l)).squeeze(-1)


def _plan_plain(s):
    page, table, T = s["case"]["page"], s["table"], s["tokens"]
    lens, new, free = s["lens"].long(), s["new"].long(), s["free"]
    starts = torch.cumsum(new, 0) - new
    old, end = -(-lens // page), -(-(lens + new) // page)
    base = torch.cumsum(end - old, 0) - (end - old)
    b = torch.arange(table.shape[1], device=DEV)
    take = base[:, None] + b - old[:, None]
    fresh = torch.where(take < free.shape[0], free[take.clamp(0, free.shape[0] - 1)], -1)
    out = torch.where((b >= old[:, None]) & (b < end[:, None]), fresh, table)
    i = torch.arange(T, device=DEV)
    r = torch.searchsorted(starts + new, i, right=True)
    pos = lens[r] + i - starts[r]
    at = out[r, pos // page].long()
    slots = torch.where(at >= 0, at * page + pos % page, -1)
    q_starts = torch.cat([starts, (starts + new)[-1:]]).to(torch.int32)
    return {"table": out.to(torch.int32), "q_starts": q_starts, "kv_lens": (lens + new).to(torch.int32), "slots": slots,
            "positions": pos.to(torch.int32), "used": (end - old).sum().to(torch.int32).view(1)}


def _append_plain(s):
    page, slots = s["case"]["page"], s["slots"]
    at = slots.clamp(min=0)
    real = (slots >= 0)[:, None, None]
    for cache, rows in ((s["k_cache"], s["k"]), (s["v_cache"], s["v"])):
        cache[at // page, at % page] = torch.where(real, rows, cache[0, 0])
    return {"k_cache": s["k_cache"], "v_cache": s["v_cache"]}


def _attend_plain(s):
    c = s["case"]
    B, Q, L, H, D = c["requests"], s["max_new"], s["max_kv"], c["heads_kv"], c["dim"]
    G = c["heads"] // H
    i = torch.arange(Q, device=DEV)
    rows = (s["q_starts"][:-1, None] + i).clamp(max=s["tokens"] - 1).long()
    q = s["q"].float()[rows].view(B, Q, H, G, D).permute(0, 2, 3, 1, 4).reshape(B, H, G * Q, D)
    k = _rows(s["k_cache"], s["table"], L, c["page"]).permute(0, 2, 3, 1).contiguous()
    v = _rows(s["v_cache"], s["table"], L, c["page"]).permute(0, 2, 1, 3).contiguous()
    j = torch.arange(L, device=DEV)
    pos = (s["kv_lens"] - s["new"])[:, None, None] + i[:, None]
    seen = j <= pos
    if c["window"]:
        seen &= (j > pos - c["window"]) | (j < c["sinks"])
    scores = torch.matmul(q, k).mul_(s["scale"]).view(B, H, G, Q, L)
    scores.masked_fill_(~seen[:, None, None], -math.inf)
    out, lse = _softmax_times(scores.view(B, H, G * Q, L), v)
    t = torch.arange(s["tokens"], device=DEV)
    r = torch.searchsorted(s["q_starts"][1:].long(), t, right=True)
    at = t - s["q_starts"].long()[r]
    out = out.view(B, H, G, Q, D)[r, :, :, at].reshape(-1, c["heads"], D)
    return {"out": out.to(s["q"].dtype), "lse": lse.view(B, H, G, Q)[r, :, :, at].reshape(-1, c["heads"])}


def _retrieved_plain(s):
    c = s["case"]
    B, L, D, page = c["requests"], c["lists"], c["dim"], c["page"]
    kv, sinks, window = s["kv_lens"].long(), c["sinks"], c["window"]
    first = torch.arange(sinks, device=DEV).expand(B, L, sinks)
    last = (kv[:, None] - window + torch.arange(window, device=DEV))[:, None].expand(B, L, window)
    ids = s["ids"].long()
    repeat = torch.zeros_like(ids, dtype=torch.bool)
    repeat[..., 1:] = ids[..., 1:] == ids[..., :-1]
    end = kv[:, None, None]
    seen = torch.cat([first < end, last >= sinks, (ids >= sinks) & (ids < end - window) & ~repeat], -1)
    j = torch.where(seen, torch.cat([first, last, ids], -1), 0)
    at = torch.gather(s["table"].long()[:, None].expand(B, L, -1), 2, j // page).clamp(min=0)
    head = (torch.arange(L, device=DEV) // (L // c["heads_kv"]))[:, None]
    k, v = s["k_cache"][at, j % page, head].float(), s["v_cache"][at, j % page, head].float()
    q = s["q"].float().view(B, L, c["heads"] // L, D)
    scores = torch.matmul(q, k.transpose(2, 3).contiguous()).mul_(s["scale"])
    out, lse = _softmax_times(scores.masked_fill_(~seen[:, :, None], -math.inf), v)
    return {"out": out.reshape(B, c["heads"], D).to(s["q"].dtype), "lse": lse.reshape(B, c["heads"])}


PLAIN = {"plan": _plan_plain, "append": _append_plain, "attend": _attend_plain, "retrieved": _retrieved_plain}


# ------------------------------------------------------------------ a pass

def run(state):
    s = state
    if not own:
        return PLAIN[s["op"]](s)
    from flashgann_amd import attention
    c = s["case"]
    if c["op"] == "plan":
        p = attention.cache_plan(s["lens"], s["new"], s["table"], s["free"], page_size=c["page"], max_tokens=s["tokens"])
        return {"table": s["table"], "q_starts": p.q_starts, "kv_lens": p.kv_lens, "slots": p.slots,
                "positions": p.positions, "used": p.used}
    if c["op"] == "append":
        attention.cache_append(s["k"], s["v"], s["k_cache"], s["v_cache"], s["slots"])
        return {"k_cache": s["k_cache"], "v_cache": s["v_cache"]}
    if c["op"] == "attend":
        out, lse = attention.attend(s["q"], s["k_cache"], s["v_cache"], s["table"], s["q_starts"], s["kv_lens"],
                                    max_q=s["max_new"], scale=s["scale"], window=c["window"] or None, sinks=c["sinks"])
    else:
        out, lse = attention.attend_retrieved(s["q"], s["k_cache"], s["v_cache"], s["table"], s["kv_lens"], s["ids"],
                                              scale=s["scale"], window=c["window"], sinks=c["sinks"])
    return {"out": out, "lse": lse}


# ------------------------------------------------------------------ what a pass cannot do without

def _pairs(n, m, window, sinks):
    """(visible pairs, visible keys) of n new tokens after m cached ones."""
    if not window:
        return n * m + n * (n + 1) // 2, n + m
    pairs = 0
    for p in range(m, m + n):
        low = max(0, p - window + 1)
        pairs += p + 1 - low + min(sinks, low)
    low = max(0, m - window + 1)
    return pairs, n + m - low + min(sinks, low) if n else 0


def work(case):
    c = case
    if c["op"] == "append":
        real = c["tokens"] - c["padding"]
        return {"bytes": 8 * real * c["heads_kv"] * c["dim"] + 8 * c["tokens"], "flops": 0}
    new, cached = _lengths(c)
    if c["op"] == "plan":
        page, B = c["page"], c["requests"]
        fresh = sum(-(-(n + m) // page) + -m // page for n, m in zip(new, cached))
        return {"bytes": 4 * (2 * B + fresh) + 4 * (2 * B + 2 + fresh) + 12 * sum(new), "flops": 0}
    D, H, T = c["dim"], c["heads"], sum(new)
    if c["op"] == "attend":
        seen = [_pairs(n, m, c["window"], c["sinks"]) for n, m in zip(new, cached)]
        pairs, keys = H * sum(p for p, _ in seen), c["heads_kv"] * sum(k for _, k in seen)
        tables = 4 * sum(-(-k // c["page"]) for _, k in seen)
    else:
        # the window and the first tokens once a key/value head, the ids once a list
        dense = sum(min(n + m, c["window"] + c["sinks"]) for n, m in zip(new, cached))
        found = c["requests"] * c["lists"] * c["ids"] * 7 // 8
        pairs, keys = H * dense + found * (H // c["lists"]), c["heads_kv"] * dense + found
        tables = 4 * (found + -(-dense // c["page"])) + 4 * c["requests"] * c["lists"] * c["ids"]
    return {"bytes": 4 * keys * D + 4 * T * H * D + 4 * T * H + tables, "flops": 4 * D * pairs}


# ------------------------------------------------------------------ the definitions in 64 bits

def _exact_row_block(q, k, v, seen, scale):
    s = (q @ k.T) * scale
    s[~seen] = -math.inf
    some = seen.any(1)
    lse = torch.logsumexp(s, 1)
    w = torch.exp(s - torch.where(some, lse, 0.0)[:, None])
    return w @ v, lse


def exact(case, seed):
    c = case
    if c["op"] == "plan":
        return None  # whole numbers
    s = prepare(case, seed)
    page = c["page"]
    if c["op"] == "append":
        got = {}
        keep = s["slots"] >= 0
        for name in ("k", "v"):
            flat = s[name + "_cache"].double().reshape(-1, c["heads_kv"], c["dim"])
            flat[s["slots"][keep]] = s[name][keep].double()
            got[name + "_cache"] = flat.view(-1, page, c["heads_kv"], c["dim"])
        return got
    new, cached = _lengths(c)
    H, D, G = c["heads"], c["dim"], c["heads"] // c["heads_kv"]
    out = torch.zeros((s["tokens"], H, D), dtype=torch.float64, device=DEV)
    lse = torch.full((s["tokens"], H), -math.inf, dtype=torch.float64, device=DEV)
    at = 0
    for r, (n, m) in enumerate(zip(new, cached)):
        j = torch.arange(n + m, device=DEV)
        where = s["table"][r].long()[j // page]
        p = torch.arange(m, m + n, device=DEV)[:, None]
        if c["op"] == "attend":
            seen = j[None] <= p
            if c["window"]:
                seen = seen & ((p - j[None] < c["window"]) | (j[None] < c["sinks"]))
        for h in range(H):
            if c["op"] == "retrieved":
                if h % (H // c["lists"]) == 0:
                    ids = s["ids"][r, h // (H // c["lists"])].long()
                    seen = ((j < c["sinks"]) | (j >= n + m - c["window"]))[None].clone()
                    seen[0, ids[ids < n + m]] = True
            if h % G == 0:
                k = s["k_cache"][where, j % page, h // G].double()
                v = s["v_cache"][where, j % page, h // G].double()
            if n:
                out[at:at + n, h], lse[at:at + n, h] = _exact_row_block(s["q"][at:at + n, h].double(), k, v, seen, s["scale"])
        at += n
    return {"out": out, "lse": lse}
