"""Performance cases of attention over selected blocks of a paged cache, and of
eviction from that cache.

Every case is a plain dict; `op` says which entry point of
flashgann_amd.attention a pass goes through:

  bounds   cache_bounds: 8-bit bounds of the keys of each page that new tokens filled
  select   select_blocks: the pages whose bounds promise a query the most
  blocks   attend_blocks: attention over the selected pages, the first and the last ones
  weigh    cache_weigh: the attention weight that every cached token has drawn so far
  evict    cache_evict: a cache back to its budget by those weights

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

def _bounds(tokens, padding, run, heads_kv, dim, page, dtype, layout):
    """run: consecutive tokens of a request (1: a decode step)."""
    return dict(op="bounds", tokens=tokens, padding=padding, run=run, heads_kv=heads_kv, dim=dim, page=page, dtype=dtype,
                layout=layout)


def _rows_of(op, requests, new, cached, heads, heads_kv, dim, page, dtype, layout, **more):
    return dict(op=op, requests=requests, new_lo=new[0], new_hi=new[1], cached_lo=cached[0], cached_hi=cached[1],
                heads=heads, heads_kv=heads_kv, dim=dim, page=page, dtype=dtype, layout=layout, **more)


def _select(requests, new, cached, heads, heads_kv, lists, dim, page, dtype, k, first=1, last=2):
    return _rows_of("select", requests, new, cached, heads, heads_kv, dim, page, dtype, "nhd", lists=lists, k=k, first=first,
                    last=last)


def _blocks(requests, new, cached, heads, heads_kv, lists, dim, page, dtype, layout, k, first=1, last=2):
    return _rows_of("blocks", requests, new, cached, heads, heads_kv, dim, page, dtype, layout, lists=lists, k=k, first=first,
                    last=last)


def _weigh(requests, new, cached, heads, heads_kv, dim, page, dtype, layout):
    return _rows_of("weigh", requests, new, cached, heads, heads_kv, dim, page, dtype, layout)


def _evict(requests, held, budget, window, sinks, heads_kv, dim, page, dtype, layout):
    return _rows_of("evict", requests, (0, 0), held, heads_kv, heads_kv, dim, page, dtype, layout, budget=budget, window=window,
                    sinks=sinks)


def listed():
    named = {
        # the pages that one decode step of 64 requests fills: about one in 16 tokens ends a page
        "bounds_decode": _bounds(64, 0, 1, 8, 128, 16, "bf16", "nhd"),
        # those of a large prefill step, a padded batch, pages laid out head by head
        "bounds_prompt": _bounds(30000, 700, 2500, 8, 128, 64, "fp16", "hnd"),
        # a serving batch of single tokens, 16-token pages, one list for each group of heads
        "select_decode": _select(32, (1, 1), (4000, 24000), 32, 8, 8, 128, 16, "bf16", 64),
        # one user with one very long document, a list for every query head
        "select_long": _select(1, (1, 1), (131070, 131070), 16, 2, 16, 128, 16, "fp16", 256),
        # a chunk of a long prompt: every token selects for itself; the largest selection
        "select_chunk": _select(1, (4096, 4096), (60001, 60001), 32, 8, 8, 128, 64, "bf16", 16),
        # the smallest attention call: drafts of one to five tokens; no size is a power of two
        "blocks_draft": _blocks(5, (1, 5), (200, 3000), 12, 4, 4, 96, 24, "fp16", "nhd", 10),
        # a serving batch of single tokens over long contexts
        "blocks_decode": _blocks(48, (1, 1), (4000, 32000), 32, 8, 8, 128, 32, "bf16", "nhd", 48),
        # a chunk of a long prompt, every token over the blocks that it selected: the largest call
        "blocks_chunk": _blocks(1, (2048, 2048), (62000, 62000), 32, 8, 8, 128, 64, "bf16", "hnd", 16),
        # a decode step's weights, added to those of the steps before
        "weigh_decode": _weigh(32, (1, 1), (500, 8000), 32, 8, 128, 16, "bf16", "nhd"),
        # the last rows of two prompts, from which their tokens' first weights come
        "weigh_prompt": _weigh(2, (300, 500), (12000, 16000), 32, 8, 128, 64, "bf16", "hnd"),
        # running requests back to their budget, a few tokens over it
        "evict_step": _evict(48, (4097, 4160), 4096, 64, 4, 8, 128, 16, "bf16", "nhd"),
        # four long prompts down to it at once
        "evict_prompt": _evict(4, (20000, 32000), 4096, 256, 4, 8, 128, 64, "fp16", "hnd"),
    }
    return [dict(name=n, **c) for n, c in named.items()]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choices(("bounds", "select", "blocks", "weigh", "evict"), (12, 24, 30, 18, 16))[0]
    heads_kv, group = rng.choice(((8, 4), (8, 8), (2, 8), (4, 3), (4, 7), (1, 16), (12, 1), (8, 2), (16, 1), (2, 20)))
    heads = heads_kv * group
    dim = rng.choice((64, 96, 128, 128, 128, 256))
    dtype, layout = rng.choice(("bf16", "bf16", "fp16")), rng.choice(("nhd", "nhd", "hnd"))
    page = rng.choice((16, 16, 32, 64, 128, 8, 24))
    if op == "bounds":
        # a decode step's single tokens, or up to 40 requests' chunks
        run, tokens = (1, _log_int(rng, 1, 512)) if rng.random() < 0.4 else (0, _log_int(rng, 1, 30_000))
        return _bounds(tokens, rng.choice((0, 0, tokens // 3)), run or rng.randint(-(-tokens // 40), tokens), heads_kv, dim,
                       rng.choice((page, page, page, 1)), dtype, layout)
    if op == "evict":
        requests = _log_int(rng, 1, 64)
        budget = _log_int(rng, 40, min(8192, 200_000 // requests))
        most = rng.choice((budget + 1, budget + _log_int(rng, 2, 200), min(budget * 8, 200_000 // requests)))
        window = rng.choice((0, 1, min(32, budget // 2), budget // 4))
        return _evict(requests, (rng.choice((1, budget, most)), max(most, budget + 1)), budget, window, rng.choice((0, 1, 4)),
                      heads_kv, dim, page, dtype, layout)
    if op == "weigh":
        requests = _log_int(rng, 1, 64)
        new = rng.choice((1, 1, 1, 4, _log_int(rng, 2, 600)))
        # the padded scores stay below those of the largest listed case
        cached = _log_int(rng, 1, max(2, min(120_000, int(5e8 / (requests * heads * new)), int(3e8 / (requests * heads_kv * dim)))))
        return _weigh(requests, (rng.choice((1, new)), new), (rng.choice((0, cached // 4, cached)), cached), heads, heads_kv, dim,
                      page, dtype, layout)
    lists = rng.choice((heads_kv, heads_kv, heads))
    first, last = rng.choice((0, 1, 1, 4)), rng.choice((1, 2, 2, 8))
    single = rng.random() < 0.55  # one token each, or the few of a draft
    new = rng.choice((1, 1, 1, 3, 5)) if single else _log_int(rng, 6, 4096)
    requests = _log_int(rng, 1, 64) if single else rng.choice((1, 1, 3))
    cached = _log_int(rng, 1, max(2, min(130_000, int(4e8 / (requests * heads_kv * dim)))))
    while requests * new * lists * (cached // page) > 33_000_000:  # the scores of the largest listed case
        new = max(1, new // 2)
    if op == "select":
        cached = max(cached, page * (first + last + 2))
        k = min(_log_int(rng, 1, 300), (cached // page - first - last + 1) // 2)
        return _select(requests, (rng.choice((1, new)), new), (rng.choice((0, cached // 3, cached)), cached), heads, heads_kv,
                       lists, dim, page, dtype, k, first, last)
    k = max(1, _log_int(rng, 8, 2048) // page)
    # the gathered keys stay below those of the largest listed case
    while requests * new * lists * (k + first + last) * page * dim > 2.2e9:
        new, k = max(1, (2 * new) // 3), max(1, (3 * k) // 4)
    return _blocks(requests, (rng.choice((1, new)), new), (rng.choice((0, cached // 3, cached)), cached), heads, heads_kv, lists,
                   dim, page, dtype, layout, k, first, last)


# ------------------------------------------------------------------ inputs

def _lengths(c):
    """(new tokens, cached tokens) of each request, the same for every seed."""
    rng = random.Random("lengths %s" % sorted((k, v) for k, v in c.items() if k not in ("name", "dtype", "layout")))
    new = [rng.randint(c["new_lo"], c["new_hi"]) for _ in range(c["requests"])]
    cached = [rng.randint(c["cached_lo"], c["cached_hi"]) for _ in range(c["requests"])]
    if c["op"] in ("evict", "select"):
        cached[0] = c["cached_hi"]  # one request at least is over its budget, or has more pages than are selected
    return new, cached


def _ints(v):
    return torch.tensor(v, dtype=torch.int32, device=DEV)


def _cache(c, pages, g, themes=0.0):
    """A cache of (pages, page, heads_kv, dim), whatever the order in memory; with `themes` the tokens of a page
    have something in common, as neighbours in a text have."""
    shape = (pages, c["heads_kv"], c["page"], c["dim"]) if c["layout"] == "hnd" else (pages, c["page"], c["heads_kv"], c["dim"])
    out = torch.randn(shape, generator=g, device=DEV, dtype=TYPES[c["dtype"]])
    out = out.permute(0, 2, 1, 3) if c["layout"] == "hnd" else out
    if themes:
        # the page's theme, and a few channels that lie off zero, as trained keys' do
        theme = torch.randn((pages, 1, c["heads_kv"], c["dim"]), generator=g, device=DEV).mul_(themes)
        theme += torch.randn((c["heads_kv"], c["dim"]), generator=g, device=DEV).mul_(0.5)
        out.mul_(0.8).add_(theme.to(out.dtype))
    return out


def prepare(case, seed):
    c = case
    g = torch.Generator(device=DEV)
    g.manual_seed(seed)
    s = dict(case=c, op=c["op"])
    page, H, D = c["page"], c["heads_kv"], c["dim"]
    if c["op"] == "bounds":
        # runs of tokens, each a request's, that begin anywhere in a page and fill pages in random order
        T, length = c["tokens"], min(c["run"], c["tokens"])
        t = torch.arange(T, device=DEV)
        runs = -(-T // length)
        each = (length + page - 2) // page + 1  # pages of a run at most
        begin = torch.randint(page, (runs,), generator=g, device=DEV)
        begin[0] = page - 1  # one page at least is filled
        order = torch.randperm(runs * each, generator=g, device=DEV)
        at = begin[t // length] + t % length
        s["slots"] = order[(t // length) * each + at // page] * page + at % page
        if c["padding"]:
            s["slots"][T - c["padding"]:] = -1
        s["k_cache"] = _cache(c, runs * each, g, 0.6)
        s["bounds"] = torch.zeros((runs * each, H, 2, D), dtype=torch.int8, device=DEV)
        s["scales"] = torch.zeros((runs * each, H), device=DEV)
        return s
    new, cached = _lengths(c)
    total = [n + m for n, m in zip(new, cached)]
    width = max(1, max(-(-t // page) for t in total))
    b = torch.arange(width, device=DEV)
    s["new"], s["kv_lens"], s["known"] = _ints(new), _ints(total), _ints(cached)
    s["q_starts"] = _ints([sum(new[:r]) for r in range(len(new) + 1)])
    s["tokens"], s["max_new"], s["max_kv"] = sum(new), max(new), max(max(total), 1)
    need = -(-s["kv_lens"] // page)  # pages that each request holds
    pages = sum(-(-t // page) for t in total) + 3
    order = torch.randperm(pages - 1, generator=g, device=DEV).to(torch.int32)  # the last page is nobody's
    first = torch.cumsum(need, 0) - need
    held = b < need[:, None]
    s["table"] = torch.where(held, order[(first[:, None] + b).clamp(max=pages - 2)], -1).to(torch.int32)
    s["k_cache"] = _cache(c, pages, g, 0.6)
    if c["op"] in ("blocks", "evict"):
        s["v_cache"] = _cache(c, pages, g)
    if c["op"] == "evict":
        # a few tokens drew most of the weight, and some of them none at all
        w = torch.exp(2.0 * torch.randn((pages, H, page), generator=g, device=DEV) - 2.0)
        s["drawn"] = w.mul_(torch.rand(w.shape, generator=g, device=DEV) > 0.2)
        s["weights"] = s["drawn"].clone()
        return s
    # the queries of a passage ask for much the same
    topic = torch.randn((-(-s["tokens"] // 24) + 1, c["heads"], D), generator=g, device=DEV)
    q = topic[torch.arange(s["tokens"], device=DEV) // 24] + 0.7 * torch.randn((s["tokens"], c["heads"], D), generator=g, device=DEV)
    s["q"] = q.to(TYPES[c["dtype"]])
    s["scale"] = D ** -0.5
    if c["op"] == "weigh":
        scores, _ = _padded_scores(s)
        r, at = _owners(s)
        lse = torch.logsumexp(scores, -1).view(c["requests"], H, -1, s["max_new"])
        s["lse"] = lse[r, :, :, at].reshape(s["tokens"], c["heads"]).contiguous()
        s["weights"] = torch.rand((pages, H, page), generator=g, device=DEV)
        return s
    s["bounds"], s["scales"] = _bounds_of(s["k_cache"])
    if c["op"] == "select":
        del s["k_cache"]
    else:
        s["ids"] = _select_plain(s)["ids"]
        del s["bounds"], s["scales"]
    return s


# ------------------------------------------------------------------ plain forms

def _power_of_two(most):
    """The least power of two of which 127 reach `most`, not below 2^-126."""
    part, exponent = torch.frexp(most)
    exponent = exponent - 7 + (part > 127 / 128).to(exponent.dtype)
    return ((exponent.clamp(min=-126) + 127) << 23).view(torch.float32)


def _bounds_of(keys):
    """Codes (n, heads_kv, 2, dim) and scales (n, heads_kv) of n pages' keys (n, page, heads_kv, dim): the largest
    and the smallest of each channel, rounded outwards.  A page with a key that is not finite: infinity and zeros."""
    k = keys.float()
    both = torch.stack([k.amax(1), k.amin(1)], 2)
    most = both.abs().amax((2, 3))
    fine = torch.isfinite(most)
    scale = _power_of_two(torch.where(fine, most, 1.0))
    codes = both / scale[:, :, None, None]
    codes = torch.where(torch.tensor([[True], [False]], device=DEV), torch.ceil(codes), torch.floor(codes))
    codes = torch.where(fine[:, :, None, None], codes, 0.0).to(torch.int8)
    return codes, torch.where(fine, scale, math.inf)


def _bounds_plain(s):
    page, slots = s["case"]["page"], s["slots"]
    done = slots[(slots >= 0) & (slots % page == page - 1)] // page
    s["bounds"][done], s["scales"][done] = _bounds_of(s["k_cache"][done])
    return {"bounds": s["bounds"] * s["scales"][:, :, None, None], "scales": s["scales"]}


def _owners(s):
    """(request, number among its new tokens) of every row."""
    t = torch.arange(s["tokens"], device=DEV)
    r = torch.searchsorted(s["q_starts"][1:].long(), t, right=True)
    return r, t - s["q_starts"].long()[r]


def _padded_rows(s, rows):
    i = torch.arange(s["max_new"], device=DEV)
    return rows[(s["q_starts"][:-1, None] + i).clamp(max=s["tokens"] - 1).long()]


def _select_plain(s):
    c = s["case"]
    B, Q, L, H, D, page = c["requests"], s["max_new"], c["lists"], c["heads_kv"], c["dim"], c["page"]
    q = s["q"].float().view(-1, L, c["heads"] // L, D)
    asked = torch.cat([q.clamp(min=0).sum(2), q.clamp(max=0).sum(2)], -1)
    asked = torch.round(asked / _power_of_two(asked.abs().amax(-1, keepdim=True)))
    asked = _padded_rows(s, asked).view(B, Q, H, L // H, 2 * D).permute(0, 2, 3, 1, 4).reshape(B, H, -1, 2 * D)
    at = s["table"].clamp(min=0).long()
    held = s["bounds"][at].float().view(B, -1, H, 2 * D).permute(0, 2, 3, 1).contiguous()
    score = torch.matmul(asked, held) * s["scales"][at].permute(0, 2, 1)[:, :, None]
    N = at.shape[1]
    score = score.view(B, H, L // H, Q, N)
    b = torch.arange(N, device=DEV)
    pos = (s["kv_lens"] - s["new"])[:, None, None] + torch.arange(Q, device=DEV)[:, None]
    seen = ((b >= c["first"]) & (b <= pos // page - c["last"]))[:, None, None]
    score = score.masked_fill_(~seen, -math.inf)
    k = min(c["k"], N)
    best, ids = score.sort(dim=-1, descending=True, stable=True)
    ids = torch.where(best[..., :k] > -math.inf, ids[..., :k], N).sort(-1).values
    ids = torch.nn.functional.pad(torch.where(ids < N, ids, -1), (0, c["k"] - k), value=-1)
    r, i = _owners(s)
    return {"ids": ids[r, :, :, i].reshape(-1, L, c["k"]).to(torch.int32)}


def _blocks_plain(s):
    c = s["case"]
    T, L, D, page = s["tokens"], c["lists"], c["dim"], c["page"]
    r, i = _owners(s)
    pos = (s["kv_lens"] - s["new"])[r] + i
    tail = (pos // page - c["last"] + 1).clamp(min=c["first"])  # the first of the last blocks
    b = torch.cat([torch.arange(c["first"], device=DEV).expand(T, L, -1), s["ids"].long(),
                   (tail[:, None] + torch.arange(c["last"], device=DEV))[:, None].expand(T, L, -1)], -1)
    j = b[..., None] * page + torch.arange(page, device=DEV)
    seen = ((b >= 0)[..., None] & (j <= pos[:, None, None, None])).view(T, L, -1)
    j = torch.where(seen, j.view(T, L, -1), 0)
    at = s["table"].long()[r[:, None, None], j // page].clamp(min=0)
    head = (torch.arange(L, device=DEV) // (L // c["heads_kv"]))[:, None]
    q = s["q"].float().view(T, L, c["heads"] // L, D)
    k = s["k_cache"][at, j % page, head].float().transpose(2, 3).contiguous()
    scores = torch.matmul(q, k).mul_(s["scale"]).masked_fill_(~seen[:, :, None], -math.inf)
    m = scores.amax(-1, keepdim=True)
    p = torch.exp(scores - m)
    l = p.sum(-1, keepdim=True)
    out = torch.matmul(p, s["v_cache"][at, j % page, head].float()) / l
    return {"out": out.view(T, c["heads"], D).to(s["q"].dtype), "lse": (m + torch.log(l)).view(T, c["heads"])}


def _padded_scores(s):
    """(scores (requests, heads_kv, group, new, tokens), -inf where unseen, and the slots of the tokens)."""
    c = s["case"]
    B, Q, L, H, D, page = c["requests"], s["max_new"], s["max_kv"], c["heads_kv"], c["dim"], c["page"]
    j = torch.arange(L, device=DEV)
    at = s["table"][:, j // page].long()
    k = s["k_cache"][at.clamp(min=0), j % page].float().permute(0, 2, 3, 1).contiguous()
    q = _padded_rows(s, s["q"].float()).view(B, Q, H, -1, D).permute(0, 2, 3, 1, 4).reshape(B, H, -1, D)
    scores = torch.matmul(q, k).mul_(s["scale"]).view(B, H, -1, Q, L)
    i = torch.arange(Q, device=DEV)[:, None]
    seen = (j <= (s["kv_lens"] - s["new"])[:, None, None] + i) & (i < s["new"][:, None, None])
    return scores.masked_fill_(~seen[:, None, None], -math.inf), at


def _weigh_plain(s):
    c = s["case"]
    B, H, page = c["requests"], c["heads_kv"], c["page"]
    scores, at = _padded_scores(s)
    lse = _padded_rows(s, s["lse"]).view(B, -1, H, c["heads"] // H).permute(0, 2, 3, 1)
    drawn = torch.exp(scores.sub_(lse[..., None])).sum((2, 3))  # (requests, heads_kv, tokens)
    j = torch.arange(s["max_kv"], device=DEV)
    r, h = torch.arange(B, device=DEV)[:, None, None], torch.arange(H, device=DEV)[:, None]
    at = torch.where((j < s["kv_lens"][:, None]) & (at >= 0), at, s["weights"].shape[0])[:, None]
    old = torch.nn.functional.pad(s["weights"], (0, 0, 0, 0, 0, 1))  # one page for what has none
    fresh = (j >= s["known"][:, None])[:, None]
    old[at.expand(B, H, -1), h.expand(B, H, -1), (j % page).expand(B, H, -1)] = torch.where(fresh, 0.0, old[at, h, j % page]) + drawn
    s["weights"].copy_(old[:-1])
    return {"weights": s["weights"]}


def _evict_plain(s):
    c = s["case"]
    B, H, page, width = c["requests"], c["heads_kv"], c["page"], s["table"].shape[1]
    budget, window, sinks = c["budget"], c["window"], c["sinks"]
    keep, N = budget - window, s["max_kv"]
    kv = s["kv_lens"].long()
    j = torch.arange(N, device=DEV)
    at = s["table"].long()[:, j // page]
    h = torch.arange(H, device=DEV)[:, None]
    # the heaviest of what is neither among the first nor among the last
    w = s["weights"][at.clamp(min=0)[:, None], h, j % page]
    end = (kv - window)[:, None, None]
    w = torch.where(j < sinks, math.inf, torch.where(j < end, w, -math.inf))
    rank = w.sort(dim=-1, descending=True, stable=True).indices
    kept = torch.zeros_like(w, dtype=torch.bool).scatter_(-1, rank[..., :keep], True) & (j < end)
    over = (kv > budget)[:, None, None]
    # place j takes the token at source[j]: holes below `keep` the survivors above it, then the last ones
    hole, late = ~kept[..., :keep], kept & (j >= keep)
    order = torch.where(late, j, N).sort(-1).values
    taken = torch.gather(order, -1, (torch.cumsum(hole, -1) - 1).clamp(min=0).expand(B, H, -1))
    source = torch.cat([torch.where(hole, taken, j[:keep]), (kv[:, None, None] - window + torch.arange(window, device=DEV)).expand(B, H, window)], -1)
    to = j[:budget]
    source = torch.where(over, source, to)
    slot = lambda x: torch.gather(at, 1, x.reshape(B, -1)).view(x.shape).clamp(min=0)  # noqa: E731
    here, there = at[:, None, :budget].expand(B, H, -1), slot(source)
    real = here >= 0
    last = s["k_cache"].shape[0] - 1  # a request shorter than its budget has fewer pages: the last page is nobody's
    here, there = torch.where(real, here, last), torch.where(real, there, last)
    from_at, to_at = torch.where(real, source % page, 0), torch.where(real, to % page, 0)
    for cache in (s["k_cache"], s["v_cache"]):
        cache[here, to_at, h] = cache[there, from_at, h]
    s["weights"][here, h, to_at] = s["weights"][there, h, from_at]
    lens = kv.clamp(max=budget)
    left, had = -(-lens // page), -(-kv // page)
    b = torch.arange(width, device=DEV)
    gone = (b >= left[:, None]) & (b < had[:, None])
    place = torch.where(gone, torch.cumsum(gone.view(-1), 0).view(B, width) - 1, B * width)
    freed = torch.full((B * width + 1,), -1, dtype=torch.int32, device=DEV)
    freed[place.view(-1)] = torch.where(gone, s["table"], -1).view(-1)
    return {"k_cache": s["k_cache"], "v_cache": s["v_cache"], "weights": s["weights"], "kv_lens": lens.to(torch.int32),
            "freed": freed[:-1], "released": gone.sum().to(torch.int32).view(1)}


PLAIN = {"bounds": _bounds_plain, "select": _select_plain, "blocks": _blocks_plain, "weigh": _weigh_plain, "evict": _evict_plain}


# ------------------------------------------------------------------ a pass

def run(state):
    s = state
    c = s["case"]
    if c["op"] == "evict":
        s["weights"].copy_(s["drawn"])  # as attention left them: a pass after another has the same to do
    if not own:
        return PLAIN[s["op"]](s)
    from flashgann_amd import attention
    if c["op"] == "bounds":
        attention.cache_bounds(s["k_cache"], s["slots"], s["bounds"], s["scales"])
        return {"bounds": s["bounds"] * s["scales"][:, :, None, None], "scales": s["scales"]}
    if c["op"] == "select":
        return {"ids": attention.select_blocks(s["q"], s["bounds"], s["scales"], s["table"], s["q_starts"], s["kv_lens"],
                                               page_size=c["page"], k=c["k"], lists=c["lists"], first_blocks=c["first"],
                                               last_blocks=c["last"])}
    if c["op"] == "blocks":
        out, lse = attention.attend_blocks(s["q"], s["k_cache"], s["v_cache"], s["table"], s["q_starts"], s["kv_lens"], s["ids"],
                                           first_blocks=c["first"], last_blocks=c["last"], scale=s["scale"])
        return {"out": out, "lse": lse}
    if c["op"] == "weigh":
        attention.cache_weigh(s["q"], s["k_cache"], s["table"], s["q_starts"], s["kv_lens"], s["lse"], s["weights"], s["known"],
                              scale=s["scale"])
        return {"weights": s["weights"]}
    e = attention.cache_evict(s["k_cache"], s["v_cache"], s["weights"], s["table"], s["kv_lens"], budget=c["budget"],
                              window=c["window"], sinks=c["sinks"])
    return {"k_cache": s["k_cache"], "v_cache": s["v_cache"], "weights": s["weights"], "kv_lens": e.kv_lens, "freed": e.freed,
            "released": e.released}


# ------------------------------------------------------------------ what a pass cannot do without

def work(case):
    c = case
    D, H, page = c["dim"], c["heads_kv"], c["page"]
    if c["op"] == "bounds":
        full = (c["tokens"] - c["padding"]) / page  # on average
        return {"bytes": int(full * H * (2 * page * D + 2 * D + 4)) + 8 * c["tokens"], "flops": 0}
    new, cached = _lengths(c)
    T = sum(new)
    if c["op"] == "evict":
        keep, rows, weights = c["budget"] - c["window"], 0, 0
        for m in cached:
            if m > c["budget"]:
                # weights fall on tokens whatever their place: so many of the kept ones lie behind the place `keep`
                rows += c["window"] + keep * (1 - keep / max(m - c["window"], 1))
                weights += m
        return {"bytes": int(H * (rows * (8 * D + 8) + 4 * weights)), "flops": 0}
    heads = c["heads"]
    if c["op"] == "weigh":
        pairs = sum(n * m + n * (n + 1) // 2 for n, m in zip(new, cached))
        keys = sum(n + m for n, m in zip(new, cached))
        return {"bytes": H * keys * (2 * D + 8) - 4 * H * T + 2 * T * heads * D + 4 * T * heads, "flops": 2 * D * heads * pairs}
    L, bytes_, pairs = c["lists"], 0, 0
    for n, m in zip(new, cached):
        blocks = [max(0, p // page - c["last"] + 1 - c["first"]) for p in range(m, m + n)]  # that a row can select from
        if c["op"] == "select":
            bytes_ += H * max(blocks, default=0) * (2 * D + 4)
            pairs += L * sum(blocks)
            continue
        # (one row's last block ends at its own token)
        rows = [min(c["k"], x) * page + min(p + 1, (c["first"] + c["last"] - 1) * page + p % page + 1) for x, p in zip(blocks, range(m, m + n))]
        bytes_ += 4 * D * min(H * (n + m), L * sum(rows))  # no key twice, whoever selected it
        pairs += heads * sum(rows)
    if c["op"] == "select":
        return {"bytes": bytes_ + 2 * T * heads * D + 4 * T * L * c["k"], "flops": 4 * D * pairs}
    return {"bytes": bytes_ + 4 * T * heads * D + 4 * T * heads + 4 * T * L * c["k"], "flops": 4 * D * pairs}


# ------------------------------------------------------------------ the definitions in 64 bits

def _tokens(s, cache, r, n):
    """Tokens 0 .. n-1 of request r: (heads_kv, n, dim) in 64 bits."""
    j = torch.arange(n, device=DEV)
    page = s["case"]["page"]
    return cache[s["table"][r].long()[j // page], j % page].double().transpose(0, 1)


def _exact_bounds(s):
    slots, page = s["slots"].tolist(), s["case"]["page"]
    values, scales = torch.zeros(s["bounds"].shape, dtype=torch.float64, device=DEV), torch.zeros_like(s["scales"], dtype=torch.float64)
    full = torch.tensor(sorted({t // page for t in slots if t >= 0 and t % page == page - 1}), dtype=torch.long, device=DEV)
    k = s["k_cache"][full].double()
    high, low = k.max(1).values, k.min(1).values
    most = torch.maximum(high.abs().max(-1).values, low.abs().max(-1).values)
    powers = torch.tensor([2.0 ** e for e in range(-126, 122)], dtype=torch.float64, device=DEV)
    step = powers[torch.searchsorted(127 * powers, most)]
    values[full, :, 0] = torch.ceil(high / step[..., None]) * step[..., None]
    values[full, :, 1] = torch.floor(low / step[..., None]) * step[..., None]
    scales[full] = step
    return {"bounds": values, "scales": scales}


def _exact_blocks(s, new, cached):
    c = s["case"]
    heads, H, L, D, page = c["heads"], c["heads_kv"], c["lists"], c["dim"], c["page"]
    out = torch.empty((s["tokens"], heads, D), dtype=torch.float64, device=DEV)
    lse = torch.empty((s["tokens"], heads), dtype=torch.float64, device=DEV)
    at = 0
    for r, (n, m) in enumerate(zip(new, cached)):
        k, v = _tokens(s, s["k_cache"], r, n + m), _tokens(s, s["v_cache"], r, n + m)
        j = torch.arange(n + m, device=DEV)
        for i in range(0, n, 8):
            rows = range(at + i, at + min(i + 8, n))
            w = len(rows)
            p = torch.arange(m + i, m + i + w, device=DEV)[:, None, None]
            chosen = torch.zeros((w, L, (n + m) // page + 2), dtype=torch.bool, device=DEV)
            ids = s["ids"][rows.start:rows.stop].long()
            chosen.scatter_(2, torch.where(ids >= 0, ids, (n + m) // page + 1), True)
            seen = chosen[..., j // page] | (j // page < c["first"]) | (j // page > p // page - c["last"])
            seen = (seen & (j <= p)).repeat_interleave(heads // L, 1).view(w, H, -1, n + m).transpose(0, 1)
            q = s["q"][rows.start:rows.stop].double().view(w, H, -1, D).transpose(0, 1)
            score = (q.reshape(H, -1, D) @ k.transpose(1, 2)).view(H, w, -1, n + m) * s["scale"]
            score[~seen] = -math.inf
            z = torch.logsumexp(score, -1)
            o = torch.exp(score - z[..., None]).view(H, -1, n + m) @ v
            out[rows.start:rows.stop] = o.view(H, w, -1, D).transpose(0, 1).reshape(w, heads, D)
            lse[rows.start:rows.stop] = z.transpose(0, 1).reshape(w, heads)
        at += n
    return {"out": out, "lse": lse}


def _exact_weigh(s, new, cached):
    c = s["case"]
    H, page = c["heads_kv"], c["page"]
    w = s["weights"].double()
    at = 0
    for r, (n, m) in enumerate(zip(new, cached)):
        k = _tokens(s, s["k_cache"], r, n + m)
        j = torch.arange(n + m, device=DEV)
        p = torch.arange(m, m + n, device=DEV)[:, None]
        where = s["table"][r].long()[j // page]
        for h in range(c["heads"]):
            if h % (c["heads"] // H) == 0:
                drawn = torch.zeros(n + m, dtype=torch.float64, device=DEV)
            score = (s["q"][at:at + n, h].double() @ k[h // (c["heads"] // H)].T) * s["scale"]
            p_ = torch.exp(score - s["lse"][at:at + n, h].double()[:, None])
            drawn += torch.where(j <= p, p_, 0.0).sum(0)
            if (h + 1) % (c["heads"] // H) == 0:
                kv_head = h // (c["heads"] // H)
                before = w[where, kv_head, j % page]
                before[m:] = 0.0
                w[where, kv_head, j % page] = before + drawn
        at += n
    return {"weights": w}


def _exact_evict(s, cached):
    c = s["case"]
    page, keep, window = c["page"], c["budget"] - c["window"], c["window"]
    k, v, w = s["k_cache"].double(), s["v_cache"].double(), s["drawn"].double()
    for r, n in enumerate(cached):
        if n <= c["budget"]:
            continue
        table = s["table"][r].tolist()
        for h in range(c["heads_kv"]):
            where = torch.tensor(table, device=DEV)
            j = torch.arange(n, device=DEV)
            drawn = w[where[j // page], h, j % page].cpu().tolist()
            inside = sorted(range(c["sinks"], n - window), key=lambda x: (-drawn[x], x))
            stay = set(range(c["sinks"])) | set(inside[:keep - c["sinks"]])
            holes = [x for x in range(keep) if x not in stay]
            late = sorted(x for x in stay if x >= keep)
            to = torch.tensor(holes + list(range(keep, c["budget"])), dtype=torch.long, device=DEV)
            of = torch.tensor(late + list(range(n - window, n)), dtype=torch.long, device=DEV)
            to_page, of_page = where[to // page], where[of // page]
            k[to_page, to % page, h] = k[of_page, of % page, h]
            v[to_page, to % page, h] = v[of_page, of % page, h]
            w[to_page, h, to % page] = w[of_page, h, of % page]
    return {"k_cache": k, "v_cache": v, "weights": w, "kv_lens": None, "freed": None, "released": None}


def exact(case, seed):
    c = case
    if c["op"] == "select":
        return None  # whole numbers
    s = prepare(case, seed)
    if c["op"] == "bounds":
        return _exact_bounds(s)
    new, cached = _lengths(c)
    if c["op"] == "blocks":
        return _exact_blocks(s, new, cached)
    return _exact_weigh(s, new, cached) if c["op"] == "weigh" else _exact_evict(s, cached)
