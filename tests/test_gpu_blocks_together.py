"""The operators over selected pages and of eviction as a program runs them: prompts in
chunks and decode steps, on other streams, captured and replayed, at the limits of what
they take."""
from __future__ import annotations

import numpy as np
import pytest
import torch

import attention_oracle as A
import blocks_oracle as O
from test_gpu_blocks import case, ints, some_ids, starts_of

pytestmark = pytest.mark.gpu

BF, FP = torch.bfloat16, torch.float16
MOST = 2 ** 31 - 1


@pytest.fixture(autouse=True)
def _gpu(gpu_available):
    torch.cuda.set_device(0)


class Serving:
    """Requests over one cache, with bounds and weights; every call is the framework's."""

    def __init__(self, requests, pages, page, heads, heads_kv, dim, dtype, seed):
        self.rng, self.page, self.heads, self.heads_kv, self.dim, self.dtype = np.random.default_rng(seed), page, heads, heads_kv, dim, dtype
        z = lambda shape, d: torch.zeros(shape, dtype=d, device="cuda")  # noqa: E731
        self.k, self.v = z((pages, page, heads_kv, dim), dtype), z((pages, page, heads_kv, dim), dtype)
        self.bounds, self.scales, self.weights = z((pages, heads_kv, 2, dim), torch.int8), z((pages, heads_kv), torch.float32), z((pages, heads_kv, page), torch.float32)
        self.table = torch.full((requests, pages), -1, dtype=torch.int32, device="cuda")
        self.free = torch.from_numpy(self.rng.permutation(pages).astype(np.int32)).cuda()
        self.lens = z(requests, torch.int32)

    def randn(self, *shape):
        return torch.from_numpy(self.rng.standard_normal(shape).astype(np.float32)).to(self.dtype).cuda()

    def append(self, new):
        from flashgann_amd import attention
        p = attention.cache_plan(self.lens, ints(new), self.table, self.free, page_size=self.page, max_tokens=sum(new))
        attention.cache_append(self.randn(sum(new), self.heads_kv, self.dim), self.randn(sum(new), self.heads_kv, self.dim), self.k, self.v, p.slots)
        attention.cache_bounds(self.k, p.slots, self.bounds, self.scales)
        self.free, self.known, self.lens = self.free[int(p.used):].contiguous(), self.lens, p.kv_lens
        return p


@pytest.mark.parametrize("dtype,dim,heads,heads_kv,page", ((BF, 128, 8, 2, 8), (FP, 96, 6, 3, 5), (BF, 64, 7, 1, 16)))
def test_prompts_and_steps_over_selected_pages(dtype, dim, heads, heads_kv, page):
    """Prompts in chunks, then tokens, then drafts: what is selected comes from the bounds that appends left, and every
    output is the definition's."""
    from flashgann_amd import attention
    s = Serving(3, 120, page, heads, heads_kv, dim, dtype, page)
    for step, new in enumerate(([40, 3, 0], [60, 90, 1], [1, 1, 1], [1, 1, 1], [4, 0, 3], [1, 30, 1])):
        p = s.append(new)
        q = s.randn(sum(new), heads, dim)
        ids = attention.select_blocks(q, s.bounds, s.scales, s.table, p.q_starts, p.kv_lens, page_size=page, k=4, first_blocks=1, last_blocks=2)
        out, lse = attention.attend_blocks(q, s.k, s.v, s.table, p.q_starts, p.kv_lens, ids, first_blocks=1, last_blocks=2)
        kv, starts, table = p.kv_lens.tolist(), starts_of(new), s.table.cpu()
        # the bounds of every full page are the definition's of its keys
        full = [int(table[r, b]) for r in range(3) for b in range(kv[r] // page)]
        k = s.k.cpu()
        want = O.bounds(k, full)
        for (pg, h), (codes, scale) in want.items():
            assert float(s.scales[pg, h]) == scale and np.array_equal(s.bounds[pg, h].cpu().numpy(), codes), (step, pg, h)
        chosen = O.select(q.cpu(), s.bounds.cpu(), s.scales.cpu(), table.numpy(), starts, kv, page, 4, heads_kv, 1, 2)
        assert np.array_equal(ids.cpu().numpy(), chosen), step
        O.attend(q.cpu(), k, s.v.cpu(), table, starts, kv, torch.from_numpy(chosen), dim ** -0.5, 1, 2).check(out, lse)


@pytest.mark.parametrize("dtype,dim,heads,heads_kv,page", ((BF, 128, 8, 2, 8), (FP, 64, 6, 6, 5)))
def test_steps_within_a_budget(dtype, dim, heads, heads_kv, page):
    """Attention, weights and eviction step by step, pages given back and taken again: each step's weights within
    their bound, each eviction the definition's of the weights before it, each output the definition's of the cache."""
    from flashgann_amd import attention
    budget, window, sinks = 48, 12, 2
    s = Serving(3, 60, page, heads, heads_kv, dim, dtype, 9)
    for step, new in enumerate(([70, 30, 47], [1, 1, 1], [1, 1, 1], [1, 40, 1], [1, 1, 1], [30, 1, 1])):
        p = s.append(new)
        q = s.randn(sum(new), heads, dim)
        before = s.weights.cpu()
        out, lse = attention.attend(q, s.k, s.v, s.table, p.q_starts, p.kv_lens, max_q=max(new))
        attention.cache_weigh(q, s.k, s.table, p.q_starts, p.kv_lens, lse, s.weights, s.known)
        kv, starts, table, k, v = p.kv_lens.tolist(), starts_of(new), s.table.cpu(), s.k.cpu(), s.v.cpu()
        A.dense(q.cpu(), k, v, table, starts, kv, dim ** -0.5).check(out, lse)
        w, tol = O.weigh(q.cpu(), k, table, starts, kv, lse.cpu(), before, s.known.tolist(), dim ** -0.5)
        assert (np.abs(s.weights.cpu().double().numpy() - w) <= tol).all(), step
        want = O.evict(k, v, s.weights.cpu(), table, kv, budget, window, sinks)
        e = attention.cache_evict(s.k, s.v, s.weights, s.table, s.lens, budget=budget, window=window, sinks=sinks)
        assert torch.equal(s.k.cpu(), want[0]) and torch.equal(s.v.cpu(), want[1]) and torch.equal(s.weights.cpu(), want[2]), step
        assert e.kv_lens.tolist() == want[3] and e.freed.tolist() == want[4] and e.released.tolist() == [want[5]]
        s.free, s.lens = torch.cat([s.free, e.freed[:want[5]]]).contiguous(), e.kv_lens
        held = [int(table[r, b]) for r in range(3) for b in range(-(-want[3][r] // page))]
        assert sorted(held + s.free.tolist()) == list(range(60)), step


def test_same_bits_every_time():
    """Whatever runs when: parts are joined in order, and sums are made in order."""
    from flashgann_amd import attention
    for new, kv, k in (([1], [9000], 200), ([150, 1, 3], [1500, 900, 70], 9), ([1] * 40, [600] * 40, 5)):
        q, kc, vc, table, starts = case(9, new, kv, 8, 2, 128, 16, BF)
        ids = some_ids(np.random.default_rng(1), new, kv, 2, k, 16).cuda()
        args = (q.cuda(), kc.cuda(), vc.cuda(), table.cuda(), ints(starts), ints(kv))
        got = [attention.attend_blocks(*args, ids) for _ in range(4)]
        weighed = []
        for _ in range(3):
            w = torch.zeros((kc.shape[0], 2, 16), device="cuda")
            attention.cache_weigh(args[0], args[1], *args[3:], got[0][1], w, ints([0] * len(kv)))
            weighed.append(w)
        assert all(torch.equal(a, got[0][0]) and torch.equal(b, got[0][1]) for a, b in got[1:])
        assert all(torch.equal(w, weighed[0]) for w in weighed[1:])


def calls(args, bounds, scales, page):
    """One of each on the current stream: (ids, out, lse, weights, eviction, caches)."""
    from flashgann_amd import attention
    q, kc, vc, table, starts, kv = args
    kc, vc = kc.clone(), vc.clone()
    w = torch.zeros((kc.shape[0], kc.shape[2], page), device="cuda")
    ids = attention.select_blocks(q, bounds, scales, table, starts, kv, page_size=page, k=5)
    out, lse = attention.attend_blocks(q, kc, vc, table, starts, kv, ids)
    attention.cache_weigh(q, kc, table, starts, kv, lse, w, kv - 1)
    e = attention.cache_evict(kc, vc, w, table, kv, budget=60, window=7, sinks=1)
    return ids, out, lse, w, *e, kc, vc


@pytest.mark.parametrize("new,kv", (([1, 1], [900, 400]), ([70, 50], [500, 400]), ([2] * 64, [100] * 64), ([400], [900])))
def test_on_another_stream(new, kv):
    from flashgann_amd import attention
    q, kc, vc, table, starts = case(10, new, kv, 8, 2, 128, 16, BF)
    args = (q.cuda(), kc.cuda(), vc.cuda(), table.cuda(), ints(starts), ints(kv))
    bounds, scales = torch.zeros((kc.shape[0], 2, 2, 128), dtype=torch.int8, device="cuda"), torch.zeros((kc.shape[0], 2), device="cuda")
    attention.cache_bounds(args[1], torch.arange(kc.shape[0] * 16, device="cuda"), bounds, scales)
    want = calls(args, bounds, scales, 16)
    torch.cuda.synchronize()
    side, other = torch.cuda.Stream(), torch.cuda.Stream()
    got = []
    for _ in range(3):
        for st in (side, other):  # two at once
            with torch.cuda.stream(st):
                got.append(calls(args, bounds, scales, 16))
    side.synchronize()
    other.synchronize()
    for g in got:
        assert all(torch.equal(a, b) for a, b in zip(g, want))


@pytest.mark.parametrize("new,kv,page", (([1, 1], [900, 400], 16), ([70, 50], [500, 400], 16), ([1], [9000], 4), ([1, 1], [20000, 300], 8), ([2] * 64, [100] * 64, 16), ([400], [900], 8)))
def test_graph_replays(new, kv, page):
    """Captured calls follow what is in device memory: replayed over other queries and lengths, with eager work and
    allocations between, against the same calls made eagerly; two graphs in turn."""
    from flashgann_amd import attention
    q, kc, vc, table, starts = case(11, new, kv, 8, 2, 64, page, FP)
    kd, vd, td, st, lens = kc.cuda(), vc.cuda(), table.cuda(), ints(starts), ints(kv)
    bounds, scales = torch.zeros((kc.shape[0], 2, 2, 64), dtype=torch.int8, device="cuda"), torch.zeros((kc.shape[0], 2), device="cuda")
    slots = torch.arange(kc.shape[0] * page, device="cuda")
    x = q.cuda()

    def step():
        attention.cache_bounds(kd, slots, bounds, scales)
        return calls((x, kd, vd, td, st, lens), bounds, scales, page)

    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        step()
    side.synchronize()
    graphs = []
    for _ in range(2):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            got = step()
        graphs.append((g, got))
    for i in range(6):
        x.copy_(torch.from_numpy(np.random.default_rng(i).standard_normal(tuple(x.shape)).astype(np.float32)).to(FP).cuda())
        lens.copy_(ints([max(m, n - 37 * i) for m, n in zip(new, kv)]))
        kd.mul_(-1)
        want = [t.clone() for t in step()]
        bounds.zero_()
        g, got = graphs[i % 2]
        g.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, want)), i


def test_offsets_past_32_bits():
    """A cache of over 4 GiB a tensor whose last pages hold the context."""
    from flashgann_amd import attention
    page, heads_kv, dim, pages = 64, 8, 128, 36000  # 4.7 GB each
    rng = np.random.default_rng(8)
    small_k, small_v = A.make_cache(rng, 6, page, heads_kv, dim, BF)
    k, v = (torch.empty((pages, page, heads_kv, dim), dtype=BF, device="cuda") for _ in range(2))
    k[pages - 6:], v[pages - 6:] = small_k.cuda(), small_v.cuda()
    small = torch.tensor([[5, 0, 3, 1], [4, 2, -1, -1]], dtype=torch.int32)
    table = torch.where(small >= 0, small + pages - 6, -1)
    kv = [250, 100]
    bounds, scales = torch.zeros((pages, heads_kv, 2, dim), dtype=torch.int8, device="cuda"), torch.zeros((pages, heads_kv), device="cuda")
    weights = torch.zeros((pages, heads_kv, page), device="cuda")
    attention.cache_bounds(k, torch.arange((pages - 6) * page, pages * page, device="cuda"), bounds, scales)
    for p in range(6):
        codes, scale = O.bounds(small_k, [p])[p, 7]
        assert float(scales[pages - 6 + p, 7]) == scale and np.array_equal(bounds[pages - 6 + p, 7].cpu().numpy(), codes)
    for new in ([1, 1], [50, 30]):
        q = torch.from_numpy(rng.standard_normal((sum(new), 16, dim)).astype(np.float32)).to(BF)
        args = ints(starts_of(new)), ints(kv)
        ids = attention.select_blocks(q.cuda(), bounds, scales, table.cuda(), *args, page_size=page, k=1, first_blocks=0)
        out, lse = attention.attend_blocks(q.cuda(), k, v, table.cuda(), *args, ids, first_blocks=0)
        assert bool((ids >= 0).any())
        o = O.attend(q, small_k, small_v, small, starts_of(new), kv, ids.cpu(), dim ** -0.5, 0, 1)
        o.check(out, lse)
        full = attention.attend(q.cuda(), k, v, table.cuda(), *args, max_q=max(new))[1]
        attention.cache_weigh(q.cuda(), k, table.cuda(), *args, full, weights, ints([0, 0]))
        w, tol = O.weigh(q, small_k, small, starts_of(new), kv, full.cpu(), torch.zeros((6, heads_kv, page)), [0, 0], dim ** -0.5)
        assert (np.abs(weights[pages - 6:].cpu().double().numpy() - w) <= tol).all()
    want = O.evict(small_k, small_v, weights[pages - 6:].cpu(), small, kv, 80, 9, 2)
    e = attention.cache_evict(k, v, weights, table.cuda(), ints(kv), budget=80, window=9, sinks=2)
    assert e.kv_lens.tolist() == [80, 80] and e.released.tolist() == [2] and e.freed.tolist() == [pages - 3, pages - 5] + [-1] * 6
    assert torch.equal(k[pages - 6:].cpu(), want[0]) and torch.equal(v[pages - 6:].cpu(), want[1]) and torch.equal(weights[pages - 6:].cpu(), want[2])


def test_lengths_past_what_the_table_names():
    """Lengths up to 2^31 - 1 over tables of a few pages: rows stand past every page, and nothing is read there."""
    from flashgann_amd import attention
    q, kc, vc, table, starts = case(2, [1, 20], [60, 60], 4, 2, 64, 8, BF)
    args = (table.cuda(), ints(starts), ints([MOST, MOST - 3]))
    bounds, scales = torch.zeros((kc.shape[0], 2, 2, 64), dtype=torch.int8, device="cuda"), torch.zeros((kc.shape[0], 2), device="cuda")
    attention.cache_bounds(kc.cuda(), torch.arange(kc.shape[0] * 8, device="cuda"), bounds, scales)
    for first, last in ((0, 1), (2, MOST), (MOST, 5)):
        ids = attention.select_blocks(q.cuda(), bounds, scales, *args, page_size=8, k=20, first_blocks=first, last_blocks=last)
        far = MOST // 8 - last >= 8
        want = [b for b in range(first, 8)] if far and first < 8 else []
        assert ids[0, 0].tolist() == want + [-1] * (20 - len(want))
        out, lse = attention.attend_blocks(q.cuda(), kc.cuda(), vc.cuda(), *args, ids, first_blocks=first, last_blocks=last)
        seen = list(range(8)) if want or first >= 8 or not far else []
        if first == 0 and far:
            # all of the table's pages were selected: what attention over them gives
            o = A.dense(q[:1], kc, vc, table[:1], [0, 1], [64], 0.125)
            o.check(out[:1], lse[:1])
        assert bool(torch.isfinite(lse).all()) == bool(seen)
    w = torch.full((kc.shape[0], 2, 8), -1.0, device="cuda")
    attention.cache_weigh(q.cuda(), kc.cuda(), *args, torch.zeros((21, 4), device="cuda"), w, ints([0, 0]))
    assert bool((w[table.flatten().long()] >= 0).all())
    e = attention.cache_evict(kc.cuda(), vc.cuda(), w, table.cuda(), ints([MOST, -5]), budget=MOST, window=MOST - 7, sinks=7)
    assert e.kv_lens.tolist() == [64, 0] and e.released.tolist() == [0]


def test_nothing_to_do():
    """No tokens, no requests, tables without columns."""
    from flashgann_amd import attention
    q, kc, vc, table, starts = case(2, [2, 3], [60, 60], 4, 2, 64, 8, BF)
    qd, kd, vd = q.cuda(), kc.cuda(), vc.cuda()
    w = torch.full((kc.shape[0], 2, 8), 2.0, device="cuda")
    none = torch.empty((2, 0), dtype=torch.int32, device="cuda")
    ids = torch.zeros((5, 2, 3), dtype=torch.int32, device="cuda")
    out, lse = attention.attend_blocks(qd, kd, vd, none, ints(starts), ints([60, 60]), ids)
    assert not out.any() and bool((lse == -np.inf).all())
    attention.cache_weigh(qd, kd, none, ints(starts), ints([60, 60]), lse, w, ints([0, 0]))
    attention.cache_weigh(qd, kd, none[:0], ints([0]), ints([]), lse, w, ints([]))
    e = attention.cache_evict(kd, vd, w, none, ints([60, 60]), budget=5, window=1)
    assert bool((w == 2).all()) and e.kv_lens.tolist() == [0, 0] and e.freed.shape == (0,) and e.released.tolist() == [0]
    assert attention.attend_blocks(qd[:0], kd, vd, table.cuda(), ints([0, 0, 0]), ints([60, 60]), ids[:0])[0].shape == (0, 4, 64)
    # no new rows: tokens without a weight get 0, the others keep theirs
    attention.cache_weigh(qd[:0], kd, table.cuda(), ints([0, 0, 0]), ints([60, 60]), lse[:0], w, ints([60, 20]))
    flat = w.permute(0, 2, 1)[table.long().cuda()].reshape(2, -1, 2)
    assert bool((flat[0, :60] == 2).all()) and bool((flat[1, :20] == 2).all()) and not flat[1, 20:60].any()


def test_written_tensors_move_their_versions():
    from flashgann_amd import attention
    q, kc, vc, table, starts = case(2, [2, 3], [60, 60], 4, 2, 64, 8, BF)
    kd, vd = kc.cuda(), vc.cuda()
    bounds, scales = torch.zeros((kc.shape[0], 2, 2, 64), dtype=torch.int8, device="cuda"), torch.zeros((kc.shape[0], 2), device="cuda")
    w = torch.zeros((kc.shape[0], 2, 8), device="cuda")
    lse = torch.zeros((5, 4), device="cuda")
    at = [t._version for t in (kd, vd, bounds, scales, w)]
    attention.cache_bounds(kd, torch.arange(8, device="cuda"), bounds, scales)
    attention.cache_weigh(q.cuda(), kd, table.cuda(), ints(starts), ints([60, 60]), lse, w, ints([0, 0]))
    attention.cache_evict(kd, vd, w, table.cuda(), ints([60, 60]), budget=20, window=2)
    assert [t._version - a for t, a in zip((kd, vd, bounds, scales, w), at)] == [1, 1, 1, 1, 2]
