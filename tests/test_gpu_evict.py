"""Drawn weights and eviction on the GPU against the definitions."""
from __future__ import annotations

import numpy as np
import pytest
import torch

import attention_oracle as A
import blocks_oracle as O
from test_gpu_blocks import case, ints, starts_of

pytestmark = pytest.mark.gpu

BF, FP = torch.bfloat16, torch.float16
NAN, INF = float("nan"), float("inf")


@pytest.fixture(autouse=True)
def _gpu(gpu_available):
    torch.cuda.set_device(0)


# ---------------------------------------------------------------- weights

def compare_weigh(new, kv, heads, heads_kv, dim, page, dtype, known, layout="nhd", seed=0, change=None, width=None, scale=None):
    from flashgann_amd import attention
    q, kc, vc, table, starts = case(seed, new, kv, heads, heads_kv, dim, page, dtype, layout, width=width)
    rng = np.random.default_rng(seed + 50)
    weights = torch.from_numpy(rng.random((kc.shape[0], heads_kv, page), np.float32) * 3)
    o = A.dense(q, kc, vc, table, starts, kv, scale or dim ** -0.5)
    lse = torch.from_numpy(o.lse.astype(np.float32))
    if change:
        change(q, kc, table, lse)
    want, tol = O.weigh(q, kc, table, starts, kv, lse, weights, known, scale or dim ** -0.5)
    wd = weights.cuda()
    attention.cache_weigh(q.cuda(), kc.cuda(), table.cuda(), ints(starts), ints(kv), lse.cuda(), wd, ints(known), scale=scale)
    got = wd.double().cpu().numpy()
    fine = np.isfinite(want)
    assert np.array_equal(np.isnan(got), np.isnan(want)) and np.array_equal(got[~fine & ~np.isnan(want)], want[~fine & ~np.isnan(want)])
    off = np.abs(got - want)[fine] - tol[fine]
    assert (off <= 0).all(), (off.max(), np.argwhere(fine)[off > 0][:5])


@pytest.mark.parametrize("dtype", (BF, FP))
@pytest.mark.parametrize("dim", (64, 96, 128, 256))
@pytest.mark.parametrize("heads,heads_kv,page,layout", ((8, 2, 16, "nhd"), (3, 3, 24, "hnd"), (7, 1, 1, "nhd"), (40, 2, 64, "hnd")))
def test_weigh_single_tokens(dtype, dim, heads, heads_kv, page, layout):
    """One token a request; its own weight begins with it, the others' go on."""
    kv = [1, 2, 63, 64, 65, 129, 0, 300]
    compare_weigh([1] * len(kv), kv, heads, heads_kv, dim, page, dtype, [n - 1 for n in kv], layout)


@pytest.mark.parametrize("dtype,dim,heads,heads_kv,page", ((BF, 128, 8, 2, 16), (FP, 96, 12, 4, 24), (BF, 64, 7, 7, 5), (FP, 256, 6, 1, 32)))
def test_weigh_chunks(dtype, dim, heads, heads_kv, page):
    """All of a context new, its last rows only, nothing new, known more and less than the rows' first position."""
    new, kv = [1, 0, 3, 90, 17, 70], [9, 77, 3, 90, 257, 270]
    for known in ([0] * 6, [8, 70, 0, 0, 240, 200], [-3, 100, 3, 50, 257, 1 << 30]):
        compare_weigh(new, kv, heads, heads_kv, dim, page, dtype, known)


def test_weigh_odd_values():
    """Keys that are not finite stay with their own token; rows of lse -infinity add nothing; missing pages have no weight."""
    def odd(q, kc, table, lse):
        kc[int(table[0, 2]), 1, 0, 3], kc[int(table[1, 1]), 7, 1, 0], kc[int(table[1, 3]), 2, 0, 5] = NAN, INF, -INF
        table[0, 1], table[1, 5] = -1, kc.shape[0]
        lse[3], lse[20, 2] = -INF, -INF
    compare_weigh([1, 30], [100, 190], 8, 2, 64, 16, BF, [99, 100], change=odd)
    compare_weigh([1, 30], [100, 190], 8, 2, 64, 16, BF, [99, 100], change=odd, width=9)
    compare_weigh([20, 5], [12, 0], 8, 2, 64, 16, FP, [0, 0])


def test_weigh_far_positions_and_many_rows():
    """Tiles far into a context, a row at a time and hundreds of rows."""
    compare_weigh([1], [3000], 2, 1, 64, 16, BF, [2999])
    compare_weigh([150], [700], 4, 2, 64, 8, BF, [300])


def test_weigh_of_everything_sums_to_the_rows():
    """Each row's weights sum to 1, so all weights do to rows times heads, and shared pages add up."""
    from flashgann_amd import attention
    new, kv, heads = [300, 40], [5000, 3000], 8
    q, kc, vc, table, starts = case(3, new, kv, heads, 2, 128, 16, BF)
    args = (q.cuda(), kc.cuda())
    rest = (table.cuda(), ints(starts), ints(kv))
    lse = attention.attend(args[0], args[1], vc.cuda(), *rest, max_q=300)[1]
    weights = torch.zeros((kc.shape[0], 2, 16), device="cuda")
    attention.cache_weigh(*args, *rest, lse, weights, ints([0, 0]))
    # per row: 5,000 weights, each off by its score's error (128 products in 32 bits) and lse's
    assert abs(float(weights.double().sum()) / (340 * heads) - 1) < 1e-4
    once = weights.clone()
    attention.cache_weigh(*args, *rest, lse, weights, ints([5000, 3000]))
    # the same weights twice: one addition
    assert torch.allclose(weights, 2 * once, rtol=2.0 ** -22, atol=0)
    both = torch.zeros_like(weights)
    twice = table[:1].repeat(2, 1).contiguous().cuda()
    attention.cache_weigh(args[0][:300].repeat(2, 1, 1).contiguous(), args[1], twice, ints([0, 300, 600]), ints([5000, 5000]), lse[:300].repeat(2, 1), both, ints([5000, 5000]))
    first = torch.zeros_like(weights)
    attention.cache_weigh(args[0][:300], args[1], table[:1].cuda(), ints([0, 300]), ints([5000]), lse[:300].contiguous(), first, ints([0]))
    assert torch.equal(both, 2 * first)


# ---------------------------------------------------------------- eviction

def compare_evict(kv, heads_kv, dim, page, dtype, budget, window, sinks, layout="nhd", seed=0, change=None, width=None):
    from flashgann_amd import attention
    rng = np.random.default_rng(seed)
    pages = sum(-(-max(n, 0) // page) for n in kv) + 3
    k, v = A.make_cache(rng, pages, page, heads_kv, dim, dtype, layout)
    table = A.make_table(rng, pages, [max(n, 0) for n in kv], page, width)
    w = torch.from_numpy(np.exp(2 * rng.standard_normal((pages, heads_kv, page))).astype(np.float32))
    w[torch.from_numpy(rng.random(w.shape) < 0.3)] = 0.0
    if change:
        change(w, table)
    want = O.evict(k, v, w, table, kv, budget, window, sinks)
    kd, vd, wd, td = k.cuda(), v.cuda(), w.cuda(), table.cuda()
    e = attention.cache_evict(kd, vd, wd, td, ints(kv), budget=budget, window=window, sinks=sinks)
    assert torch.equal(td.cpu(), table)
    for name, a, b in (("k", kd, want[0]), ("v", vd, want[1]), ("weights", wd, want[2])):
        a = a.cpu()
        assert torch.equal(torch.nan_to_num(a, nan=7777.0), torch.nan_to_num(b, nan=7777.0)), (name, torch.nonzero((a != b).reshape(a.shape[0], -1).any(1))[:5])
    assert e.kv_lens.tolist() == want[3] and e.freed.tolist() == want[4] and e.released.tolist() == [want[5]]
    return e


@pytest.mark.parametrize("dtype", (BF, FP))
@pytest.mark.parametrize("dim", (64, 96, 128, 256))
@pytest.mark.parametrize("heads_kv,page,layout", ((2, 16, "nhd"), (3, 24, "hnd"), (1, 1, "nhd"), (5, 7, "nhd")))
def test_evict(dtype, dim, heads_kv, page, layout):
    """Requests below, at and past the budget, by one and by far."""
    compare_evict([0, 1, 39, 40, 41, 47, 200, 130], heads_kv, dim, page, dtype, 40, 9, 3, layout)


@pytest.mark.parametrize("budget,window,sinks", ((1, 0, 0), (1, 1, 0), (1, 0, 1), (10, 10, 0), (10, 0, 10), (10, 5, 5), (50, 0, 0), (64, 33, 1), (150, 100, 7), (500, 3, 3)))
def test_evict_shares(budget, window, sinks):
    compare_evict([300, budget + 1, budget, budget + 2 * window + 1], 2, 64, 8, BF, budget, window, sinks)


def test_evict_window_over_itself():
    """A window much longer than what goes: its places overlap, over many steps of a move."""
    for n in (901, 907, 1200, 1500, 2000):
        compare_evict([n], 2, 64, 16, FP, 900, 800, 2, seed=n)


def test_evict_odd_weights():
    """Ties, all equal, infinities, NaN, zeros of both signs, negative weights; a table that names no page here and there."""
    for seed, change in enumerate((lambda w, t: w.fill_(2.0), lambda w, t: w.copy_((w * 2).floor()), lambda w, t: w.zero_(),
                                   lambda w, t: w.mul_(torch.where(w > 1, 1.0, -1.0)))):
        compare_evict([200, 90], 2, 64, 8, BF, 50, 7, 2, seed=seed, change=change)

    def odd(w, t):
        w.view(-1)[::7], w.view(-1)[1::11], w.view(-1)[2::13], w.view(-1)[3::17] = NAN, INF, -INF, -0.0
        w.view(torch.int32).view(-1)[4::19] = -1  # a NaN with a sign
        t[0, 3], t[0, 20], t[1, 0] = -1, w.shape[0], 1 << 30
    compare_evict([200, 90], 2, 64, 8, BF, 50, 7, 2, seed=9, change=odd)
    compare_evict([200, 90], 2, 64, 8, BF, 5, 2, 0, seed=9, change=odd)


def test_evict_table_narrower_than_a_request():
    compare_evict([200, 90, 30], 2, 64, 8, BF, 50, 7, 2, width=15)
    compare_evict([200, -5], 2, 64, 8, BF, 50, 7, 2, width=5)


@pytest.mark.parametrize("kv,budget,page", (([9000, 300, 8200], 1000, 16), ([40000, 33000], 2000, 64)))
def test_evict_long(kv, budget, page):
    """Weights in LDS and past what it holds."""
    compare_evict(kv, 2, 64, page, BF, budget, 100, 4)


def test_evict_many_requests():
    rng = np.random.default_rng(4)
    compare_evict(rng.integers(0, 30, 1500).tolist(), 1, 64, 4, BF, 12, 3, 1)


def test_evict_again_and_again():
    """Step by step: the same as the definition applied step by step."""
    from flashgann_amd import attention
    rng = np.random.default_rng(6)
    k, v = A.make_cache(rng, 30, 8, 2, 64, BF)
    w = torch.from_numpy(rng.random((30, 2, 8), np.float32))
    table = A.make_table(rng, 30, [100, 90], 8)
    kd, vd, wd, td = k.cuda(), v.cuda(), w.cuda(), table.cuda()
    for n in ([100, 90], [90, 90], [89, 60], [60, 61]):
        budget = min(n) - 5
        k, v, w, lens, _, _ = O.evict(k, v, w, table, n, budget, 6, 2)
        e = attention.cache_evict(kd, vd, wd, td, ints(n), budget=budget, window=6, sinks=2)
        assert e.kv_lens.tolist() == lens and torch.equal(kd.cpu(), k) and torch.equal(vd.cpu(), v) and torch.equal(wd.cpu(), w)
