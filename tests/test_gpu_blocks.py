"""Bounds of pages, selection by them and attention over selected pages on the GPU
against the definitions: types, head layouts, page sizes, strides, chunks and single
tokens, ties, rows that have nothing to select, and what hides in masked places."""
from __future__ import annotations

import numpy as np
import pytest
import torch

import attention_oracle as A
import blocks_oracle as O

pytestmark = pytest.mark.gpu

BF, FP = torch.bfloat16, torch.float16
NAN, INF = float("nan"), float("inf")


@pytest.fixture(autouse=True)
def _gpu(gpu_available):
    torch.cuda.set_device(0)


def ints(v):
    return torch.tensor(v, dtype=torch.int32).cuda()


def starts_of(new):
    out = [0]
    for m in new:
        out.append(out[-1] + m)
    return out


def case(seed, new, kv, heads, heads_kv, dim, page, dtype, layout="nhd", spare=3, width=None):
    """CPU tensors of one batch: (q, k_cache, v_cache, table, q_starts)."""
    rng = np.random.default_rng(seed)
    pages = sum(-(-n // page) for n in kv) + spare
    k, v = A.make_cache(rng, pages, page, heads_kv, dim, dtype, layout)
    table = A.make_table(rng, pages, kv, page, width)
    q = torch.from_numpy(rng.standard_normal((sum(new), heads, dim)).astype(np.float32) * 1.5).to(dtype)
    return q, k, v, table, starts_of(new)


def bounds_on_gpu(k, slots, bounds=None, scales=None):
    from flashgann_amd import attention
    pages, page, heads_kv, dim = k.shape
    bounds = torch.full((pages, heads_kv, 2, dim), 77, dtype=torch.int8, device="cuda") if bounds is None else bounds
    scales = torch.full((pages, heads_kv), 5.0, device="cuda") if scales is None else scales
    attention.cache_bounds(k.cuda(), torch.tensor(slots, dtype=torch.int64).cuda(), bounds, scales)
    return bounds, scales


def check_bounds(k, slots):
    pages, page, heads_kv, dim = k.shape
    got, scales = bounds_on_gpu(k, slots)
    got, scales = got.cpu().numpy(), scales.cpu().numpy()
    want = O.bounds(k, O.full_pages(slots, page, pages))
    for p in range(pages):
        for h in range(heads_kv):
            codes, scale = want.get((p, h), (77, 5.0))
            assert scales[p, h] == scale, (p, h)
            assert np.array_equal(got[p, h], np.broadcast_to(codes, (2, dim))), (p, h)


@pytest.mark.parametrize("dtype", (BF, FP))
@pytest.mark.parametrize("dim", (64, 96, 128, 256))
@pytest.mark.parametrize("heads_kv,page,layout", ((2, 16, "nhd"), (3, 24, "hnd"), (1, 1, "nhd"), (5, 7, "nhd"), (2, 64, "hnd"), (1, 300, "nhd")))
def test_bounds(dtype, dim, heads_kv, page, layout):
    """Slots in any order, twice, of no page, past the cache; only full pages are written."""
    rng = np.random.default_rng(dim + page)
    pages = 9
    k, _ = A.make_cache(rng, pages, page, heads_kv, dim, dtype, layout)
    k[2] *= 100.0
    k[3] = 0.0
    k[4, :, 0] = -k[4, :, 0].abs()
    slots = rng.permutation(pages * page)[:max(3, pages * page * 2 // 3)].tolist()
    check_bounds(k, slots + slots[:2] + [-1, pages * page, pages * page + page - 1, 1 << 40, -page - 1])
    check_bounds(k, [page * pages - 1])


@pytest.mark.parametrize("dtype", (BF, FP))
def test_bounds_of_odd_values(dtype):
    """Infinities and NaN mark their page and head alone; the largest, the smallest, values at a scale's end."""
    page, dim = 4, 64
    k, _ = A.make_cache(np.random.default_rng(1), 12, page, 2, dim, dtype)
    k[0, 1, 0, 3], k[1, 0, 1, 9], k[2, 3, 0, 63] = NAN, INF, -INF
    k[3], k[4] = torch.finfo(dtype).max, -torch.finfo(dtype).max
    k[5] = 0
    k[5, 0, 0, 0] = torch.finfo(dtype).smallest_normal
    k[6] = 0
    k[6, 2, 1, 5] = 127.0 if dtype == BF else 127.0 / 64
    k[7] = 0
    k[7, 2, 1, 5] = -127.5 if dtype == BF else -127.5 / 64
    k[8] = 1e-6
    k[9] = torch.finfo(dtype).smallest_normal / 2
    check_bounds(k, list(range(12 * page)))


def test_bounds_strides_and_streams():
    """A cache inside a larger one, written on another stream; no slots at all."""
    from flashgann_amd import attention
    big, _ = A.make_cache(np.random.default_rng(2), 10, 8, 6, 128, BF)
    k = big[1:9, :, 2:5]
    kd = big.cuda()[1:9, :, 2:5]
    slots = torch.arange(64, device="cuda")
    bounds, scales = torch.zeros((8, 3, 2, 128), dtype=torch.int8, device="cuda"), torch.zeros((8, 3), device="cuda")
    attention.cache_bounds(kd, slots[:0], bounds, scales)
    assert not bounds.any()
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        attention.cache_bounds(kd, slots, bounds, scales)
    s.synchronize()
    for (p, h), (codes, scale) in O.bounds(k, range(8)).items():
        assert float(scales[p, h]) == scale and np.array_equal(bounds[p, h].cpu().numpy(), codes)


# ---------------------------------------------------------------- select

def compare_select(new, kv, heads, heads_kv, dim, page, dtype, k, lists, first, last, seed=0, change=None, width=None, q_change=None):
    from flashgann_amd import attention
    q, kc, _, table, starts = case(seed, new, kv, heads, heads_kv, dim, page, dtype, width=width)
    if change:
        change(kc, table)
    if q_change:
        q_change(q)
    bounds, scales = bounds_on_gpu(kc, list(range(kc.shape[0] * page)))
    ids = attention.select_blocks(q.cuda(), bounds, scales, table.cuda(), ints(starts), ints(kv), page_size=page, k=k, lists=lists,
                                  first_blocks=first, last_blocks=last)
    assert ids.dtype == torch.int32 and ids.shape == (sum(new), lists, k)
    want = O.select(q, bounds.cpu(), scales.cpu(), table.numpy(), starts, kv, page, k, lists, first, last)
    got = ids.cpu().numpy()
    assert np.array_equal(got, want), np.argwhere((got != want).any(-1))[:5]


@pytest.mark.parametrize("dtype", (BF, FP))
@pytest.mark.parametrize("dim", (64, 96, 128, 256))
@pytest.mark.parametrize("heads,heads_kv,lists,page", ((8, 2, 2, 16), (3, 3, 3, 24), (7, 1, 7, 4), (40, 2, 2, 8)))
def test_select_single_tokens(dtype, dim, heads, heads_kv, lists, page):
    kv = [1, 2, page, 5 * page, 5 * page + 1, 0, 300, 700]
    compare_select([1] * len(kv), kv, heads, heads_kv, dim, page, dtype, 5, lists, 1, 2)


@pytest.mark.parametrize("first,last,k", ((0, 1, 1), (1, 1, 7), (3, 4, 40), (0, 100, 3), (100, 1, 3), (2, 2, 1000), ((1 << 31) - 1, (1 << 31) - 1, 2)))
def test_select_chunks(first, last, k):
    """Rows of one tile select from different ranges; lists longer than what there is; a request with nothing new."""
    compare_select([1, 0, 3, 40, 17, 130], [9, 77, 3, 190, 217, 131], 8, 2, 64, 4, BF, k, 4, first, last)
    compare_select([33, 16], [900, 16], 6, 2, 64, 8, FP, k, 2, first, last)


@pytest.mark.parametrize("seed", range(4))
def test_select_ties(seed):
    """Pages with the same keys, and queries of zeros: equal scores go to the lower block."""
    def same(kc, table):
        for p in range(kc.shape[0]):
            kc[p] = kc[p % 3]
    compare_select([1, 20], [700, 600], 8, 2, 64, 4, BF, 9, 2, 1, 1, seed, same)
    compare_select([1, 20], [700, 600], 8, 2, 64, 4, BF, 9, 2, 1, 1, seed, None, None, lambda q: q.zero_())
    compare_select([1, 20], [700, 600], 8, 2, 64, 4, FP, 150, 8, 0, 1, seed, same)


def test_select_odd_values():
    """Missing pages, a table too narrow, pages that are not finite, queries that are not, and scores past the largest float."""
    def odd(kc, table):
        table[0, 3], table[0, 9], table[1, 5] = -1, kc.shape[0], 1 << 30
        for b, x in ((4, NAN), (7, INF), (20, -INF)):
            kc[int(table[1, b]), 1, 0, 5] = x
    compare_select([1, 30], [200, 333], 8, 2, 64, 8, BF, 6, 2, 1, 1, 3, odd)
    compare_select([1, 30], [200, 333], 8, 2, 64, 8, BF, 2, 2, 1, 1, 3, odd)
    compare_select([1, 30], [200, 333], 8, 2, 64, 8, BF, 6, 2, 1, 1, 3, odd, 25)

    def odd_q(q):
        q[0, 1, 3], q[4, 6, 0], q[7, 0, 63] = NAN, INF, -INF
    compare_select([1, 30], [200, 333], 8, 2, 64, 8, FP, 6, 2, 1, 1, 4, None, None, odd_q)

    def huge(kc, table):
        kc[::2] *= 2.0 ** 120
    compare_select([1, 30], [200, 333], 8, 2, 64, 8, BF, 6, 2, 1, 1, 5, huge)

    def tiny(kc, table):
        kc *= 2.0 ** -120
    compare_select([1, 30], [200, 333], 8, 2, 64, 8, BF, 6, 2, 1, 1, 5, tiny)


def plain_select(q, bounds, scales, table, starts, kv, page, k, lists, first, last):
    """Many rows at once with whole numbers in 64 bits, on the GPU: requests of equal new lengths."""
    B, T = len(kv), q.shape[0]
    new, heads_kv, dim = T // B, scales.shape[1], q.shape[2]
    per = q.shape[1] // lists
    up = torch.zeros((T, lists, dim), device="cuda")
    down = torch.zeros((T, lists, dim), device="cuda")
    qs = q.cuda().float().view(T, lists, per, dim)
    for h in range(per):
        up, down = up + qs[:, :, h].clamp(min=0), down + qs[:, :, h].clamp(max=0)
    both = torch.cat([up, down], -1).double()
    most = both.abs().amax(-1, keepdim=True)
    powers = torch.tensor([2.0 ** e for e in range(-126, 122)], dtype=torch.float64, device="cuda")
    codes = torch.round(both / powers[torch.searchsorted(127 * powers, most)])
    at = table.cuda().long().clamp(min=0)
    ids = []
    for r in range(B):
        c = codes[r * new:(r + 1) * new].view(new, heads_kv, -1, 2 * dim)
        s = torch.einsum("nhld,bhd->nhlb", c, bounds[at[r]].double().view(-1, heads_kv, 2 * dim)) * scales[at[r]].double().t()[:, None]
        s = s.reshape(new, lists, -1)
        b = torch.arange(s.shape[-1], device="cuda")
        pos = kv[r] - new + torch.arange(new, device="cuda")
        seen = (b >= first) & (b <= (pos // page - last)[:, None])
        s = s.masked_fill(~seen[:, None], -INF)
        best, at_b = s.sort(dim=-1, descending=True, stable=True)
        n = s.shape[-1]
        x = torch.where(best > -INF, at_b, n)
        x = torch.nn.functional.pad(x, (0, max(0, k - n)), value=n)[..., :k].sort(-1).values
        ids.append(torch.where(x < n, x, -1))
    return torch.cat(ids).to(torch.int32)


@pytest.mark.parametrize("new,kv,heads,heads_kv,lists,page,k", (
    (1, [40000], 8, 2, 8, 4, 300),           # few rows over many blocks: made and picked by different workgroups
    (1, [5000] * 40, 8, 4, 4, 4, 64),        # a workgroup a row
    (50, [12000, 9000], 4, 2, 2, 4, 33),     # 8 rows in LDS
    (40, [30000], 4, 2, 2, 2, 4096),         # 2 rows in LDS
    (5, [70000, 66000], 4, 2, 2, 1, 100),    # more blocks than LDS holds
    (1, [150000], 2, 2, 2, 1, 17),
    (1, [150000] * 40, 4, 4, 4, 1, 2),       # scratch, one row each
))
def test_select_long(new, kv, heads, heads_kv, lists, page, k):
    from flashgann_amd import attention
    q, kc, _, table, starts = case(7, [new] * len(kv), [max(kv)] * len(kv) if len(kv) > 10 else kv, heads, heads_kv, 64, page, BF) if len(kv) <= 10 else _shared(new, kv, heads, heads_kv, page)
    bounds, scales = torch.zeros((kc.shape[0], heads_kv, 2, 64), dtype=torch.int8, device="cuda"), torch.zeros((kc.shape[0], heads_kv), device="cuda")
    attention.cache_bounds(kc.cuda(), torch.arange(kc.shape[0] * page, device="cuda"), bounds, scales)
    ids = attention.select_blocks(q.cuda(), bounds, scales, table.cuda(), ints(starts), ints(kv), page_size=page, k=k, lists=lists)
    want = plain_select(q, bounds, scales, table, starts, kv, page, k, lists, 1, 1)
    assert torch.equal(ids, want)


@pytest.mark.parametrize("new,kv,page,k", ((300, 4000, 4, 16), (300, 4000, 4, 32), (300, 4000, 4, 33), (300, 12000, 4, 20), (300, 30000, 4, 20), (300, 60000, 4, 300),
                                           (300, 70000, 2, 9)))
def test_select_tiles_of_rows(new, kv, page, k):
    """Many rows at once: 16 of a tile in LDS, and over longer tables with their keys in memory; few and many to pick."""
    from flashgann_amd import attention
    q, kc, _, table, starts = case(17, [new], [kv], 4, 2, 64, page, BF)
    bounds, scales = torch.zeros((kc.shape[0], 2, 2, 64), dtype=torch.int8, device="cuda"), torch.zeros((kc.shape[0], 2), device="cuda")
    attention.cache_bounds(kc.cuda(), torch.arange(kc.shape[0] * page, device="cuda"), bounds, scales)
    ids = attention.select_blocks(q.cuda(), bounds, scales, table.cuda(), ints(starts), ints([kv]), page_size=page, k=k)
    assert torch.equal(ids, plain_select(q, bounds, scales, table, starts, [kv], page, k, 2, 1, 1))


def test_select_ties_in_tiles_of_rows():
    """Equal scores go to the lower block however rows are picked from: all equal, a few values, infinite ones."""
    def same(n):
        def change(kc, table):
            for p in range(kc.shape[0]):
                kc[p] = kc[p % n]
        return change
    for n, k in ((1, 7), (3, 7), (3, 32), (40, 20), (3, 60)):
        compare_select([300], [700], 4, 2, 64, 4, BF, k, 2, 1, 1, n, same(n))
    compare_select([300], [700], 4, 2, 64, 4, BF, 9, 2, 1, 1, 8, None, None, lambda q: q.zero_())

    def odd(kc, table):
        table[0, 3], table[0, 9] = -1, kc.shape[0]
        for b, x in ((4, NAN), (7, INF), (20, -INF), (33, NAN)):
            kc[int(table[0, b]), 1, 0, 5] = x
    for k in (2, 3, 4, 9):
        compare_select([300], [700], 4, 2, 64, 4, FP, k, 2, 1, 1, 3, odd)


@pytest.mark.parametrize("new,kv,page,k", ((8400, 17000, 8, 16), (3400, 20000, 4, 33), (1700, 20000, 2, 20), (850, 20000, 1, 7), (490, 35000, 1, 9)))
def test_select_more_keys_than_are_kept(new, kv, page, k):
    """More than 1 GB of keys: tiles of 8, 4, 2 rows and one in LDS, and more blocks than it holds, where a workgroup
    takes several rows one after another."""
    from flashgann_amd import attention
    q, kc, _, table, starts = case(18, [new], [kv], 16, 2, 64, page, BF)
    bounds, scales = torch.zeros((kc.shape[0], 2, 2, 64), dtype=torch.int8, device="cuda"), torch.zeros((kc.shape[0], 2), device="cuda")
    attention.cache_bounds(kc.cuda(), torch.arange(kc.shape[0] * page, device="cuda"), bounds, scales)
    ids = attention.select_blocks(q.cuda(), bounds, scales, table.cuda(), ints(starts), ints([kv]), page_size=page, k=k, lists=16)
    for i in range(0, new, 500):  # the rows some at a time, each part as the last of its request
        n = min(500, new - i)
        want = plain_select(q[i:i + n], bounds, scales, table, [0, n], [kv - new + i + n], page, k, 16, 1, 1)
        assert torch.equal(ids[i:i + n], want), i


@pytest.mark.parametrize("new,blocks", ((100, 1000), (100, 1030), (100, 2100), (33, 4000)))
@pytest.mark.parametrize("lists,k", ((2, 16), (8, 64)))
def test_select_few_tiles(new, blocks, lists, k):
    """Few tiles of rows over many blocks, of two requests of different lengths and one without new tokens."""
    compare_select([new, 0, 17], [4 * blocks, 50, 1500], 8, 2, 64, 4, BF, k, lists, 1, 1, 13)


@pytest.mark.parametrize("n,k", ((1, 7), (3, 32), (40, 20), (0, 5)))
def test_select_ties_in_long_tiles_of_rows(n, k):
    """As above over 2,200 and 2,600 blocks: n different pages in turn; 0: queries of zeros."""
    def same(kc, table):
        for p in range(kc.shape[0]):
            kc[p] = kc[p % n]
    compare_select([140], [8800], 8, 2, 64, 4, BF, k, 4, 1, 1, 11, same if n else None, None, None if n else (lambda q: q.zero_()))
    compare_select([130], [5200], 8, 2, 64, 2, FP, k, 4, 1, 1, 12, same if n else None, None, None if n else (lambda q: q.zero_()))


def _shared(new, kv, heads, heads_kv, page):
    """Requests whose tables name the same pages in different orders."""
    rng = np.random.default_rng(8)
    pages = max(-(-n // page) for n in kv)
    k, v = A.make_cache(rng, pages, page, heads_kv, 64, BF)
    table = torch.from_numpy(np.stack([rng.permutation(pages) for _ in kv]).astype(np.int32))
    q = torch.from_numpy(rng.standard_normal((new * len(kv), heads, 64)).astype(np.float32)).to(BF)
    return q, k, v, table, starts_of([new] * len(kv))


def test_select_rows_outside():
    """Rows before the first request and behind the last are left as they were; no rows, no requests."""
    from flashgann_amd import attention
    q, kc, _, table, _ = case(1, [30], [200, 100], 4, 2, 64, 8, BF)
    bounds, scales = bounds_on_gpu(kc, list(range(kc.shape[0] * 8)))
    qd = q.cuda()
    ids = attention.select_blocks(qd, bounds, scales, table.cuda(), ints([4, 20, 25]), ints([200, 100]), page_size=8, k=3)
    for s, e, r in ((4, 20, 0), (20, 25, 1)):
        alone = attention.select_blocks(qd[s:e], bounds, scales, table[r:r + 1].cuda(), ints([0, e - s]), ints([[200, 100][r]]), page_size=8, k=3)
        assert torch.equal(ids[s:e], alone)
    none = attention.select_blocks(qd[:0], bounds, scales, table.cuda(), ints([0, 0, 0]), ints([200, 100]), page_size=8, k=3)
    assert none.shape == (0, 2, 3)
    none = attention.select_blocks(qd, bounds, scales, table[:0].cuda(), ints([0]), ints([]), page_size=8, k=3)
    assert none.shape == (30, 2, 3)


# ---------------------------------------------------------------- attend

def some_ids(rng, new, kv, lists, k, page):
    """Ascending ids of each row and list, -1 behind them; some of them of first or last blocks."""
    ids = np.full((sum(new), lists, k), -1, np.int32)
    t = 0
    for m, n in zip(new, kv):
        for _ in range(m):
            for lst in range(lists):
                have = max(1, -(-n // page))
                some = rng.permutation(have)[:rng.integers(0, k + 1)]
                ids[t, lst, :len(some)] = np.sort(some)
            t += 1
    return torch.from_numpy(ids)


def compare_attend(new, kv, heads, heads_kv, dim, page, dtype, lists, k, first, last, layout="nhd", seed=0, change=None, scale=None, width=None):
    from flashgann_amd import attention
    q, kc, vc, table, starts = case(seed, new, kv, heads, heads_kv, dim, page, dtype, layout, width=width)
    ids = some_ids(np.random.default_rng(seed + 100), new, kv, lists, k, page)
    if change:
        change(q, kc, vc, table, ids)
    out, lse = attention.attend_blocks(q.cuda(), kc.cuda(), vc.cuda(), table.cuda(), ints(starts), ints(kv), ids.cuda(), first_blocks=first,
                                       last_blocks=last, scale=scale)
    assert out.dtype == dtype and lse.dtype == torch.float32
    O.attend(q, kc, vc, table, starts, kv, ids, scale or dim ** -0.5, first, last).check(out, lse)


@pytest.mark.parametrize("dtype", (BF, FP))
@pytest.mark.parametrize("dim", (64, 96, 128, 256))
@pytest.mark.parametrize("heads,heads_kv,lists,page,layout", ((8, 2, 2, 16, "nhd"), (3, 3, 3, 24, "hnd"), (7, 1, 7, 1, "nhd"), (40, 2, 2, 8, "hnd"),
                                                               (20, 1, 1, 5, "nhd")))
def test_attend_single_tokens(dtype, dim, heads, heads_kv, lists, page, layout):
    """One token a request: contexts of one token, around a page, and none at all."""
    kv = [1, 2, page, page + 1, 4 * page, 129, 0, 300]
    compare_attend([1] * len(kv), kv, heads, heads_kv, dim, page, dtype, lists, 6, 1, 2, layout)


@pytest.mark.parametrize("dtype,dim,heads,heads_kv,lists,page", ((BF, 128, 8, 2, 2, 16), (FP, 96, 12, 4, 4, 24), (BF, 64, 7, 7, 7, 5), (FP, 256, 6, 1, 2, 8),
                                                                 (BF, 128, 36, 2, 2, 4)))
@pytest.mark.parametrize("first,last,k", ((0, 1, 3), (1, 2, 5), (0, 1, 0), (3, 40, 2), (50, 1, 4), (2, 3, 60)))
def test_attend_chunks(dtype, dim, heads, heads_kv, lists, page, first, last, k):
    """Rows of a tile with different lists; chunks and single tokens in one batch, a request with nothing new."""
    new, kv = [1, 0, 3, 21, 17, 1], [9, 77, 3, 90, 217, 260]
    layout = "hnd" if page == 24 else "nhd"
    compare_attend(new, kv, heads, heads_kv, dim, page, dtype, lists, k, first, last, layout)
    compare_attend([70, 0, 1, 33], [75, 77, 3, 290], heads, heads_kv, dim, page, dtype, lists, k, first, last, layout, 1)


@pytest.mark.parametrize("page,kv,k,first,last", ((1, 3000, 20, 3, 2), (1, 700, 300, 0, 600), (2, 4000, 5, 900, 1), (8, 9000, 3, 0, 1), (200, 5000, 2, 1, 1), (64, 3000, 4, 0, 2)))
def test_attend_windows_of_blocks(page, kv, k, first, last):
    """Chunks whose blocks are far apart, next to each other over many windows, larger than a tile."""
    compare_attend([30, 9], [kv, kv // 2], 4, 1, 64, page, BF, 2, k, first, last, seed=page)


def test_attend_lists_of_any_order():
    """Ids out of order, twice, negative, past the context and the largest of all: the rule for each, and nothing read out of range."""
    def mess(q, kc, vc, table, ids):
        rng = np.random.default_rng(5)
        ids.copy_(torch.from_numpy(rng.choice(np.array([-5, -1, 0, 1, 2, 3, 3, 5, 8, 9, 12, 30, 90, (1 << 31) - 1], np.int32), ids.shape)))
        ids[3:6] = ids[3:6].sort(-1).values
    for seed in range(3):
        compare_attend([1, 9, 30], [200, 150, 44], 8, 2, 64, 8, BF, 2, 7, 1, 2, seed=seed, change=mess)
        compare_attend([1, 9, 30], [200, 150, 44], 6, 2, 64, 1, FP, 6, 70, 0, 1, seed=seed, change=mess)


def test_attend_missing_pages():
    def gone(q, kc, vc, table, ids):
        table[0, 1], table[0, 5], table[1, :], table[2, 3] = -1, kc.shape[0], -7, 1 << 30
    compare_attend([1, 3, 30], [100, 90, 260], 8, 2, 128, 16, FP, 2, 8, 1, 2, change=gone, width=12)


@pytest.mark.parametrize("heads", (4, 48))
def test_attend_rows_that_see_nothing(heads):
    """More new tokens than tokens: the first rows stand before the context and see nothing."""
    from flashgann_amd import attention
    compare_attend([20, 5, 50], [12, 0, 20], heads, 2, 64, 16, BF, 2, 2, 1, 1)
    q, kc, vc, table, starts = case(1, [20], [12], heads, 2, 64, 16, BF)
    out, lse = attention.attend_blocks(q.cuda(), kc.cuda(), vc.cuda(), table.cuda(), ints(starts), ints([12]), ints(np.zeros((20, 2, 3))))
    assert torch.all(out[:8] == 0) and torch.all(lse[:8] == -np.inf)


@pytest.mark.parametrize("dtype", (BF, FP))
@pytest.mark.parametrize("what", (NAN, INF, -INF))
def test_attend_masked_places_hold_anything(dtype, what):
    """What a row does not see may be infinite or NaN: pages off its list though on its neighbours',
    the end of a page past the context, tokens after the row's own."""
    def odd(q, kc, vc, table, ids):
        used = set(table.flatten().tolist())
        for p in range(kc.shape[0]):
            if p not in used:
                kc[p], vc[p] = what, what
        for r, n in enumerate((100, 333)):
            kc[int(table[r, n // 16]), n % 16:] = what
            vc[int(table[r, n // 16]), n % 16:] = what
            vc[int(table[r, (n - 1) // 16]), (n - 1) % 16, 1, 7] = what
        ids[:, :, :] = -1
        ids[0::3, :, 0], ids[1::3, :, 0] = 3, 2
        vc[int(table[0, 3]), 5, 0, 1], kc[int(table[1, 2]), 3, 1, 9] = what, what
        vc[int(table[1, 3]), 7, 1, 33] = what
    compare_attend([6, 40], [100, 333], 8, 2, 64, 16, dtype, 2, 3, 1, 1, change=odd)
    compare_attend([1, 1], [100, 333], 8, 2, 64, 16, dtype, 2, 3, 1, 1, change=odd)


def test_attend_all_blocks_is_dense():
    """Every block on the list, or all of them last ones: what attend gives, within both's rounding."""
    new, kv = [1, 50], [300, 170]
    q, kc, vc, table, starts = case(9, new, kv, 8, 2, 128, 16, BF)
    from flashgann_amd import attention
    o = A.dense(q, kc, vc, table, starts, kv, 128 ** -0.5)
    args = (q.cuda(), kc.cuda(), vc.cuda(), table.cuda(), ints(starts), ints(kv))
    every = torch.arange(20, dtype=torch.int32).expand(51, 2, 20).contiguous().cuda()
    for ids, first, last in ((every, 0, 1), (every[:, :, :0].contiguous(), 0, 100), (every[:, :, :0].contiguous(), 100, 1)):
        o.check(*attention.attend_blocks(*args, ids, first_blocks=first, last_blocks=last))


@pytest.mark.parametrize("requests,new,kv,heads,heads_kv,lists,page,k,dim", (
    (1, 1, 9000, 8, 2, 2, 16, 200, 128), (1, 1, 9000, 4, 4, 4, 1, 4096, 64), (3, 2, 5000, 8, 1, 1, 64, 30, 256), (1, 40, 3000, 4, 1, 2, 8, 128, 96)))
def test_attend_long(requests, new, kv, heads, heads_kv, lists, page, k, dim):
    """Many pages of few rows: parts joined by a second kernel, lists as long as they may be."""
    compare_attend([new] * requests, [kv - 7 * r for r in range(requests)], heads, heads_kv, dim, page, BF, lists, k, 2, 3)


def test_attend_strides_out_and_rows_outside():
    """q and out inside larger tensors, given outputs, and rows of no request left as they were."""
    from flashgann_amd import attention
    q, kc, vc, table, _ = case(3, [40], [90, 60], 8, 2, 64, 8, BF)
    ids = some_ids(np.random.default_rng(4), [40], [60], 2, 4, 8)
    qd = torch.empty((40, 8, 2, 64), dtype=BF, device="cuda")[:, :, 1]
    qd.copy_(q)
    od, lse = torch.full((40, 16, 64), 3.0, dtype=BF, device="cuda")[:, ::2], torch.full((40, 8), 3.0, device="cuda")
    starts = [5, 20, 33]
    got = attention.attend_blocks(qd, kc.cuda(), vc.cuda(), table.cuda(), ints(starts), ints([90, 60]), ids.cuda(), out=od, lse=lse)
    assert got[0].data_ptr() == od.data_ptr() and got[1].data_ptr() == lse.data_ptr()
    O.attend(q, kc, vc, table, starts, [90, 60], ids, 64 ** -0.5, 1, 1).check(od, lse)
    for rows in (slice(0, 5), slice(33, 40)):
        assert torch.all(od[rows] == 3) and torch.all(lse[rows] == 3)


# ---------------------------------------------------------------- attend, tiles of 32 rows

MANY = [1, 0, 3, 21, 40, 1, 2, 5, 1, 1, 9, 0, 33, 1, 1, 4]
KV = [9, 77, 3, 90, 217, 60, 2, 130, 1, 40, 9, 5, 70, 300, 17, 111]


@pytest.mark.parametrize("dtype,dim,heads,heads_kv,lists,page", ((BF, 128, 16, 8, 8, 16), (FP, 96, 24, 8, 8, 24), (BF, 64, 16, 2, 16, 5), (FP, 128, 32, 8, 8, 4), (BF, 96, 8, 8, 8, 1)))
@pytest.mark.parametrize("first,last,k", ((0, 1, 3), (1, 2, 5), (0, 1, 0), (3, 40, 2), (50, 1, 4), (2, 3, 60)))
def test_attend_many_requests(dtype, dim, heads, heads_kv, lists, page, first, last, k):
    """Chunks, drafts and single tokens of many requests in one batch."""
    compare_attend(MANY, KV, heads, heads_kv, dim, page, dtype, lists, k, first, last, "hnd" if page == 24 else "nhd", page)


def test_attend_many_heads_of_a_list():
    """More query heads of a list than a tile has rows."""
    compare_attend(MANY * 2, KV * 2, 80, 2, 64, 8, BF, 2, 4, 1, 2)


@pytest.mark.parametrize("page,kv,k,first,last", ((1, 2500, 20, 3, 2), (1, 700, 300, 0, 600), (2, 4000, 5, 900, 1), (8, 9000, 3, 0, 1), (200, 5000, 2, 1, 1), (64, 3000, 4, 0, 2)))
def test_attend_many_windows_of_blocks(page, kv, k, first, last):
    """Blocks far apart, next to each other over several windows, larger than a tile."""
    compare_attend([5] + [2] * 7 + [9], [kv - 11 * r for r in range(9)], 16, 16, 64, page, BF, 16, k, first, last, seed=page)


@pytest.mark.parametrize("dtype", (BF, FP))
def test_attend_many_odd_lists_and_values(dtype):
    """Ids out of order, pages missing, infinities and NaN where only some rows see them."""
    def mess(q, kc, vc, table, ids):
        rng = np.random.default_rng(5)
        ids.copy_(torch.from_numpy(rng.choice(np.array([-5, -1, 0, 1, 2, 3, 3, 5, 8, 9, 12, 30, 90, (1 << 31) - 1], np.int32), ids.shape)))
        ids[3:30] = ids[3:30].sort(-1).values
    compare_attend(MANY, KV, 16, 8, 64, 8, dtype, 8, 7, 1, 2, seed=1, change=mess)

    def gone(q, kc, vc, table, ids):
        table[0, 1], table[4, 5], table[3, :], table[12, 3] = -1, kc.shape[0], -7, 1 << 30
    compare_attend(MANY, KV, 16, 8, 128, 8, dtype, 8, 8, 1, 2, change=gone, width=30)

    for what in (NAN, INF, -INF):
        def odd(q, kc, vc, table, ids):
            used = set(table.flatten().tolist())
            for p in range(kc.shape[0]):
                if p not in used:
                    kc[p], vc[p] = what, what
            for r in (3, 4, 7, 12):
                n = KV[r]
                if n % 8:
                    kc[int(table[r, n // 8]), n % 8:] = what
                    vc[int(table[r, n // 8]), n % 8:] = what
                vc[int(table[r, (n - 1) // 8]), (n - 1) % 8, 1, 7] = what
                vc[int(table[r, 3]), 5, 0, 33], kc[int(table[r, 2]), 3, 1, 9] = what, what
            ids[:, :, :] = -1
            ids[0::3, :, 0], ids[1::3, :, 0] = 3, 2
        compare_attend(MANY, KV, 16, 8, 64, 8, dtype, 8, 3, 1, 1, change=odd)
