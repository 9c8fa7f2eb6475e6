"""The attention kernels where a workgroup walks an item's tokens for long and where
many rows are joined: what large batches and long chunks reach.  The sizes are checked
on the host to give such pieces; a few rows of each request are held against the
64-bit oracle."""
from __future__ import annotations

import numpy as np
import pytest
import torch
from threadpoolctl import threadpool_limits

import attention_oracle as A
import attention_split as S

pytestmark = pytest.mark.gpu

BF, FP = torch.bfloat16, torch.float16
PAGE, PAGES = 16, 200  # of the requests together: each names all of them, in an order of its own
REQUESTS = 70


@pytest.fixture(autouse=True)
def _gpu(gpu_available):
    torch.cuda.set_device(0)
    with threadpool_limits(1):  # the oracle's products are small: threads cost more than they bring
        yield


def ints(x):
    return torch.tensor(x, dtype=torch.int32).cuda()


class Batch:
    """Requests over shared pages.  Every third has a page of its own at its end: infinite values in the last token
    but one, NaN past the last; every fourth lacks a page past the first thousand tokens."""

    def __init__(self, seed, new, kv, heads, heads_kv, dim, dtype):
        self.rng = rng = np.random.default_rng(seed)
        self.new, self.kv, self.dim = new, kv, dim
        self.k, self.v = A.make_cache(rng, PAGES + REQUESTS, PAGE, heads_kv, dim, dtype)
        self.table = torch.from_numpy(np.stack([rng.permutation(PAGES) for _ in kv]).astype(np.int32))
        for r, n in enumerate(kv):
            if r % 4 == 1 and n > 1400:
                self.table[r, 1100 // PAGE + r % 9] = -1
            if r % 3 == 0 and n > 1 and n % PAGE != 1:
                last, off = PAGES + r, (n - 1) % PAGE
                self.table[r, (n - 1) // PAGE] = last
                self.k[last, off + 1:], self.v[last, off + 1:] = float("nan"), float("nan")
                if new[r] > 2:
                    self.v[last, off - 1, 0, 3] = float("inf")
        self.starts = [0, *np.cumsum(new).tolist()]
        self.q = torch.from_numpy(rng.standard_normal((self.starts[-1], heads, dim)).astype(np.float32)).to(dtype)
        self.on = [t.cuda() for t in (self.q, self.k, self.v, self.table)]

    def check_dense(self, out, lse, window, sinks):
        o = A.Oracle(self.q, self.k, self.v, self.table, self.dim ** -0.5)
        for r, (m, n) in enumerate(zip(self.new, self.kv)):
            for i in {0, int(self.rng.integers(m)), m - 1} if m else ():
                tokens = A.seen_tokens(o.table, r, n, n - m + i, PAGE, o.pages, window, sinks)
                for h in range(self.q.shape[1]):
                    o.row(self.starts[r] + i, h, r, tokens)
        o.check(out, lse)


def lengths(seed, most_new, lo=1500, hi=3000):
    """70 requests, some of them empty or with nothing new."""
    rng = np.random.default_rng(seed)
    kv = rng.integers(lo, hi, REQUESTS)
    new = rng.integers(1, most_new + 1, REQUESTS)
    new[[3, 40]], kv[[10, 41]], new[[10, 41]] = 0, 0, 0
    kv[50], new[50] = 37, min(20, most_new)
    return new.tolist(), kv.tolist()


@pytest.mark.parametrize("dim,dtype,window,sinks", ((64, BF, None, 0), (64, FP, 1500, 20), (96, FP, None, 0), (96, BF, 1300, 1), (128, BF, None, 0),
                                                    (128, FP, 1500, 20), (256, FP, None, 0), (256, BF, 1300, 5)))
def test_long_pieces_of_tiles(dim, dtype, window, sinks):
    from flashgann_amd import attention
    heads, heads_kv = 16, 4
    new, kv = lengths(dim, 40)
    new[7], kv[7] = 300, 2900
    rows, tile = (128, 32) if dim == 256 else (256, 64)
    ps = S.pieces(new, kv, heads // heads_kv, heads_kv, rows, window=window, sinks=sinks, **S.TILES)
    long = [p for p in ps if p.t_hi - p.t_lo > 20 * tile]  # past the ring of 16 tiles' places
    assert len(long) > 20 and any(p.rows > rows - 32 for p in long) and any(p.rows <= rows - 32 for p in long)
    assert S.joined_rows(ps) > 2048
    b = Batch(dim, new, kv, heads, heads_kv, dim, dtype)
    out, lse = attention.attend(*b.on, ints(b.starts), ints(kv), max_q=max(new), window=window, sinks=sinks)
    b.check_dense(out, lse, window, sinks)


@pytest.mark.parametrize("dim,dtype,window,sinks", ((64, FP, None, 0), (96, BF, None, 0), (128, BF, None, 0), (128, FP, 1900, 20), (256, FP, None, 0)))
def test_long_pieces_of_few_rows(dim, dtype, window, sinks):
    from flashgann_amd import attention
    heads, heads_kv = 32, 8
    new, kv = lengths(dim + 1, 4)
    ps = S.pieces(new, kv, heads // heads_kv, heads_kv, 16, window=window, sinks=sinks, **S.FEW)
    assert len([p for p in ps if p.t_hi - p.t_lo > 1300]) > 20 and S.joined_rows(ps) > 512  # past 1,024 places, joined by rows
    b = Batch(dim + 1, new, kv, heads, heads_kv, dim, dtype)
    out, lse = attention.attend(*b.on, ints(b.starts), ints(kv), max_q=4, window=window, sinks=sinks)
    b.check_dense(out, lse, window, sinks)


@pytest.mark.parametrize("dim,dtype,lists", ((64, BF, 16), (96, FP, 8), (128, BF, 8), (256, FP, 8)))
def test_long_pieces_of_retrieved(dim, dtype, lists):
    from flashgann_amd import attention
    heads, heads_kv, K, window, sinks = 32, 8, 700, 900, 10
    _, kv = lengths(dim + 2, 1)
    new = [1] * REQUESTS
    ps = S.pieces(new, kv, heads // lists, lists, 16, window=window, sinks=sinks, ids=K, **S.FEW)
    assert len([p for p in ps if p.t_hi - p.t_lo > 1200]) > 20 and S.joined_rows(ps) > 512
    b = Batch(dim + 2, new, kv, heads, heads_kv, dim, dtype)
    ids = np.stack([np.stack([b.rng.permutation(max(n, K) + 50)[:K] for _ in range(lists)]) for n in kv]).astype(np.int32)
    ids[:, ::2, K - 100:] = ids[:, ::2, K - 101:K - 100]  # a short beam's repeats
    ids[:, 1, 5] = -1
    out, lse = attention.attend_retrieved(*b.on, ints(kv), torch.from_numpy(ids).cuda(), window=window, sinks=sinks)
    some = sorted({0, 1, 10, 50, *b.rng.permutation(REQUESTS)[:20].tolist()})
    want = A.retrieved(b.q[some], b.k, b.v, b.table[some], [kv[r] for r in some], ids[some], dim ** -0.5, window, sinks)
    want.check(out[some], lse[some])


@pytest.mark.parametrize("dim,dtype", ((64, BF), (96, FP), (128, BF), (256, FP)))
def test_graph_replays_with_joins(dim, dtype):
    """Captured calls of every kernel follow the lengths in device memory: replayed over other lengths, with eager
    work between, the bits are those of the same calls made eagerly."""
    from flashgann_amd import attention
    heads, heads_kv, K = 16, 4, 300
    new, kv = lengths(dim + 3, 30)
    b = Batch(dim + 3, new, kv, heads, heads_kv, dim, dtype)
    q, k, v, table = b.on
    starts, lens = ints(b.starts), ints(kv)
    few = q[:REQUESTS]
    ids = torch.from_numpy(np.stack([b.rng.permutation(2000)[:K] for _ in range(REQUESTS * heads_kv)]).astype(np.int32)).view(REQUESTS, heads_kv, K).cuda()
    one = torch.arange(REQUESTS + 1, dtype=torch.int32).cuda()

    def step():
        return (*attention.attend(q, k, v, table, starts, lens, max_q=30), *attention.attend(few, k, v, table, one, lens, max_q=1),
                *attention.attend_retrieved(few, k, v, table, lens, ids, window=800, sinks=7))

    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        step()
    side.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = step()
    for i in range(4):
        lens.copy_(ints([max(n - 211 * i * (r % 3), 0) for r, n in enumerate(kv)]))
        graph.replay()
        torch.cuda.synchronize()
        want = step()
        for x, y in zip(got, want):
            assert torch.equal(x.view(torch.int32 if x.dtype == torch.float32 else torch.int16), y.view(torch.int32 if y.dtype == torch.float32 else torch.int16)), i
