"""The paged cache and its attention on the GPU against the 64-bit oracle: types,
head layouts, lengths from nothing to thousands, odd page sizes, strides, masks
that leave a row empty, and what hides in masked places."""
from __future__ import annotations

import numpy as np
import pytest
import torch

import attention_oracle as A

pytestmark = pytest.mark.gpu

BF, FP = torch.bfloat16, torch.float16


@pytest.fixture(autouse=True)
def _gpu(gpu_available):
    torch.cuda.set_device(0)


def dev(*ts):
    return [t.cuda() for t in ts]


def case(seed, new, kv, heads, heads_kv, dim, page, dtype, layout="nhd", spare=3, width=None):
    """CPU tensors of one batch: (q, k_cache, v_cache, table, q_starts)."""
    rng = np.random.default_rng(seed)
    pages = sum(-(-n // page) for n in kv) + spare
    k, v = A.make_cache(rng, pages, page, heads_kv, dim, dtype, layout)
    table = A.make_table(rng, pages, kv, page, width)
    q = torch.from_numpy(rng.standard_normal((sum(new), heads, dim)).astype(np.float32) * 1.5).to(dtype)
    starts = [0]
    for m in new:
        starts.append(starts[-1] + m)
    return q, k, v, table, starts


def run(q, k, v, table, starts, kv, **kw):
    from flashgann_amd import attention
    new = [b - a for a, b in zip(starts, starts[1:])]
    kw.setdefault("max_q", max(new))
    qd, kd, vd, td = dev(q, k, v, table)
    return attention.attend(qd, kd, vd, td, torch.tensor(starts, dtype=torch.int32).cuda(),
                            torch.tensor(kv, dtype=torch.int32).cuda(), **kw)


def compare(new, kv, heads, heads_kv, dim, page, dtype, layout="nhd", window=None, sinks=0, seed=0, scale=None, **kw):
    q, k, v, table, starts = case(seed, new, kv, heads, heads_kv, dim, page, dtype, layout)
    out, lse = run(q, k, v, table, starts, kv, window=window, sinks=sinks, scale=scale, **kw)
    assert out.dtype == dtype and lse.dtype == torch.float32
    A.dense(q, k, v, table, starts, kv, scale or dim ** -0.5, window, sinks).check(out, lse)


# ---------------------------------------------------------------- attend

@pytest.mark.parametrize("dtype", (BF, FP))
@pytest.mark.parametrize("dim", (64, 96, 128, 256))
@pytest.mark.parametrize("heads,heads_kv,page,layout", ((8, 2, 16, "nhd"), (3, 3, 24, "hnd"), (7, 1, 1, "nhd"), (40, 2, 64, "hnd")))
def test_single_tokens(dtype, dim, heads, heads_kv, page, layout):
    """One token a request: contexts of one token, around a tile and a unit, and none at all."""
    kv = [1, 2, 31, 32, 33, 129, 0, 300]
    compare([1] * len(kv), kv, heads, heads_kv, dim, page, dtype, layout)


@pytest.mark.parametrize("dtype,dim,heads,heads_kv,page", ((BF, 128, 8, 2, 16), (FP, 96, 12, 4, 24), (BF, 64, 7, 7, 5),
                                                           (FP, 256, 6, 1, 32), (BF, 128, 36, 2, 64)))
@pytest.mark.parametrize("window,sinks", ((None, 0), (1, 0), (13, 3), (64, 4), (500, 100), (5, 200)))
def test_chunks(dtype, dim, heads, heads_kv, page, window, sinks):
    """Chunks and single tokens in one batch, a request with nothing new, one whose whole context is new."""
    new, kv = [1, 0, 3, 40, 17, 130, 1], [9, 77, 3, 90, 217, 131, 260]
    compare(new, kv, heads, heads_kv, dim, page, dtype, "hnd" if page == 24 else "nhd", window, sinks)


@pytest.mark.parametrize("max_q", (0, 1, 5, 1000))
def test_max_q_is_a_hint(max_q):
    compare([3, 70, 1], [50, 200, 90], 8, 2, 128, 16, BF, max_q=max_q)
    compare([3, 70, 1], [50, 200, 90], 8, 2, 128, 16, BF, max_q=max_q, window=20, sinks=2)


@pytest.mark.parametrize("heads", (4, 96))
def test_rows_that_see_nothing(heads):
    """More new tokens than tokens: the first rows stand before the context and see nothing."""
    new, kv = [20, 5, 150], [12, 0, 20]
    q, k, v, table, starts = case(1, new, kv, heads, 2, 64, 16, BF)
    out, lse = run(q, k, v, table, starts, kv)
    assert torch.all(out[:8] == 0) and torch.all(lse[:8] == -np.inf) and torch.all(lse[20:25] == -np.inf)
    A.dense(q, k, v, table, starts, kv, 64 ** -0.5).check(out, lse)


@pytest.mark.parametrize("new", ([1, 1, 1], [3, 1, 2], [60, 70, 150]))
def test_missing_pages(new):
    """Page ids below zero and past the cache, a table too narrow: those tokens are invisible."""
    kv = [100, 90, 260]
    q, k, v, table, starts = case(2, new, kv, 8, 2, 128, 16, FP)
    table[0, 1], table[0, 5], table[1, :], table[2, 3] = -1, k.shape[0], -7, 1 << 30
    table = table[:, :12].contiguous()
    out, lse = run(q, k, v, table, starts, kv)
    o = A.dense(q, k, v, table, starts, kv, 128 ** -0.5)
    o.check(out, lse)
    assert torch.all(lse[starts[1]:starts[2]] == -np.inf)


@pytest.mark.parametrize("dtype", (BF, FP))
@pytest.mark.parametrize("new", ([5, 1], [90, 200], [2, 3]))
@pytest.mark.parametrize("what", (float("nan"), float("inf"), -float("inf")))
def test_masked_places_hold_anything(dtype, new, what):
    """Keys and values that a row can't see may be infinite or NaN: pages of nobody, the end of a page past
    the context, tokens after the row's own, tokens between the first ones and the window."""
    kv = [100, 333]
    q, k, v, table, starts = case(3, new, kv, 8, 2, 128, 16, dtype)
    used = set(table.flatten().tolist())
    for p in range(k.shape[0]):
        if p not in used:
            k[p], v[p] = what, what
    for r, n in enumerate(kv):
        k[int(table[r, n // 16]) if n % 16 else 0, n % 16 or 16:] = what
        v[int(table[r, n // 16]) if n % 16 else 0, n % 16 or 16:] = what
    for r, n in enumerate(kv):  # the last token: only its own row sees it
        k[int(table[r, (n - 1) // 16]), (n - 1) % 16, 1, 7] = what
        v[int(table[r, (n - 1) // 16]), (n - 1) % 16, 0, 3] = what
    out, lse = run(q, k, v, table, starts, kv)
    first = np.array([t for r in range(2) for t in range(starts[r], starts[r + 1] - 1)], np.int64)
    assert torch.isfinite(out[torch.from_numpy(first).cuda()].float()).all() and torch.isfinite(lse[torch.from_numpy(first).cuda()]).all()
    A_o = A.dense(q, k, v, table, starts, kv, 128 ** -0.5)
    A_o.rows[[starts[1] - 1, starts[2] - 1]] = False
    A_o.check(out, lse)
    # the rows that see it carry it: head 0's values, nothing else of them
    last = out[[starts[1] - 1, starts[2] - 1]].float().cpu()
    assert not torch.isfinite(last[:, :4, 3]).any() and torch.isfinite(last[:, :4, 4:]).all()
    # and with a window the token between goes unseen
    k2, v2 = k.clone(), v.clone()
    k2[int(table[1, 2]), 3], v2[int(table[1, 2]), 3] = what, what
    out, lse = run(q, k2, v2, table, starts, kv, window=9, sinks=4)
    o = A.dense(q, k2, v2, table, starts, kv, 128 ** -0.5, 9, 4)
    o.rows[[starts[1] - 1, starts[2] - 1]] = False
    far = [t for t in range(starts[1], starts[2]) if kv[1] - new[1] + (t - starts[1]) - 9 < 35 <= kv[1] - new[1] + (t - starts[1])]
    o.rows[far] = False
    o.check(out, lse)


@pytest.mark.parametrize("new", ([1, 1], [70, 90]))
def test_large_scores(new):
    """Scores in the thousands, of either sign: one token takes all the weight."""
    kv = [200, 300]
    q, k, v, table, starts = case(4, new, kv, 4, 2, 64, 16, BF)
    out, lse = run(q, k, v, table, starts, kv, scale=80.0)
    A.dense(q, k, v, table, starts, kv, 80.0).check(out, lse)
    q2 = -q.abs()
    out, lse = run(q2, k.abs(), v, table, starts, kv, scale=30.0)
    A.dense(q2, k.abs(), v, table, starts, kv, 30.0).check(out, lse)


@pytest.mark.parametrize("new", ([1, 1, 1], [4, 33, 140]))
def test_strides(new):
    """q out of a packed product, out into a wider buffer, tables and caches inside larger ones."""
    from flashgann_amd import attention
    kv, heads, heads_kv, dim, page = [40, 75, 300], 8, 2, 128, 16
    q, k, v, table, starts = case(5, new, kv, heads, heads_kv, dim, page, BF)
    T = q.shape[0]
    packed = torch.zeros((T, heads + 4, dim), dtype=BF)
    packed[:, 2:2 + heads] = q
    wide = torch.full((T, heads * dim + 64), 7.0, dtype=BF).cuda()
    out = wide[:, 64:].view(T, heads, dim)
    table2 = torch.full((3, table.shape[1] + 5), 12345, dtype=torch.int32)
    table2[:, :table.shape[1]] = table
    both = torch.stack([k, v], 1).cuda()  # (pages, 2, page, heads_kv, dim)
    got, lse = attention.attend(packed.cuda()[:, 2:2 + heads], both[:, 0], both[:, 1], table2.cuda()[:, :table.shape[1]],
                                torch.tensor(starts, dtype=torch.int32).cuda(), torch.tensor(kv, dtype=torch.int32).cuda(),
                                max_q=max(new), out=out)
    assert got.data_ptr() == out.data_ptr() and torch.all(wide[:, :64] == 7.0)
    A.dense(q, k, v, table, starts, kv, dim ** -0.5).check(got, lse)


@pytest.mark.parametrize("heads,heads_kv,dim,dtype", ((16, 2, 128, FP), (5, 5, 64, BF), (9, 1, 256, BF)))
def test_long_context(heads, heads_kv, dim, dtype):
    """One request over thousands of tokens: keys split over the device, parts joined."""
    compare([1], [20011], heads, heads_kv, dim, 16, dtype)
    compare([3], [9000], heads, heads_kv, dim, 64, dtype, "hnd")
    compare([1, 1, 1], [9000, 1, 700], heads, heads_kv, dim, 16, dtype, window=4001, sinks=5)


def test_long_chunk():
    """A few hundred rows over a longer context, in parts and whole."""
    compare([200, 1], [3000, 40], 8, 2, 128, 32, BF)
    compare([260], [900], 6, 2, 96, 16, FP, window=150, sinks=7)


def test_many_requests():
    """More requests than threads of a workgroup, most of them short or without new tokens."""
    rng = np.random.default_rng(6)
    kv = [int(x) for x in rng.integers(0, 40, 700)]
    new = [min(int(x), n) for x, n in zip(rng.integers(0, 3, 700), kv)]
    compare(new, kv, 4, 2, 64, 8, BF)


def test_rows_outside_every_request_stay():
    q, k, v, table, starts = case(7, [3, 4], [30, 40], 4, 2, 64, 16, BF)
    from flashgann_amd import attention
    q = torch.cat([q, q[:2]])
    out = torch.full(q.shape, 5.0, dtype=BF).cuda()
    lse = torch.full(q.shape[:2], 5.0).cuda()
    qd, kd, vd, td = dev(q, k, v, table)
    attention.attend(qd, kd, vd, td, torch.tensor(starts, dtype=torch.int32).cuda(),
                     torch.tensor([30, 40], dtype=torch.int32).cuda(), max_q=4, out=out, lse=lse)
    assert torch.all(out[7:] == 5.0) and torch.all(lse[7:] == 5.0)
    A.dense(q, k, v, table, starts, [30, 40], 64 ** -0.5).check(out, lse)


def test_offsets_past_32_bits():
    """A cache of over 4 GiB a tensor whose last pages hold the context."""
    from flashgann_amd import attention
    page, heads_kv, dim, pages = 64, 8, 128, 36000  # 4.7 GB each
    rng = np.random.default_rng(8)
    small_k, small_v = A.make_cache(rng, 6, page, heads_kv, dim, BF)
    k, v = (torch.empty((pages, page, heads_kv, dim), dtype=BF, device="cuda") for _ in range(2))
    k[pages - 6:], v[pages - 6:] = small_k.cuda(), small_v.cuda()
    q = torch.from_numpy(rng.standard_normal((141, 16, dim)).astype(np.float32)).to(BF)
    small = torch.tensor([[5, 0, 3, 1], [4, 2, -1, -1]], dtype=torch.int32)
    table = torch.where(small >= 0, small + pages - 6, -1)
    starts, kv = [0, 140, 141], [250, 100]
    args = torch.tensor(starts, dtype=torch.int32).cuda(), torch.tensor(kv, dtype=torch.int32).cuda()
    out, lse = attention.attend(q.cuda(), k, v, table.cuda(), *args, max_q=140)
    A.dense(q, small_k, small_v, small, starts, kv, dim ** -0.5).check(out, lse)
    ids = torch.tensor([[[7, 99, 50]], [[3, 60, 60]]], dtype=torch.int32).expand(2, 16, 3).contiguous()
    out, lse = attention.attend_retrieved(q[:2].cuda(), k, v, table.cuda(), args[1], ids.cuda(), window=8, sinks=2)
    A.retrieved(q[:2], small_k, small_v, small, kv, ids, dim ** -0.5, 8, 2).check(out, lse)
    slots = torch.tensor([(pages - 1) * page + 5, (pages - 6) * page, pages * page, -1], dtype=torch.int64).cuda()
    rows = torch.from_numpy(rng.standard_normal((4, heads_kv, dim)).astype(np.float32)).to(BF).cuda()
    attention.cache_append(rows, -rows, k, v, slots)
    assert torch.equal(k[pages - 1, 5], rows[0]) and torch.equal(v[pages - 6, 0], -rows[1])
    assert torch.equal(k[pages - 1, 6].cpu(), small_k[5, 6])


def test_same_bits_every_time():
    """Parts are joined in their order, whatever ran when."""
    for new, kv, window in (([1], [9000], None), ([150, 1, 3], [4000, 3000, 70], None), ([300], [2000], 77)):
        q, k, v, table, starts = case(9, new, kv, 8, 2, 128, 16, BF)
        got = [run(q, k, v, table, starts, kv, window=window) for _ in range(4)]
        for out, lse in got[1:]:
            assert torch.equal(out, got[0][0]) and torch.equal(lse, got[0][1])


def test_on_another_stream():
    """Work queued on a stream of its own waits for nothing else and is waited for by it alone."""
    from flashgann_amd import attention
    q, k, v, table, starts = case(10, [2, 90], [500, 400], 8, 2, 128, 16, BF)
    want = run(q, k, v, table, starts, [500, 400])
    side = torch.cuda.Stream()
    qd, kd, vd, td = dev(q, k, v, table)
    st, kv = torch.tensor(starts, dtype=torch.int32).cuda(), torch.tensor([500, 400], dtype=torch.int32).cuda()
    torch.cuda.synchronize()
    with torch.cuda.stream(side):
        outs = [attention.attend(qd, kd, vd, td, st, kv, max_q=90) for _ in range(3)]
    side.synchronize()
    for out, lse in outs:
        assert torch.equal(out, want[0]) and torch.equal(lse, want[1])


def test_graph_replays():
    """A captured step follows the lengths in device memory: plan, append and attention replayed over growing
    contexts, with eager work between, against the same calls made eagerly."""
    from flashgann_amd import attention
    B, heads, heads_kv, dim, page, steps = 3, 8, 2, 64, 16, 6
    rng = np.random.default_rng(11)
    lens0 = [30, 1, 100]

    def fresh():
        k, v = (t.cuda() for t in A.make_cache(np.random.default_rng(12), 40, page, heads_kv, dim, BF))
        table = A.make_table(np.random.default_rng(13), 30, lens0, page, 12).cuda()
        held = set(table.flatten().tolist())
        free = torch.tensor([p for p in range(40) if p not in held], dtype=torch.int32).cuda()
        return k, v, table, free, torch.tensor(lens0, dtype=torch.int32).cuda()

    xs = [torch.from_numpy(rng.standard_normal((3, B, heads, dim)).astype(np.float32)).to(BF).cuda() for _ in range(steps)]
    one = torch.ones(B, dtype=torch.int32, device="cuda")

    def step(x, k, v, table, free, lens):
        p = attention.cache_plan(lens, one, table, free, page_size=page, max_tokens=B + 2)
        attention.cache_append(x[1, :, :heads_kv], x[2, :, :heads_kv], k, v, p.slots[:B])
        out, lse = attention.attend(x[0], k, v, table, p.q_starts, p.kv_lens, max_q=1)
        return out, lse, p.kv_lens, p.used

    k, v, table, free, lens = fresh()
    want = []
    for x in xs:
        out, lse, kv, used = step(x, k, v, table, free, lens)
        want.append((out, lse))
        lens, free = kv, free[int(used):].contiguous()
    # the same with a graph; the free list moves on the device
    k, v, table, free, lens = fresh()
    x = xs[0].clone()
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        step(x, k.clone(), v.clone(), table.clone(), free, lens)
    side.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out, lse, kv, used = step(x, k, v, table, free, lens)
    for i in range(steps):
        x.copy_(xs[i])
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, want[i][0]) and torch.equal(lse, want[i][1]), i
        lens.copy_(kv)
        free.copy_(torch.roll(free, -int(used)))


# ---------------------------------------------------------------- attend_retrieved

def run_retrieved(q, k, v, table, kv, ids, **kw):
    from flashgann_amd import attention
    qd, kd, vd, td, i = dev(q, k, v, table, ids)
    return attention.attend_retrieved(qd, kd, vd, td, torch.tensor(kv, dtype=torch.int32).cuda(), i, **kw)


@pytest.mark.parametrize("dtype,dim", ((BF, 64), (FP, 96), (BF, 128), (FP, 256)))
@pytest.mark.parametrize("lists", (2, 4, 8))
@pytest.mark.parametrize("K,window,sinks", ((0, 5, 0), (1, 0, 0), (37, 0, 3), (100, 64, 4), (500, 1, 0), (20, 4000, 0)))
def test_retrieved(dtype, dim, lists, K, window, sinks):
    """Lists for each head, for each key/value head and between; ids anywhere, past the context, repeated."""
    rng = np.random.default_rng(K + dim)
    kv, heads, heads_kv, page = [0, 1, 40, 333, 700], 8, 2, 16
    q, k, v, table, _ = case(K, [1] * 5, kv, heads, heads_kv, dim, page, dtype, "hnd" if dim == 96 else "nhd")
    ids = np.stack([np.stack([rng.permutation(max(K, n) + 3)[:K] for _ in range(lists)]) for n in kv]).astype(np.int64)
    if K > 4:
        ids[:, ::2, K // 2:] = ids[:, ::2, K // 2 - 1:K // 2]  # a short beam's repeats
        ids[:, 0, 1] = -1
    for typed in (ids.astype(np.int32), ids.astype(np.uint32)):
        out, lse = run_retrieved(q, k, v, table, kv, torch.from_numpy(typed), window=window, sinks=sinks)
        A.retrieved(q, k, v, table, kv, ids, dim ** -0.5, window, sinks).check(out, lse)


def test_retrieved_missing_pages():
    q, k, v, table, _ = case(20, [1, 1], [200, 90], 4, 2, 64, 16, BF)
    table[0, 2], table[1, :] = -1, 1 << 20
    ids = torch.from_numpy(np.random.default_rng(1).permutation(200)[:60].astype(np.int32)).expand(2, 2, 60).contiguous()
    out, lse = run_retrieved(q, k, v, table, [200, 90], ids, window=30, sinks=40)
    A.retrieved(q, k, v, table, [200, 90], ids, 0.125, 30, 40).check(out, lse)
    assert torch.all(lse[1] == -np.inf) and torch.all(out[1] == 0)


def test_retrieved_everything_is_dense():
    """All positions as ids give what attend gives, whatever their order."""
    kv = [500, 61]
    q, k, v, table, starts = case(21, [1, 1], kv, 8, 2, 128, 16, BF)
    ids = torch.from_numpy(np.random.default_rng(2).permutation(500).astype(np.int32)).expand(2, 2, 500).contiguous()
    out, lse = run_retrieved(q, k, v, table, kv, ids, window=0, sinks=0)
    A.dense(q, k, v, table, starts, kv, 128 ** -0.5).check(out, lse)


# ---------------------------------------------------------------- plan and append

@pytest.mark.parametrize("seed,requests,page,most_new,width,nfree", (
    (0, 1, 16, 1, 8, 5), (1, 5, 16, 40, 12, 100), (2, 64, 1, 3, 300, 400), (3, 700, 24, 90, 40, 6000),
    (4, 300, 16, 5, 30, 20), (5, 33, 7, 60, 4, 500), (6, 4096, 64, 2, 3, 8000), (7, 3, 128, 5000, 80, 200), (8, 4, 16, 9, 6, 0)))
@pytest.mark.parametrize("slack", (0, 7, -3))
def test_plan(seed, requests, page, most_new, width, nfree, slack):
    from flashgann_amd import attention
    rng = np.random.default_rng(seed)
    lens = rng.integers(-2, width * page // 2 + 2, requests).astype(np.int32)
    new = rng.integers(-1, most_new + 1, requests).astype(np.int32)
    total = max(nfree, 1) + int(np.maximum(lens, 0).sum()) // page + requests + 1
    order = rng.permutation(total).astype(np.int32)
    free, table, at = order[:nfree], np.full((requests, width + 2), -1, np.int32), nfree
    for r in range(requests):
        n = min(-(-max(int(lens[r]), 0) // page), width)
        table[r, :n] = order[at:at + n]
        at += n
    T = max(0, int(np.maximum(new, 0).sum()) + slack)
    dtable = torch.from_numpy(table).cuda()
    got = attention.cache_plan(torch.from_numpy(lens).cuda(), torch.from_numpy(new).cuda(), dtable[:, :width],
                               torch.from_numpy(free).cuda(), page_size=page, max_tokens=T)
    want = A.plan(lens.tolist(), new.tolist(), table[:, :width], free, page, T)
    assert np.array_equal(dtable[:, :width].cpu().numpy(), want[0])
    assert np.array_equal(dtable[:, width:].cpu().numpy(), table[:, width:])
    for name, x, y in zip(("q_starts", "kv_lens", "slots", "positions"), got, want[1:]):
        assert np.array_equal(x.cpu().numpy(), np.asarray(y)), name
    assert int(got.used) == want[5]


@pytest.mark.parametrize("dtype,dim,heads_kv,page,layout", ((BF, 128, 8, 16, "nhd"), (FP, 96, 3, 24, "hnd"), (BF, 64, 1, 1, "nhd"),
                                                            (FP, 256, 20, 64, "hnd")))
@pytest.mark.parametrize("tokens", (0, 1, 63, 700))
def test_append(dtype, dim, heads_kv, page, layout, tokens):
    from flashgann_amd import attention
    rng = np.random.default_rng(tokens)
    pages = -(-2 * max(tokens, 1) // page) + 1
    k, v = A.make_cache(rng, pages, page, heads_kv, dim, dtype, layout)
    rows = torch.from_numpy(rng.standard_normal((tokens, 2, heads_kv + 1, dim)).astype(np.float32)).to(dtype)
    slots = rng.permutation(pages * page)[:tokens].astype(np.int64)
    slots[::5] = -1
    slots[1::7] = pages * page + 3
    kd, vd, rd = dev(k, v, rows)
    kd, vd = (t.permute(0, 2, 1, 3).contiguous().permute(0, 2, 1, 3) if layout == "hnd" else t for t in (kd, vd))
    attention.cache_append(rd[:, 0, 1:], rd[:, 1, :-1], kd, vd, torch.from_numpy(slots).cuda())
    k, v = k.clone(), v.clone()
    for t, s in enumerate(slots):
        if 0 <= s < pages * page:
            k[s // page, s % page], v[s // page, s % page] = rows[t, 0, 1:], rows[t, 1, :-1]
    assert torch.equal(kd.cpu(), k) and torch.equal(vd.cpu(), v)


def test_nothing_to_do():
    """No tokens, no requests: shapes come back empty, nothing is launched on nothing."""
    from flashgann_amd import attention
    k, v = (torch.zeros((4, 16, 2, 64), dtype=BF, device="cuda") for _ in range(2))
    ints = lambda *x: torch.tensor(x, dtype=torch.int32, device="cuda")  # noqa: E731
    out, lse = attention.attend(torch.zeros((0, 4, 64), dtype=BF, device="cuda"), k, v, ints(0, 1).view(1, 2), ints(0, 0),
                                ints(9), max_q=0)
    assert out.shape == (0, 4, 64) and lse.shape == (0, 4)
    out, lse = attention.attend_retrieved(torch.zeros((0, 4, 64), dtype=BF, device="cuda"), k, v, ints().view(0, 2), ints(),
                                          ints().view(0, 2, 0), window=3)
    assert out.shape == (0, 4, 64)
