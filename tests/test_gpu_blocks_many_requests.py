"""As many requests as the calls take: more workgroups' worth of work than a grid has, so
that workgroups go on to further items.  Keys, queries and values are small whole numbers,
whose scores are exact."""
from __future__ import annotations

import pytest
import torch

pytestmark = pytest.mark.gpu

BF = torch.bfloat16
DIM = 64


@pytest.fixture(autouse=True)
def _gpu(gpu_available):
    torch.cuda.set_device(0)


def whole(g, *shape):
    return torch.randint(-1, 2, shape, generator=g, device="cuda")


def batch(requests, most, page, heads, heads_kv, seed, rows=1):
    """(q, k, v, table, starts, kv): pages are shared, lengths 0 to `most` and, a quarter, `most` itself."""
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    width, pages = -(-most // page), 3000
    kv = torch.randint(0, most + 1, (requests,), generator=g, device="cuda")
    kv = torch.where(torch.rand(requests, generator=g, device="cuda") < 0.25, most, kv).int()
    table = torch.randint(0, pages, (requests, width), generator=g, device="cuda").int()
    k, v = (whole(g, pages, page, heads_kv, DIM).to(BF) for _ in range(2))
    q = whole(g, requests * rows, heads, DIM).to(BF)
    return q, k, v, table, torch.arange(requests + 1, device="cuda").int() * rows, kv, g


def scores_of(q, k, table, first, last, heads_kv):
    """(requests, heads_kv, group, tokens) of requests first .. last - 1, exact."""
    n, group = last - first, q.shape[1] // heads_kv
    keys = k[table[first:last].long()].flatten(1, 2).permute(0, 2, 3, 1).float().contiguous()
    return torch.matmul(q[first:last].float().view(n, heads_kv, group, DIM), keys)


@pytest.mark.parametrize("requests,heads_kv,most", ((9000, 8, 300), (3000, 8, 1500), (65536, 1, 40)))
def test_weigh(requests, heads_kv, most):
    """72,000, 24,000 and 65,536 heads: several tokens' tiles of a head, and several heads, to a workgroup."""
    from flashgann_amd import attention
    page, heads = 8, 2 * heads_kv
    q, k, _, table, starts, kv, g = batch(requests, most, page, heads, heads_kv, 1)
    lse = 3 + torch.rand((requests, heads), generator=g, device="cuda")
    weights = torch.zeros((k.shape[0], heads_kv, page), device="cuda")
    attention.cache_weigh(q, k, table, starts, kv, lse, weights, kv, scale=0.125)  # all known: pages add up
    want, off = (torch.zeros(weights.shape, dtype=torch.float64, device="cuda") for _ in range(2))
    times = torch.zeros(k.shape[0], dtype=torch.float64, device="cuda")
    j = torch.arange(table.shape[1] * page, device="cuda")
    for a in range(0, requests, 1000):
        b = min(a + 1000, requests)
        s = 0.125 * scores_of(q, k, table, a, b, heads_kv).double()
        z = lse[a:b].view(b - a, heads_kv, 2, 1).double()
        e = torch.exp(s - z) * (j < kv[a:b, None])[:, None, None]
        # the difference in base 2 (two roundings of its terms) and the exponential
        error = e * ((s.abs() + z + 2) * 2.0 ** -22)
        at = (table[a:b].long()[:, :, None] * heads_kv * page + torch.arange(page, device="cuda")).flatten(1)[:, None] + (torch.arange(heads_kv, device="cuda") * page)[:, None]
        want.view(-1).index_add_(0, at.flatten(), e.sum(2).flatten())
        off.view(-1).index_add_(0, at.flatten(), error.sum(2).flatten())
        times.index_add_(0, table[a:b].long().flatten(), torch.ones(table[a:b].numel(), dtype=torch.float64, device="cuda"))
    # sums in 32 bits, each addition to what there is by then
    tol = off + want * (times[:, None, None] + 4) * 2.0 ** -24
    assert bool(((weights.double() - want).abs() <= tol).all())


def test_selection_and_attention():
    """65,536 single tokens: what each selects, and attention over it."""
    from flashgann_amd import attention
    requests, page, heads, heads_kv, k = 65536, 4, 4, 2, 3
    q, kc, vc, table, starts, kv, _ = batch(requests, 40, page, heads, heads_kv, 2)
    codes, scales = torch.zeros((kc.shape[0], heads_kv, 2, DIM), dtype=torch.int8, device="cuda"), torch.zeros((kc.shape[0], heads_kv), device="cuda")
    attention.cache_bounds(kc, torch.arange(kc.shape[0] * page, device="cuda"), codes, scales)
    assert torch.equal(codes[:, :, 0].float() * scales[..., None], kc.float().amax(1)) and torch.equal(codes[:, :, 1].float() * scales[..., None], kc.float().amin(1))
    ids = attention.select_blocks(q, codes, scales, table, starts, kv, page_size=page, k=k)
    out, lse = attention.attend_blocks(q, kc, vc, table, starts, kv, ids, scale=0.125)
    assert attention.select_blocks(q, codes, scales, table, starts, kv, page_size=page, k=k).equal(ids)
    width = table.shape[1]
    b = torch.arange(width, device="cuda")
    for a in range(0, requests, 8192):
        z = min(a + 8192, requests)
        n = z - a
        # a list's queries summed, small whole numbers: their codes are themselves times a power of two
        x = q[a:z].float().view(n, heads_kv, 2, DIM)
        asked = torch.cat([x.clamp(min=0).sum(2), x.clamp(max=0).sum(2)], -1)
        at = table[a:z].long()
        held = (codes[at].float() * scales[at][..., None, None]).flatten(3).permute(0, 2, 3, 1).contiguous()
        score = torch.matmul(asked[:, :, None], held)[:, :, 0]
        c = (kv[a:z] - 1) // page
        score = score.masked_fill(~((b >= 1) & (b <= c[:, None] - 1) & (kv[a:z, None] > 0))[:, None], -torch.inf)
        best, order = score.sort(dim=-1, descending=True, stable=True)
        want = torch.where(best[..., :k] > -torch.inf, order[..., :k], width).sort(-1).values
        assert torch.equal(ids[a:z].long(), torch.where(want < width, want, -1))
        listed = (want[..., None] == b).any(-2)
        blocks = (listed | (b == 0) | (b == c[:, None])[:, None]) & (b <= c[:, None])[:, None]
        j = torch.arange(width * page, device="cuda")
        seen = blocks.repeat_interleave(page, -1) & (j < kv[a:z, None])[:, None]
        s = (0.125 * scores_of(q, kc, table, a, z, heads_kv)).masked_fill(~seen[:, :, None], -torch.inf)
        values = vc[at].flatten(1, 2).permute(0, 2, 1, 3).float().contiguous()
        p = torch.exp(s.double()).float()
        l = p.sum(-1, keepdim=True)
        there = (kv[a:z] > 0)[:, None]
        o = torch.where(l > 0, torch.matmul(p, values) / l.clamp(min=1e-30), 0.0).view(n, heads, DIM)
        spread = torch.where(l > 0, torch.matmul(p, values.abs()) / l.clamp(min=1e-30), 0.0).view(n, heads, DIM)
        # the output's rounding; weights in two parts, sums of 12 tokens here and there in 32 bits
        assert bool(((out[a:z].float() - o).abs() <= 2.0 ** -8 * 1.01 * o.abs() + 2.0 ** -15 * spread).all())
        want_lse = torch.log(l.double()).view(n, heads)
        assert bool(((lse[a:z].double() - want_lse).abs() <= 2.0 ** -20 * (1 + want_lse.abs()))[there.expand(-1, heads)].all())
        assert bool((lse[a:z][~there[:, 0]] == -torch.inf).all())


def test_evict():
    """4,096 requests of 16 heads, a quarter of them over their budget."""
    from flashgann_amd import attention
    requests, page, heads_kv, budget, window, sinks = 4096, 4, 16, 30, 5, 2
    g = torch.Generator(device="cuda")
    g.manual_seed(3)
    width = 10
    kv = torch.randint(0, 41, (requests,), generator=g, device="cuda").int()
    table = torch.randperm(requests * width, generator=g, device="cuda").int().view(requests, width)
    k, v = (torch.randint(-9999, 9999, (requests * width, page, heads_kv, DIM), generator=g, device="cuda").to(BF) for _ in range(2))
    w = torch.rand((requests * width, heads_kv, page), generator=g, device="cuda")
    at = table.long()

    def rows(x):  # (requests, heads_kv, tokens, ..) by place
        return x[at].flatten(1, 2).transpose(1, 2)
    k0, v0, w0 = rows(k).clone(), rows(v).clone(), w[at].permute(0, 2, 1, 3).flatten(2).clone()
    e = attention.cache_evict(k, v, w, table, kv, budget=budget, window=window, sinks=sinks)
    k1, v1, w1 = rows(k), rows(v), w[at].permute(0, 2, 1, 3).flatten(2)
    assert torch.equal(e.kv_lens, kv.clamp(max=budget))
    within = kv <= budget
    assert torch.equal(k1[within], k0[within]) and torch.equal(v1[within], v0[within]) and torch.equal(w1[within], w0[within])
    keep = budget - window
    for r in torch.nonzero(~within).flatten().tolist()[::7]:
        n = int(kv[r])
        drawn = w0[r, :, sinks:n - window]
        chosen = torch.zeros((heads_kv, n), dtype=torch.bool, device="cuda")
        chosen[:, :sinks] = True
        chosen[:, sinks:n - window].scatter_(1, drawn.sort(dim=1, descending=True, stable=True).indices[:, :keep - sinks], True)
        for h in range(0, heads_kv, 5):
            stay, place = chosen[h].nonzero().flatten(), torch.arange(budget, device="cuda")
            place[:keep][~chosen[h, :keep]] = stay[stay >= keep]
            place[keep:] = torch.arange(n - window, n, device="cuda")
            assert torch.equal(k1[r, h, :budget], k0[r, h, place]) and torch.equal(v1[r, h, :budget], v0[r, h, place]) and torch.equal(w1[r, h, :budget], w0[r, h, place])
    held = torch.arange(width, device="cuda")
    gone = (held >= (-(-kv.clamp(max=budget) // page))[:, None]) & (held < (-(-kv // page))[:, None])
    assert int(e.released) == int(gone.sum()) and torch.equal(e.freed[:int(e.released)], table[gone]) and bool((e.freed[int(e.released):] == -1).all())
