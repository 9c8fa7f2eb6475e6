"""The paged cache and its attention at the limits of what they take: lengths that
pass 31 bits, weights below what 16 bits hold."""
from __future__ import annotations

import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu

MOST = 2 ** 31 - 1


@pytest.fixture(autouse=True)
def _gpu(gpu_available):
    torch.cuda.set_device(0)


def ints(*x):
    return torch.tensor(x, dtype=torch.int32).cuda()


@pytest.mark.parametrize("page", (16, 24, 65537))
@pytest.mark.parametrize("new", (40, 40000))
def test_plan_past_the_longest_request(page, new):
    """A request that would pass 2^31 - 1 tokens ends there; it takes no page for what lies past it, and the
    request after it gets its own.  (65537: the page counts past 2^31 tokens would wrap.)"""
    from flashgann_amd import attention
    table = torch.tensor([[9, 8, 7, 6], [-1, -1, -1, -1]], dtype=torch.int32).cuda()
    p = attention.cache_plan(ints(MOST - 19, 0), ints(new, 7), table, ints(3, 4), page_size=page, max_tokens=new + 9)
    assert p.q_starts.tolist() == [0, new, new + 7] and p.kv_lens.tolist() == [MOST, 7] and p.used.tolist() == [1]
    assert table.tolist() == [[9, 8, 7, 6], [3, -1, -1, -1]]
    want = [min(MOST - 19 + i, MOST) for i in range(new)] + list(range(7)) + [0, 0]
    assert np.array_equal(p.positions.cpu().numpy(), np.asarray(want))
    assert p.slots.tolist() == [-1] * new + [3 * page + i for i in range(7)] + [-1, -1]


def test_plan_up_to_the_longest_request():
    """With pages for them the tokens up to 2^31 - 1 have slots, those past it none."""
    from flashgann_amd import attention
    page = 1 << 29
    table = torch.tensor([[3, 1, 0, 2]], dtype=torch.int32).cuda()
    p = attention.cache_plan(ints(MOST - 19), ints(40), table, ints(), page_size=page, max_tokens=40)
    assert p.kv_lens.tolist() == [MOST] and p.used.tolist() == [0] and table.tolist() == [[3, 1, 0, 2]]
    assert p.slots.tolist() == [2 * page + (MOST - 19 + i) % page for i in range(19)] + [-1] * 21
    assert p.positions.tolist() == [min(MOST - 19 + i, MOST) for i in range(40)]


def small_weights(form, dim):
    """float16, one token with most of the weight and values of 0, and 65,600 with 2^-26 of its weight each, together
    0.1% of the row, and values of 1.  As many requests (over the same pages) and heads as there are workgroups, so
    that one of them walks all of a row's tokens after that one.  Returns (out, lse, the small ones of each row, their
    weight together), the row's weight being 1 more than that."""
    from flashgann_amd import attention
    kv, page, heads_kv, new = 65601, 64, 8, 20 if form == "tiles" else 1
    requests = (256 if form == "tiles" else 512) // heads_kv
    pages = -(-kv // page)
    shape = (pages, page, heads_kv, dim)
    k, v = torch.zeros(shape, dtype=torch.float16, device="cuda"), torch.ones(shape, dtype=torch.float16, device="cuda")
    k[3, 5, :, 0], v[3, 5] = 4.2421875, 0.0
    q = torch.zeros((requests * new, 2 * heads_kv, dim), dtype=torch.float16, device="cuda")
    q[:, :, 0] = 4.25
    table = torch.arange(pages, dtype=torch.int32).expand(requests, pages).contiguous().cuda()
    lens = ints(*[kv] * requests)
    if form == "retrieved":
        ids = torch.arange(1000, dtype=torch.int32).expand(requests, heads_kv, 1000).contiguous().cuda()
        out, lse = attention.attend_retrieved(q, k, v, table, lens, ids, window=kv - 1000, scale=1.0)
    else:
        out, lse = attention.attend(q, k, v, table, ints(*range(0, requests * new + 1, new)), lens, max_q=new, scale=1.0)
    n = np.tile(kv - new + np.arange(new), requests)  # a row's tokens but the one
    return out.double().cpu().numpy(), lse.double().cpu().numpy(), n, n * np.exp(-4.2421875 * 4.25)


@pytest.mark.parametrize("form", ("rows", "tiles", "retrieved"))
@pytest.mark.parametrize("dim", (64, 96, 128, 256))
def test_many_small_weights(form, dim):
    """They are in the denominator, so they have to be in the numerator."""
    out, _, n, w = small_weights(form, dim)
    want = (w / (1 + w))[:, None, None]
    # a weight in 16 bits is off by 2^-32 at most, 32-bit scores and sums, the output rounded once
    tol = n[:, None, None] * 2.0 ** -32 + want * ((n[:, None, None] + 8) * 2.0 ** -22 + 18.1 * (dim + 8) * 2.0 ** -23 + 2.0 ** -11)
    off = np.abs(out - want)
    assert (off <= tol).all(), (float(off.max()), float(tol.max()), float(want.max()))


@pytest.mark.parametrize("form", ("rows", "tiles", "retrieved"))
@pytest.mark.parametrize("dim", (64, 96, 128, 256))
def test_many_small_weights_in_the_sum(form, dim):
    """Nor may they get lost in the denominator, next to 1."""
    _, lse, n, w = small_weights(form, dim)
    want = (4.2421875 * 4.25 + np.log1p(w))[:, None]
    off = np.abs(lse - want)
    assert (off <= 18.1 * (dim + 8) * 2.0 ** -24 + 2.0 ** -21 * 20 + (n[:, None] + 8) * 2.0 ** -24 * w[:, None]).all(), float(off.max())
