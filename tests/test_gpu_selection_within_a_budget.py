"""Selection of pages in a cache that is held to a budget: after each eviction the bounds of
the pages that are still full are written again, and what is selected and attended to is the
definition's of the cache as it is then."""
from __future__ import annotations

import numpy as np
import pytest
import torch

import blocks_oracle as O
from test_gpu_blocks import ints, starts_of
from test_gpu_blocks_together import Serving

pytestmark = pytest.mark.gpu

BF, FP = torch.bfloat16, torch.float16


@pytest.fixture(autouse=True)
def _gpu(gpu_available):
    torch.cuda.set_device(0)


@pytest.mark.parametrize("dtype,dim,heads,heads_kv,page", ((BF, 128, 8, 2, 8), (FP, 64, 6, 3, 5)))
def test_selection_after_evictions(dtype, dim, heads, heads_kv, page):
    from flashgann_amd import attention
    budget, window, sinks = 50, 12, 2
    s = Serving(3, 60, page, heads, heads_kv, dim, dtype, 21)
    for step, new in enumerate(([70, 30, 47], [1, 1, 1], [1, 20, 1], [9, 1, 1], [1, 1, 40])):
        p = s.append(new)
        q = s.randn(sum(new), heads, dim)
        ids = attention.select_blocks(q, s.bounds, s.scales, s.table, p.q_starts, p.kv_lens, page_size=page, k=3)
        out, lse = attention.attend_blocks(q, s.k, s.v, s.table, p.q_starts, p.kv_lens, ids)
        kv, starts, table, k = p.kv_lens.tolist(), starts_of(new), s.table.cpu(), s.k.cpu()
        full = [int(table[r, b]) for r in range(3) for b in range(kv[r] // page)]
        for (pg, h), (codes, scale) in O.bounds(k, full).items():
            assert float(s.scales[pg, h]) == scale and np.array_equal(s.bounds[pg, h].cpu().numpy(), codes), (step, pg, h)
        chosen = O.select(q.cpu(), s.bounds.cpu(), s.scales.cpu(), table.numpy(), starts, kv, page, 3, heads_kv, 1, 1)
        assert np.array_equal(ids.cpu().numpy(), chosen), step
        O.attend(q.cpu(), k, s.v.cpu(), table, starts, kv, torch.from_numpy(chosen), dim ** -0.5, 1, 1).check(out, lse)
        # all of the context gives the tokens their shares
        lse = attention.attend(q, s.k, s.v, s.table, p.q_starts, p.kv_lens, max_q=max(new))[1]
        attention.cache_weigh(q, s.k, s.table, p.q_starts, p.kv_lens, lse, s.weights, s.known)
        e = attention.cache_evict(s.k, s.v, s.weights, s.table, s.lens, budget=budget, window=window, sinks=sinks)
        s.free, s.lens = torch.cat([s.free, e.freed[:int(e.released)]]).contiguous(), e.kv_lens
        b = torch.arange(s.table.shape[1], device="cuda")
        last = torch.where(b < s.lens[:, None] // page, s.table.long() * page + page - 1, -1)
        attention.cache_bounds(s.k, last.flatten(), s.bounds, s.scales)
    assert s.lens.tolist() == [min(n, budget) for n in kv] == [50, 50, 50]
