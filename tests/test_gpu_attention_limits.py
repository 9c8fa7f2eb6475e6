"""The paged cache and its attention at the limits of what they take: lengths that
pass 31 bits."""
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
