"""One infinite value or NaN anywhere in a tile of values, whatever its channel, reaches the
rows that see its token, there alone: all other outputs are as without it, bit for bit."""
from __future__ import annotations

import numpy as np
import pytest
import torch

from test_gpu_blocks import KV, MANY, case, ints

pytestmark = pytest.mark.gpu

BF, FP = torch.bfloat16, torch.float16
NAN, INF = float("nan"), float("inf")


@pytest.fixture(autouse=True)
def _gpu(gpu_available):
    torch.cuda.set_device(0)


@pytest.mark.parametrize("dtype", (BF, FP))
@pytest.mark.parametrize("dim", (64, 96, 128, 256))
@pytest.mark.parametrize("new,kv,heads,heads_kv,lists", ((MANY, KV, 16, 8, 8), ([6, 40], [100, 333], 8, 2, 2), ([1, 1], [100, 333], 8, 2, 2)))
def test_each_channel(dtype, dim, new, kv, heads, heads_kv, lists):
    """In 32 rows a tile, 16, and one token's: a value on the list of every other row, in each channel in turn."""
    from flashgann_amd import attention
    q, kc, vc, table, starts = case(7, new, kv, heads, heads_kv, dim, 8, dtype)
    r = int(np.argmax([min(n, m // 8 - 6) for n, m in zip(new, kv)]))  # a request with many rows past its block 3
    rows = torch.arange(starts[r], starts[r + 1])
    ids = torch.full((sum(new), lists, 2), -1, dtype=torch.int32)
    ids[:, :, 0] = 2
    ids[rows[::2], :, 1] = 3
    args = (q.cuda(), kc.cuda())
    rest = (table.cuda(), ints(starts), ints(kv), ids.cuda())
    vd = vc.cuda()
    group, page = heads // heads_kv, int(table[r, 3])
    # those that see block 3: on the list, with it behind their last block, or in it
    pos = kv[r] - new[r] + np.arange(new[r])
    sees = torch.from_numpy(((np.arange(new[r]) % 2 == 0) & (pos // 8 >= 4)) | ((pos // 8 == 3) & (pos % 8 >= 5)))
    assert bool(sees.any())
    vd[page, 5] = 0
    plain, plain_lse = attention.attend_blocks(*args, vd, *rest)
    assert bool(torch.isfinite(plain).all())
    seen, hidden = rows[sees].cuda(), rows[~sees].cuda()
    wrong = []
    for c in range(dim):
        h, what = c % heads_kv, (NAN, INF, -INF)[c % 3]
        vd[page, 5, h, c] = what
        out, lse = attention.attend_blocks(*args, vd, *rest)
        vd[page, 5, h, c] = 0
        there = out[seen, h * group:(h + 1) * group, c].float()
        ok = bool(torch.isnan(there).all()) if np.isnan(what) else bool((there == what).all())
        out[seen, h * group:(h + 1) * group, c] = plain[seen, h * group:(h + 1) * group, c]
        if not (ok and torch.equal(out, plain) and torch.equal(lse, plain_lse)):
            wrong.append((c, what))
    assert not wrong, (len(wrong), wrong[:8])
