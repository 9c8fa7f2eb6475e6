"""Where attention over selected pages may write: rows of their own, q's among them."""
from __future__ import annotations

import numpy as np
import pytest

from flashgann_amd import _lib
from test_attention_refusals import cache_bytes, refused
from test_blocks_refusals import attend, blocks_bytes


def test_rows_that_share_memory():
    refused(attend(cache_bytes(), blocks_bytes(out_token=0)), "share memory")
    refused(attend(cache_bytes(), blocks_bytes(out_head=0)), "share memory")
    assert _lib.lib().fg_attend_blocks_workspace_bytes(cache_bytes(), blocks_bytes(out_head=0)) == _lib.FG_EINVAL
    # of one row the stride says nothing
    one = blocks_bytes(out_token=0, out_head=0, tokens=1, heads=1, lists=1, requests=1, nids=4096)
    assert _lib.lib().fg_attend_blocks_workspace_bytes(cache_bytes(heads_kv=1), one) > 0


@pytest.mark.gpu
@pytest.mark.parametrize("new,kv,heads,k,dim", (([1], [5000], 8, 100, 128), ([1] * 60, [300] * 60, 8, 4, 64), ([600], [900], 16, 5, 128), ([90], [700], 12, 5, 256)))
def test_out_may_be_q(gpu_available, new, kv, heads, k, dim):
    """Parts joined afterwards, single tokens, chunks: the same bits as into memory of its own."""
    import torch

    from flashgann_amd import attention
    from test_gpu_blocks import case, ints, some_ids
    q, kc, vc, table, starts = case(31, new, kv, heads, 2, dim, 16, torch.bfloat16)
    ids = some_ids(np.random.default_rng(2), new, kv, 2, k, 16).cuda()
    rest = (kc.cuda(), vc.cuda(), table.cuda(), ints(starts), ints(kv), ids)
    want, want_lse = attention.attend_blocks(q.cuda(), *rest)
    x = q.cuda()
    out, lse = attention.attend_blocks(x, *rest, out=x)
    assert out.data_ptr() == x.data_ptr() and torch.equal(x, want) and torch.equal(lse, want_lse)
    with pytest.raises(_lib.FlashGannError, match="share memory"):
        attention.attend_blocks(q.cuda(), *rest, out=torch.empty((sum(new), 1, dim), dtype=torch.bfloat16, device="cuda").expand(-1, heads, -1))
