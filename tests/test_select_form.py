"""Where a selection keeps its keys: in memory over tables too long for LDS to hold the keys of
enough rows, which comes the sooner the larger a page's bounds are.  Told by the workspace."""
from __future__ import annotations

import pytest

from flashgann_amd import _lib
from test_attention_refusals import cache_bytes
from test_blocks_refusals import blocks_bytes


@pytest.mark.parametrize("dim,held,stored", ((64, 3000, 3700), (96, 2500, 3100), (128, 2100, 2250), (256, 2000, 2100)))
def test_keys_in_lds_and_in_memory(dim, held, stored):
    def need(width, tokens):
        a = blocks_bytes(tokens=tokens, requests=1, heads=32, lists=8, q_token=32 * dim, q_head=dim, table_width=width + 1, sinks=1)
        return _lib.lib().fg_select_blocks_workspace_bytes(cache_bytes(dim=dim, heads_kv=8), a)
    assert need(held, 1600) == 0
    assert need(stored, 1600) == 1600 * 8 * (stored | 1) * 4
    assert need(stored, 16000) == 0  # past 1 GiB of keys
