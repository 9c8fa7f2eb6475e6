"""What eviction asks for: two lists of the tokens that may move, a count for each request and
head, and, where registers do not hold them, weights."""
from __future__ import annotations

import pytest

from flashgann_amd import _lib
from test_attention_refusals import cache_bytes


@pytest.mark.parametrize("width,requests,heads_kv,budget,moves,keys", (
    (260, 48, 8, 4096, 64, 0),             # a few tokens over their budget
    (256, 48, 8, 4096, 0, 0),              # none can be
    (100, 48, 8, 4096, 0, 0),
    (500, 4, 8, 4096, 3904, 0),            # less room past the budget than in it
    (1000, 4, 8, 4096, 4096, 0),           # more
    (4096, 4, 8, 4096, 4096, 32 * 65536),  # weights of a scratch for each request and head
))
def test_sizes(width, requests, heads_kv, budget, moves, keys):
    need = _lib.lib().fg_cache_evict_workspace_bytes(cache_bytes(heads_kv=heads_kv, page_size=16), width, requests, budget)
    pairs = requests * heads_kv
    assert need == 8 * pairs * moves + -(-pairs * 4 // 16) * 16 + 4 * keys
