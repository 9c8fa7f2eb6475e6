"""Eviction moves rows in place: a cache whose places share memory is refused, before any
device call."""
from __future__ import annotations

import pytest

from test_attention_refusals import cache_bytes, refused
from test_blocks_refusals import evict


@pytest.mark.parametrize("stride,size", (("k_page", "pages"), ("v_page", "pages"), ("k_token", "page_size"), ("v_token", "page_size"), ("k_head", "heads_kv"), ("v_head", "heads_kv")))
def test_strides_of_zero(stride, size):
    refused(evict(cache_bytes(**{stride: 0})), "share memory")
    # of one place the stride says nothing: the next thing that is wrong is named
    refused(evict(cache_bytes(**{stride: 0, size: 1}), work=None), "workspace")


@pytest.mark.gpu
def test_tensors_that_repeat_a_head(gpu_available):
    """Views that name one head's memory as several, and those that only have a size of 1 there."""
    import torch

    from flashgann_amd import _lib, attention
    k, v = (torch.zeros((4, 16, 1, 64), dtype=torch.bfloat16, device="cuda") for _ in range(2))
    table, lens = torch.arange(4, dtype=torch.int32, device="cuda").view(2, 2), torch.tensor([30, 9], dtype=torch.int32, device="cuda")
    with pytest.raises(_lib.FlashGannError, match="share memory"):
        attention.cache_evict(k.expand(-1, -1, 3, -1), v.expand(-1, -1, 3, -1), torch.zeros((4, 3, 16), device="cuda"), table, lens, budget=20, window=3)
    e = attention.cache_evict(k.squeeze(2).unsqueeze(2), v.expand(-1, -1, 1, -1), torch.zeros((4, 1, 16), device="cuda"), table, lens, budget=20, window=3)
    assert e.kv_lens.tolist() == [20, 9]
