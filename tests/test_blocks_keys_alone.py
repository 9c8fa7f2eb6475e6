"""Bounds and drawn weights read keys alone: a cache without values serves them, and
every other call refuses it."""
from __future__ import annotations

import ctypes as C

import pytest

from flashgann_amd import _lib
from test_attention_refusals import AT, attention_bytes, cache_bytes, dense, refused
from test_blocks_refusals import attend, blocks_bytes, bounds, evict, weigh


def test_no_values():
    keys = cache_bytes(v=0)
    assert bounds(keys, tokens=0) == _lib.FG_OK
    refused(bounds(keys, slots=None), "NULL device buffer")
    assert weigh(keys, attention_bytes(requests=0)) == _lib.FG_OK
    assert weigh(keys, attention_bytes(table_width=0, table=0)) == _lib.FG_OK
    for rc in (bounds(cache_bytes(k=0), tokens=0), weigh(cache_bytes(k=0), attention_bytes(requests=0)), attend(keys, blocks_bytes(tokens=0)), evict(keys),
               dense(keys, attention_bytes(tokens=0)), _lib.lib().fg_cache_append(keys, AT, AT, 256, 128, 256, 128, AT, 0, None)):
        refused(rc, "NULL cache buffer")


@pytest.mark.gpu
def test_no_values_on_the_gpu(gpu_available):
    """The same bounds and weights as with a cache that has values."""
    import torch

    from flashgann_amd import attention
    g = torch.Generator(device="cuda")
    g.manual_seed(3)
    k = torch.randn((10, 16, 2, 128), generator=g, device="cuda").to(torch.bfloat16)
    q = torch.randn((3, 8, 128), generator=g, device="cuda").to(torch.bfloat16)
    slots = torch.arange(160, device="cuda")
    table = torch.arange(9, dtype=torch.int32, device="cuda").view(3, 3)
    starts, lens, known, lse = (torch.tensor(x, device="cuda") for x in ([0, 1, 2, 3], [48, 40, 17], [47, 39, 16], [[9.0] * 8] * 3))
    starts, lens, known = starts.int(), lens.int(), known.int()
    codes, scales = torch.zeros((2, 10, 2, 2, 128), dtype=torch.int8, device="cuda"), torch.zeros((2, 10, 2), device="cuda")
    weights = torch.zeros((2, 10, 2, 16), device="cuda")
    attention.cache_bounds(k, slots, codes[0], scales[0])
    attention.cache_weigh(q, k, table, starts, lens, lse, weights[0], known)
    keys = cache_bytes(k=k.data_ptr(), v=0)
    a = attention_bytes(q=q.data_ptr(), out=0, lse=lse.data_ptr(), table=table.data_ptr(), table_row=3, table_width=3, q_starts=starts.data_ptr(), kv_lens=lens.data_ptr(),
                        scale=128 ** -0.5)
    L, stream = _lib.lib(), C.c_void_p(torch.cuda.current_stream().cuda_stream)
    assert L.fg_cache_bounds(keys, slots.data_ptr(), 160, codes[1].data_ptr(), scales[1].data_ptr(), stream) == _lib.FG_OK
    assert L.fg_cache_weigh(keys, a, weights[1].data_ptr(), known.data_ptr(), stream) == _lib.FG_OK
    assert bool(codes[0].any()) and bool(weights[0].any())
    assert torch.equal(codes[0], codes[1]) and torch.equal(scales[0], scales[1]) and torch.equal(weights[0], weights[1])
