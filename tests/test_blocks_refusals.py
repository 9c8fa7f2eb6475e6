"""What the entry points over selected pages and of eviction refuse, before any device
call: the pointers here are numbers that nothing may follow."""
from __future__ import annotations

import pytest

from flashgann_amd import _lib, attention
from test_attention_refusals import AT, BAD_CACHES, attention_bytes, cache_bytes, refused

BLOCKS = dict(window=2, sinks=1, lists=2, nids=7)
COMMON = ((dict(heads=7), "heads"), (dict(heads=0), "heads"), (dict(heads=2048), "heads"), (dict(tokens=1 << 30, requests=1 << 30), "tokens"),
          (dict(requests=65537), "requests"), (dict(table_row=-1), "table"), (dict(table_width=1 << 31), "table"), (dict(table_width=1 << 27), "table_width"),
          (dict(q=0), "NULL"), (dict(table=0), "NULL"), (dict(kv_lens=0), "NULL"), (dict(q_starts=0), "NULL"), (dict(q=AT + 2), "aligned"),
          (dict(q_head=130), "strides"))


def bounds(cache=None, slots=AT, tokens=4, codes=AT, scales=AT):
    return _lib.lib().fg_cache_bounds(cache_bytes() if cache is None else cache, slots, tokens, codes, scales, None)


def select(cache, a, codes=AT, scales=AT, ids=AT, work=AT, bytes_=1 << 40):
    return _lib.lib().fg_select_blocks(cache, a, codes, scales, ids, work, bytes_, None)


def attend(cache, a, work=AT, bytes_=1 << 40):
    return _lib.lib().fg_attend_blocks(cache, a, work, bytes_, None)


def weigh(cache, a, weights=AT, known=AT):
    return _lib.lib().fg_cache_weigh(cache, a, weights, known, None)


def evict(cache=None, weights=AT, table=AT, row=100, width=100, lens=AT, requests=3, budget=40, window=8, sinks=4, outs=(AT, AT, AT), work=AT, bytes_=1 << 40):
    return _lib.lib().fg_cache_evict(cache_bytes() if cache is None else cache, weights, table, row, width, lens, requests, budget, window, sinks, *outs,
                                     work, bytes_, None)


def blocks_bytes(**kw):
    return attention_bytes(**{**BLOCKS, **kw})


@pytest.mark.parametrize("bad,word", BAD_CACHES)
def test_caches(bad, word):
    L, cache = _lib.lib(), cache_bytes(**bad)
    refused(bounds(cache), word)
    refused(attend(cache, blocks_bytes()), word)
    refused(weigh(cache, attention_bytes()), word)
    refused(evict(cache), word)
    assert L.fg_attend_blocks_workspace_bytes(cache, blocks_bytes()) == _lib.FG_EINVAL
    if not {"k", "v", "k_token", "v_page"} & set(bad):  # the shape alone
        refused(select(cache, blocks_bytes()), word)
        assert L.fg_select_blocks_workspace_bytes(cache, blocks_bytes()) == _lib.FG_EINVAL
        assert L.fg_cache_evict_workspace_bytes(cache, 100, 3, 40) == _lib.FG_EINVAL


@pytest.mark.parametrize("bad,word", COMMON)
def test_rows(bad, word):
    refused(select(cache_bytes(), blocks_bytes(**bad)), word)
    refused(attend(cache_bytes(), blocks_bytes(**bad)), word)
    refused(weigh(cache_bytes(), attention_bytes(**bad)), word)


def test_bounds():
    refused(bounds(slots=None), "NULL")
    refused(bounds(codes=None), "NULL")
    refused(bounds(scales=None), "NULL")
    refused(bounds(codes=AT + 4), "aligned")
    refused(bounds(tokens=1 << 31), "tokens")
    assert bounds(tokens=0, slots=None) == _lib.FG_OK


def test_lists_and_ranges():
    for call in (select, attend):
        for lists in (0, 1, 3, 16):
            refused(call(cache_bytes(), blocks_bytes(lists=lists)), "lists")
        for window in (0, -1, -5):
            refused(call(cache_bytes(), blocks_bytes(window=window)), "last blocks")
        refused(call(cache_bytes(), blocks_bytes(sinks=1 << 31)), "first blocks")
        refused(call(cache_bytes(), blocks_bytes(nids=4097)), "4")
        refused(call(cache_bytes(), blocks_bytes(tokens=(1 << 22) + 1, requests=9)), "tokens")
        refused(call(None, blocks_bytes()), "NULL")
        refused(call(cache_bytes(), None), "NULL")
        assert call(cache_bytes(), blocks_bytes(tokens=0)) == _lib.FG_OK
        assert call(cache_bytes(), blocks_bytes(requests=0)) == _lib.FG_OK
    refused(select(cache_bytes(), blocks_bytes(nids=0)), "blocks of a list")
    refused(select(cache_bytes(), blocks_bytes(tokens=1 << 20, nids=2000)), "2^31")
    for bad in (dict(codes=None), dict(scales=None), dict(ids=None)):
        refused(select(cache_bytes(), blocks_bytes(), **bad), "NULL")
    refused(select(cache_bytes(), blocks_bytes(), codes=AT + 8), "aligned")
    for bad, word in ((dict(scale=0.0), "scale"), (dict(scale=float("nan")), "scale"), (dict(out=0), "NULL"), (dict(ids=0), "NULL"), (dict(out=AT + 2), "aligned"),
                      (dict(out_token=4), "strides")):
        refused(attend(cache_bytes(), blocks_bytes(**bad)), word)


def test_nothing_new_over_a_wide_table():
    """No tokens or no requests: nothing to do, however wide the table."""
    L = _lib.lib()
    for width in (500, 5000, 500000):
        for none in (dict(tokens=0), dict(requests=0), dict(requests=0, tokens=15, heads=256, lists=256), dict(requests=0, tokens=0)):
            a = blocks_bytes(**{**none, "table_width": width})
            assert L.fg_select_blocks_workspace_bytes(cache_bytes(), a) == 0
            assert L.fg_attend_blocks_workspace_bytes(cache_bytes(), a) == 0
            assert select(cache_bytes(), a) == _lib.FG_OK and attend(cache_bytes(), a) == _lib.FG_OK


def test_workspaces():
    """What a call needs at most, from its sizes; a smaller, absent or odd one is refused."""
    L = _lib.lib()
    for need_of, call, a in ((L.fg_select_blocks_workspace_bytes, select, blocks_bytes(table_width=5000)),
                             (L.fg_select_blocks_workspace_bytes, select, blocks_bytes(table_width=60000, tokens=4000, requests=4000)),
                             (L.fg_attend_blocks_workspace_bytes, attend, blocks_bytes(nids=100))):
        need = need_of(cache_bytes(), a)
        assert need > 0
        for work, n in ((None, need), (AT + 4, need), (AT, need - 1)):
            refused(call(cache_bytes(), a, work=work, bytes_=n), "workspace")
    assert L.fg_select_blocks_workspace_bytes(cache_bytes(), blocks_bytes(table_width=500)) == 0
    assert L.fg_attend_blocks_workspace_bytes(cache_bytes(), blocks_bytes(tokens=0)) == 0
    need = L.fg_cache_evict_workspace_bytes(cache_bytes(), 100, 3, 40)
    assert need > 0
    for work, n in ((None, need), (AT + 4, need), (AT, need - 1)):
        refused(evict(work=work, bytes_=n), "workspace")
    # the largest that the arguments allow: no overflow on the way
    assert L.fg_cache_evict_workspace_bytes(cache_bytes(heads_kv=1024, page_size=16), (1 << 26) - 1, 31, (1 << 31) - 1) > 1 << 40


def test_weigh():
    refused(weigh(cache_bytes(), attention_bytes(), weights=None), "NULL")
    refused(weigh(cache_bytes(), attention_bytes(), known=None), "NULL")
    refused(weigh(cache_bytes(), attention_bytes(lse=0)), "NULL")
    refused(weigh(cache_bytes(), attention_bytes(scale=-1.0)), "scale")
    refused(weigh(cache_bytes(), None), "NULL")
    assert weigh(cache_bytes(), attention_bytes(requests=0)) == _lib.FG_OK
    assert weigh(cache_bytes(), attention_bytes(table_width=0, table=0)) == _lib.FG_OK


def test_evict():
    for bad, word in ((dict(requests=0), "requests"), (dict(requests=4097), "requests"), (dict(budget=0), "budget"), (dict(budget=1 << 31), "budget"),
                      (dict(window=37, sinks=4), "budget"), (dict(window=(1 << 32) - 4, sinks=8), "budget"), (dict(row=-1), "table_row"), (dict(width=1 << 27), "table_width"),
                      (dict(width=(1 << 26) - 1, requests=4000), "table_width"), (dict(weights=None), "NULL"), (dict(table=None), "NULL"), (dict(lens=None), "NULL")):
        refused(evict(**bad), word)
    for i in range(3):
        refused(evict(outs=tuple(None if j == i else AT for j in range(3))), "NULL")
    # keys and values in one memory, lengths written over those that are read
    refused(evict(cache_bytes(k=AT, v=AT)), "same memory")
    apart = cache_bytes(k=AT, v=AT + 64)
    for lens in (AT, AT + 8, AT - 8):
        refused(evict(apart, lens=lens), "overlap")


def test_more_tiles_of_rows_than_a_grid_holds():
    refused(attend(cache_bytes(), blocks_bytes(tokens=1 << 22, heads=256, lists=256)), "2^23 tiles")


def test_tensors_of_the_host_are_refused():
    import torch
    k = torch.zeros((4, 16, 2, 64), dtype=torch.bfloat16)
    ints = torch.zeros(2, dtype=torch.int32)
    q = torch.zeros((1, 4, 64), dtype=torch.bfloat16)
    codes, scales, w = torch.zeros((4, 2, 2, 64), dtype=torch.int8), torch.zeros((4, 2)), torch.zeros((4, 2, 16))
    calls = (lambda: attention.cache_bounds(k, torch.zeros(3, dtype=torch.int64), codes, scales),
             lambda: attention.select_blocks(q, codes, scales, ints.view(1, 2), ints, ints[:1], page_size=16, k=2),
             lambda: attention.attend_blocks(q, k, k, ints.view(1, 2), ints, ints[:1], ints.view(1, 2, 1)),
             lambda: attention.cache_weigh(q, k, ints.view(1, 2), ints, ints[:1], torch.zeros((1, 4)), w, ints[:1]),
             lambda: attention.cache_evict(k, k, w, ints.view(1, 2), ints[:1], budget=3, window=1))
    for call in calls:
        with pytest.raises(ValueError, match="CUDA device"):
            call()


def test_tensors_that_want_a_gradient_are_refused():
    import torch
    k = torch.zeros((4, 16, 2, 64), dtype=torch.bfloat16)
    g = k.clone().requires_grad_()
    ints = torch.zeros(2, dtype=torch.int32)
    q = torch.zeros((1, 4, 64), dtype=torch.bfloat16)
    qg = q.clone().requires_grad_()
    codes, scales, w = torch.zeros((4, 2, 2, 64), dtype=torch.int8), torch.zeros((4, 2)), torch.zeros((4, 2, 16))
    lse = torch.zeros((1, 4))
    calls = (lambda: attention.cache_bounds(g, torch.zeros(3, dtype=torch.int64), codes, scales),
             lambda: attention.select_blocks(qg, codes, scales, ints.view(1, 2), ints, ints[:1], page_size=16, k=2),
             lambda: attention.select_blocks(q, codes, scales.clone().requires_grad_(), ints.view(1, 2), ints, ints[:1], page_size=16, k=2),
             lambda: attention.attend_blocks(qg, k, k, ints.view(1, 2), ints, ints[:1], ints.view(1, 2, 1)),
             lambda: attention.cache_weigh(q, k, ints.view(1, 2), ints, ints[:1], lse.clone().requires_grad_(), w, ints[:1]),
             lambda: attention.cache_weigh(q, k, ints.view(1, 2), ints, ints[:1], lse, w.clone().requires_grad_(), ints[:1]),
             lambda: attention.cache_evict(k, g, w, ints.view(1, 2), ints[:1], budget=3, window=1))
    for call in calls:
        with pytest.raises(ValueError, match="gradient"):
            call()
        with torch.no_grad(), pytest.raises(ValueError, match="CUDA device"):
            call()


@pytest.mark.gpu
def test_tensors_of_the_wrong_kind(gpu_available):
    import torch
    z = lambda *s, d=torch.bfloat16: torch.zeros(s, dtype=d, device="cuda")  # noqa: E731
    i32, i64, f32, i8 = torch.int32, torch.int64, torch.float32, torch.int8
    k, codes, scales, w = z(4, 16, 2, 64), z(4, 2, 2, 64, d=i8), z(4, 2, d=f32), z(4, 2, 16, d=f32)

    def each(call, good, bads):
        call(**good)
        for bad in bads:
            with pytest.raises(ValueError):
                call(**{**good, **bad})

    each(attention.cache_bounds, dict(k_cache=k, slots=z(5, d=i64), bounds=codes, scales=scales),
         (dict(slots=z(5, d=i32)), dict(slots=z(5, 1, d=i64)), dict(slots=z(8, d=i64)[::2]), dict(bounds=z(4, 2, 2, 64, d=torch.uint8)), dict(bounds=z(3, 2, 2, 64, d=i8)),
          dict(bounds=z(4, 2, 64, 2, d=i8).transpose(2, 3)), dict(scales=z(4, 3, d=f32)), dict(scales=z(2, 4, d=f32).t()), dict(scales=z(4, 2)), dict(k_cache=k.float()),
          dict(k_cache=z(4, 16, 3, 64))))
    rows = dict(block_table=z(2, 2, d=i32), q_starts=z(3, d=i32), kv_lens=z(2, d=i32))
    bad_rows = (dict(q=z(3, 4, 128)), dict(q=z(3, 64)), dict(q=z(3, 64, 4).transpose(1, 2)), dict(q=z(3, 4, 64, d=f32)), dict(block_table=z(3, 2, d=i32)),
                dict(block_table=z(2, 2, d=i64)), dict(q_starts=z(2, d=i32)), dict(kv_lens=z(2, d=i64)))
    each(attention.select_blocks, dict(q=z(3, 4, 64), bounds=codes, scales=scales, page_size=16, k=2, **rows),
         bad_rows + (dict(k=0), dict(lists=0), dict(last_blocks=0), dict(first_blocks=-1), dict(page_size=0), dict(scales=z(3, 2, d=f32)), dict(bounds=z(4, 2, 128, d=i8))))
    for bad in (dict(lists=3), dict(k=4097)):
        with pytest.raises(_lib.FlashGannError):
            attention.select_blocks(**{**dict(q=z(3, 4, 64), bounds=codes, scales=scales, page_size=16, k=2, **rows), **bad})
    each(attention.attend_blocks, dict(q=z(3, 4, 64), k_cache=k, v_cache=k.clone(), ids=z(3, 2, 5, d=i32), **rows),
         bad_rows + (dict(q=z(3, 4, 64, d=torch.float16)), dict(ids=z(2, 2, 5, d=i32)), dict(ids=z(3, 2, 5, d=i64)), dict(ids=z(3, 2, 10, d=i32)[..., ::2]), dict(ids=z(3, 10, d=i32)),
                     dict(last_blocks=0), dict(out=z(3, 4, 128)), dict(lse=z(3, 4)), dict(scale="x")))
    each(attention.cache_weigh, dict(q=z(3, 4, 64), k_cache=k, lse=z(3, 4, d=f32), weights=w, known=z(2, d=i32), **rows),
         bad_rows + (dict(lse=z(3, 4)), dict(lse=z(4, 3, d=f32).t()), dict(weights=z(4, 16, 2, d=f32)), dict(weights=z(4, 16, 2, d=f32).transpose(1, 2)), dict(known=z(3, d=i32)),
                     dict(known=z(2, d=i64)), dict(weights=z(4, 2, 16))))
    each(attention.cache_evict, dict(k_cache=k, v_cache=k.clone(), weights=w, block_table=z(2, 2, d=i32), kv_lens=z(2, d=i32), budget=5, window=1),
         (dict(weights=z(4, 2, 8, d=f32)), dict(kv_lens=z(2, d=i64)), dict(block_table=z(3, 2, d=i32)), dict(budget=0), dict(window=-1), dict(sinks=-1), dict(v_cache=z(4, 16, 2, 128))))
    with pytest.raises(_lib.FlashGannError, match="budget"):
        attention.cache_evict(k, k.clone(), w, z(2, 2, d=i32), z(2, d=i32), budget=5, window=4, sinks=2)
