"""What the cache and attention entry points refuse, before any device call: the
pointers here are numbers that nothing may follow."""
from __future__ import annotations

import struct

import pytest

from flashgann_amd import _lib, attention

CACHE_FIELDS, ATTENTION_FIELDS = struct.Struct("2Q6q4IiI"), struct.Struct("3Q4qQq3Q5Ii3If")  # the header's structs

AT = 1 << 20  # an aligned address of nothing
CACHE = dict(k=AT, v=AT, k_page=4096, k_token=256, k_head=128, v_page=4096, v_token=256, v_head=128, pages=10, page_size=16,
             heads_kv=2, dim=128, dtype=0, reserved=0)
ATTENTION = dict(q=AT, out=AT, lse=AT, q_token=1024, q_head=128, out_token=1024, out_head=128, table=AT, table_row=5,
                 q_starts=AT, kv_lens=AT, ids=AT, table_width=500, requests=3, tokens=3,
                 heads=8, max_q=1, window=-1, sinks=0, lists=0, nids=7, scale=0.1)


def refused(rc, word):
    assert rc == _lib.FG_EINVAL, rc
    assert word in _lib.lib().fg_last_error().decode(), _lib.lib().fg_last_error()


def cache_bytes(**kw):
    return CACHE_FIELDS.pack(*{**CACHE, **kw}.values())


def attention_bytes(**kw):
    return ATTENTION_FIELDS.pack(*{**ATTENTION, **kw}.values())


def dense(cache, a, work=AT, bytes_=1 << 40):
    return _lib.lib().fg_attend(cache, a, work, bytes_, None)


def found(cache, a, work=AT, bytes_=1 << 40):
    return _lib.lib().fg_attend_retrieved(cache, a, work, bytes_, None)


FOUND = dict(window=3, lists=2)


BAD_CACHES = ((dict(dim=80), "dim"), (dict(dim=0), "dim"), (dict(dtype=2), "dtype"), (dict(heads_kv=0), "heads_kv"),
              (dict(pages=0), "tokens"), (dict(page_size=0), "tokens"), (dict(pages=1 << 20, page_size=1 << 11), "tokens"),
              (dict(k=0), "NULL"), (dict(v=AT + 8), "aligned"), (dict(k_token=100), "strides"), (dict(v_page=4), "strides"))


@pytest.mark.parametrize("bad,word", BAD_CACHES)
def test_caches(bad, word):
    L = _lib.lib()
    refused(dense(cache_bytes(**bad), attention_bytes()), word)
    refused(found(cache_bytes(**bad), attention_bytes(**FOUND)), word)
    assert L.fg_attend_workspace_bytes(cache_bytes(**bad), attention_bytes()) == _lib.FG_EINVAL
    refused(L.fg_cache_append(cache_bytes(**bad), AT, AT, 256, 128, 256, 128, AT, 4, None), word)


@pytest.mark.parametrize("bad,word", (
    (dict(heads=7), "heads"), (dict(heads=0), "heads"), (dict(heads=2048), "heads"), (dict(scale=0.0), "scale"),
    (dict(scale=-1.0), "scale"), (dict(scale=float("nan")), "scale"), (dict(scale=float("inf")), "scale"),
    (dict(tokens=1 << 30, requests=1 << 30), "tokens"), (dict(tokens=65537, requests=65537), "requests"),
    (dict(table_row=-1), "table"), (dict(table_width=1 << 31), "table"),
    (dict(sinks=1 << 31), "sinks"), (dict(q=0), "NULL"), (dict(out=0), "NULL"), (dict(table=0), "NULL"), (dict(kv_lens=0), "NULL"),
    (dict(q=AT + 2), "aligned"), (dict(q_head=130), "strides"), (dict(out_token=4), "strides"),
    (dict(table_width=1 << 27), "table_width")))
def test_attention(bad, word):
    refused(dense(cache_bytes(), attention_bytes(**bad)), word)
    refused(found(cache_bytes(), attention_bytes(**{**FOUND, **bad})), word)


def test_attention_of_one_kind():
    refused(dense(cache_bytes(), attention_bytes(window=0)), "window")
    refused(dense(cache_bytes(), attention_bytes(window=-2)), "window")
    refused(dense(cache_bytes(), attention_bytes(q_starts=0)), "NULL")
    refused(dense(cache_bytes(), attention_bytes(lists=2)), "lists")
    refused(found(cache_bytes(), attention_bytes(window=-1, lists=2)), "window")
    for lists in (0, 1, 3, 16):
        refused(found(cache_bytes(), attention_bytes(window=3, lists=lists)), "lists")
    refused(found(cache_bytes(), attention_bytes(**FOUND, tokens=4)), "row")
    refused(found(cache_bytes(), attention_bytes(**FOUND, ids=0)), "NULL")
    refused(found(cache_bytes(), attention_bytes(**FOUND, nids=1 << 29)), "ids")
    refused(dense(None, attention_bytes()), "NULL")
    refused(dense(cache_bytes(), None), "NULL")


def test_workspace():
    """What a call needs: nothing where no item is cut, and a smaller, absent or odd one is refused."""
    L = _lib.lib()
    for a, call in ((attention_bytes(), dense), (attention_bytes(max_q=1000), dense),
                    (attention_bytes(window=900, lists=2, sinks=4), found)):
        need = L.fg_attend_workspace_bytes(cache_bytes(), a)
        assert need > 0
        for work, n in ((None, need), (AT + 4, need), (AT, need - 1)):
            refused(call(cache_bytes(), a, work, n), "workspace")
    assert L.fg_attend_workspace_bytes(cache_bytes(), attention_bytes(window=3, lists=2)) == 0
    assert L.fg_attend_workspace_bytes(cache_bytes(), attention_bytes(table_width=20)) == 0
    assert L.fg_attend_workspace_bytes(cache_bytes(), attention_bytes(tokens=0)) == 0


def test_plan():
    L = _lib.lib()

    def plan(lens=AT, new=AT, requests=3, table=AT, row=9, width=9, free=AT, nfree=4, page=16, tokens=5, outs=(AT,) * 5):
        return L.fg_cache_plan(lens, new, requests, table, row, width, free, nfree, page, tokens, *outs, None)

    refused(plan(requests=0), "requests")
    refused(plan(requests=4097), "requests")
    refused(plan(page=0), "page_size")
    refused(plan(tokens=1 << 31), "max_tokens")
    refused(plan(width=1 << 30), "table_width")
    refused(plan(lens=None), "NULL")
    refused(plan(table=None), "NULL")
    refused(plan(free=None), "NULL")
    for i in range(5):
        refused(plan(outs=tuple(None if j == i else AT for j in range(5))), "NULL")


def test_append():
    L = _lib.lib()
    refused(L.fg_cache_append(cache_bytes(), AT + 2, AT, 256, 128, 256, 128, AT, 4, None), "aligned")
    refused(L.fg_cache_append(cache_bytes(), AT, AT, 256, 12, 256, 128, AT, 4, None), "strides")
    refused(L.fg_cache_append(cache_bytes(), AT, AT, 256, 128, 256, 128, None, 4, None), "NULL")
    refused(L.fg_cache_append(cache_bytes(), AT, AT, 256, 128, 256, 128, AT, 1 << 31, None), "tokens")
    assert L.fg_cache_append(cache_bytes(), None, None, 256, 128, 256, 128, None, 0, None) == _lib.FG_OK


def test_tensors_of_the_host_are_refused():
    import torch
    k = torch.zeros((4, 16, 2, 64), dtype=torch.bfloat16)
    ints = torch.zeros(2, dtype=torch.int32)
    with pytest.raises(ValueError, match="CUDA device"):
        attention.attend(torch.zeros((1, 4, 64), dtype=torch.bfloat16), k, k, ints.view(1, 2), ints, ints[:1], max_q=1)
    with pytest.raises(ValueError, match="CUDA device"):
        attention.cache_append(k[0], k[0], k, k, torch.zeros(16, dtype=torch.int64))
    with pytest.raises(ValueError, match="CUDA device"):
        attention.cache_plan(ints, ints, ints.view(2, 1), ints, page_size=16, max_tokens=4)


@pytest.mark.gpu
def test_tensors_of_the_wrong_kind(gpu_available):
    import torch
    z = lambda *s, d=torch.bfloat16: torch.zeros(s, dtype=d, device="cuda")  # noqa: E731
    i32 = torch.int32
    good = dict(q=z(3, 4, 64), k_cache=z(4, 16, 2, 64), v_cache=z(4, 16, 2, 64), block_table=z(2, 2, d=i32),
                q_starts=z(3, d=i32), kv_lens=z(2, d=i32), max_q=1)
    attention.attend(**good)
    for bad in (dict(q=z(3, 4, 128)), dict(q=z(3, 4, 64, d=torch.float16)), dict(q=z(3, 64)), dict(q=z(3, 64, 4).transpose(1, 2)),
                dict(v_cache=z(4, 16, 2, 128)), dict(k_cache=z(4, 16, 2, 64, d=torch.float32)), dict(k_cache=z(4, 16, 64, 2).transpose(2, 3)),
                dict(block_table=z(3, 2, d=i32)), dict(block_table=z(2, 2, d=torch.int64)), dict(block_table=z(2, 2, d=i32).t()),
                dict(q_starts=z(2, d=i32)), dict(kv_lens=z(2, d=torch.int64)), dict(kv_lens=z(4, d=i32)[::2]), dict(window=0),
                dict(sinks=-1), dict(out=z(3, 4, 128)), dict(lse=z(3, 4)), dict(max_q=-1), dict(q_starts=None)):
        with pytest.raises(ValueError):
            attention.attend(**{**good, **bad})
    with pytest.raises(_lib.FlashGannError, match="dim"):
        attention.attend(**{**good, "q": z(3, 4, 80), "k_cache": z(4, 16, 2, 80), "v_cache": z(4, 16, 2, 80)})
    with pytest.raises(_lib.FlashGannError, match="heads"):
        attention.attend(**{**good, "q": z(3, 5, 64)})
    found = dict(q=z(2, 4, 64), k_cache=good["k_cache"], v_cache=good["v_cache"], block_table=good["block_table"],
                 kv_lens=good["kv_lens"], ids=z(2, 2, 5, d=i32), window=2)
    attention.attend_retrieved(**found)
    for bad in (dict(ids=z(3, 2, 5, d=i32)), dict(ids=z(2, 2, 5, d=torch.int64)), dict(ids=z(2, 2, 10, d=i32)[..., ::2]),
                dict(ids=None), dict(window=-1)):
        with pytest.raises(ValueError):
            attention.attend_retrieved(**{**found, **bad})
    with pytest.raises(_lib.FlashGannError, match="lists"):
        attention.attend_retrieved(**{**found, "ids": z(2, 3, 5, d=i32)})
    with pytest.raises(ValueError):
        attention.cache_append(z(3, 2, 64), z(3, 2, 64), good["k_cache"], good["v_cache"], z(4, d=torch.int64))
