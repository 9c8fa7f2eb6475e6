"""Rows that belong to no request keep what lay in the list of pages, in every form of the
selection; eviction whose workgroups take several requests and heads, in every form; tokens
and places without a page."""
from __future__ import annotations

import ctypes as C

import numpy as np
import pytest
import torch

from test_attention_refusals import attention_bytes, cache_bytes
from test_gpu_blocks import bounds_on_gpu, case, ints, plain_select
from test_gpu_evict import compare_evict

pytestmark = pytest.mark.gpu

BF = torch.bfloat16
LEFT = 123456  # what lies in the ids before the call


@pytest.fixture(autouse=True)
def _gpu(gpu_available):
    torch.cuda.set_device(0)


def select_into(ids, q, bounds, scales, table, starts, kv, page, k, lists):
    """fg_select_blocks over the caller's ids, with first_blocks and last_blocks 1."""
    from flashgann_amd import _lib
    L = _lib.lib()
    cache = cache_bytes(k=0, v=0, pages=bounds.shape[0], page_size=page, heads_kv=bounds.shape[1], dim=q.shape[2])
    a = attention_bytes(q=q.data_ptr(), out=0, lse=0, ids=0, q_token=q.stride(0), q_head=q.stride(1), table=table.data_ptr(), table_row=table.stride(0),
                        table_width=table.shape[1], q_starts=starts.data_ptr(), kv_lens=kv.data_ptr(), requests=kv.shape[0], tokens=q.shape[0], heads=q.shape[1],
                        max_q=0, window=1, sinks=1, lists=lists, nids=k)
    need = L.fg_select_blocks_workspace_bytes(cache, a)
    assert need >= 0
    work = torch.empty(max(need, 1), dtype=torch.uint8, device="cuda")
    rc = L.fg_select_blocks(cache, a, bounds.data_ptr(), scales.data_ptr(), ids.data_ptr(), work.data_ptr() if need else None, need,
                            C.c_void_p(torch.cuda.current_stream().cuda_stream))
    assert rc == _lib.FG_OK, L.fg_last_error()
    torch.cuda.synchronize()
    return need


@pytest.mark.parametrize("rows,begin,new,kv,page,memory", (
    (30, 4, 21, 200, 8, False),      # a workgroup a row
    (700, 33, 640, 3000, 8, False),  # tiles of 16 rows
    (700, 37, 641, 6000, 4, False),  # of 16 rows, more blocks
    (60, 5, 50, 12000, 4, True),     # few tiles over many blocks
    (3, 1, 1, 20000, 4, True),       # a row over many blocks
    (700, 31, 640, 12000, 4, False), # of 8 rows
    (700, 31, 640, 16000, 4, True),  # keys in memory
))
@pytest.mark.parametrize("k", (7, 40))
def test_select_leaves_rows_outside(rows, begin, new, kv, page, memory, k):
    q, kc, _, table, _ = case(rows + k, [rows], [kv], 4, 2, 64, page, BF)
    bounds, scales = torch.zeros((kc.shape[0], 2, 2, 64), dtype=torch.int8, device="cuda"), torch.zeros((kc.shape[0], 2), device="cuda")
    bounds_on_gpu(kc, list(range(page - 1, kc.shape[0] * page, page)), bounds, scales)
    qd, td = q.cuda(), table.cuda()
    guard = 64  # and so does what lies around the list
    ids = torch.full((2 * guard + rows * 2 * k,), LEFT, dtype=torch.int32, device="cuda")
    # rows before the request, behind it, and a request without rows between
    need = select_into(ids[guard:], qd, bounds, scales, td.repeat(2, 1), ints([begin, begin, begin + new]), ints([50, kv]), page, k, 2)
    assert (need > 0) == memory
    got = ids[guard:guard + rows * 2 * k].view(rows, 2, k)
    assert bool((ids[:guard] == LEFT).all()) and bool((ids[-guard:] == LEFT).all())
    assert bool((got[:begin] == LEFT).all()) and bool((got[begin + new:] == LEFT).all())
    assert torch.equal(got[begin:begin + new], plain_select(q[begin:begin + new], bounds, scales, table, [0, new], [kv], page, k, 2, 1, 1))


def many_lengths(requests, budget, some):
    """Mostly within the budget, a few over it, `some` of them given by request."""
    kv = np.random.default_rng(requests).integers(0, 2 * budget // 3, requests)
    kv[3::17] = budget + 1 + np.arange(len(kv[3::17])) % 40
    for r, n in some.items():
        kv[r] = n
    return kv.tolist()


@pytest.mark.parametrize("page,width,budget,window,some", (
    (64, 520, 60, 9, {5: 33000, 20: 900, 261: 20000, 276: 33280}),  # past what registers hold: 512 workgroups share 600 choices
    (64, 520, 60, 0, {0: 61, 256: 33280, 299: 33280}),
    (64, 300, 60, 20, {7: 19200, 290: 9000}),                       # in registers, moved by the other kernels
    (8, 65, 60, 9, {7: 520, 290: 300}),                             # moved by those that choose
))
def test_evict_many_choices(page, width, budget, window, some):
    """300 requests of two heads, short and long, in one call."""
    compare_evict(many_lengths(300, budget, some), 2, 64, page, BF, budget, window, 2, width=width)


@pytest.mark.parametrize("kv,page,budget,width", (([200, 90, 130], 8, 50, 25), ([9000, 700], 16, 600, 600), ([40000], 64, 2000, 640)))
def test_evict_places_without_a_page(kv, page, budget, width):
    """A token whose place has no page is lost, one without a page has nothing to move, and the pages given back are
    the table's entries as they are: in each form."""
    def gone(w, t):
        keep = (budget - 9) // page
        t[0, 1], t[0, keep], t[0, keep - 1] = -1, -1, w.shape[0]  # places of the heaviest and of the window
        t[0, kv[0] // page - 1], t[0, kv[0] // page - 2], t[-1, 0] = 1 << 30, -7, -1
    compare_evict(kv, 2, 64, page, BF, budget, 9, 2, seed=5, change=gone, width=width)
