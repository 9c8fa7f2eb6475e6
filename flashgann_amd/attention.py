"""A paged key/value cache on the GPU and the attention that reads it, for
programs that answer with what a search found.

  cache_plan        block tables and slot maps from request lengths
  cache_append      new keys and values into their slots
  attend            a chunk of new tokens (one to many a request) over the
                    cache, with or without a sliding window and first tokens
                    that stay visible
  attend_retrieved  one token a request over the first tokens, the last ones
                    and the ids that `Index.search_device` returned

Tensors are torch tensors on the current device; calls are queued on its current
stream and return without synchronising.  A cache is two tensors of shape
(pages, page_size, heads_kv, dim), bfloat16 or float16, dim 64, 96, 128 or 256;
any order in memory whose last dimension is contiguous serves, such as
(pages, heads_kv, page_size, dim) permuted.  All compute goes through
libflashgann.so; there is no fallback.
"""
from __future__ import annotations

import struct
from typing import NamedTuple

import torch

from ._lib import FG_BF16, FG_F16, check, lib

__all__ = ["CachePlan", "cache_plan", "cache_append", "attend", "attend_retrieved"]

_DTYPES = {torch.bfloat16: FG_BF16, torch.float16: FG_F16}
_IDS = (torch.int32, torch.uint32)
_CACHE = struct.Struct("2Q6q4IiI")         # fg_kv_cache
_ATTENTION = struct.Struct("3Q4qQq5Q5Ii3If")  # fg_attention


class CachePlan(NamedTuple):
    """What `cache_plan` returns."""
    q_starts: torch.Tensor   # (requests + 1,) int32
    kv_lens: torch.Tensor    # (requests,) int32
    slots: torch.Tensor      # (max_tokens,) int64
    positions: torch.Tensor  # (max_tokens,) int32
    used: torch.Tensor       # (1,) int32


def _need(ok: bool, what: str) -> None:
    if not ok:
        raise ValueError(what)


def _stream(device: int) -> int:
    _need(device >= 0 and device == torch.cuda.current_device(), "tensors must be on the current CUDA device")
    return torch.cuda.current_stream(device).cuda_stream


def _vector(t: torch.Tensor, n: int | None, dtype: torch.dtype, device: int, name: str) -> int:
    _need(t.dtype == dtype and t.ndim == 1 and (n is None or t.shape[0] == n) and t.is_contiguous()
          and t.get_device() == device,
          f"{name} must be a contiguous {dtype} vector" + ("" if n is None else f" of {n}") + " on the same device")
    return t.data_ptr()


def _cache(k: torch.Tensor, v: torch.Tensor, device: int) -> tuple[bytes, tuple]:
    shape, ks, vs = k.shape, k.stride(), v.stride()
    _need(len(shape) == 4 and v.shape == shape, "k_cache and v_cache must have shape (pages, page_size, heads_kv, dim)")
    dtype = _DTYPES.get(k.dtype)
    _need(dtype is not None and v.dtype == k.dtype, "k_cache and v_cache must be bfloat16 or float16")
    _need(k.get_device() == device and v.get_device() == device, "k_cache and v_cache must be on the same device")
    _need(ks[3] == 1 and vs[3] == 1, "the last dimension of k_cache and v_cache must be contiguous")
    return _CACHE.pack(k.data_ptr(), v.data_ptr(), ks[0], ks[1], ks[2], vs[0], vs[1], vs[2], shape[0], shape[1],
                       shape[2], shape[3], dtype, 0), shape


def _table(t: torch.Tensor, requests: int, device: int) -> tuple[int, int, int]:
    _need(t.dtype == torch.int32 and t.ndim == 2 and t.shape[0] == requests and t.get_device() == device
          and (t.shape[1] <= 1 or t.stride(1) == 1) and t.stride(0) >= 0,
          f"block_table must be int32 of shape ({requests}, width), its rows contiguous, on the same device")
    return t.data_ptr(), t.stride(0), t.shape[1]


def cache_plan(lens: torch.Tensor, new_lens: torch.Tensor, block_table: torch.Tensor, free_pages: torch.Tensor, *,
               page_size: int, max_tokens: int) -> CachePlan:
    """Gives each request the pages that its new tokens need, in one launch.

    lens, new_lens: (requests,) int32, tokens held and tokens to come;
    block_table: (requests, width) int32, written in place where a request gets
    a page (-1 once free_pages is used up); free_pages: (n,) int32;
    max_tokens: the length of the slot map, at least the sum of new_lens for
    every token to have an entry.  Entries past the last token hold slot -1.
    `used` is the number of pages taken: drop so many from free_pages."""
    device = lens.get_device()
    requests = lens.shape[0]
    stream = _stream(device)
    _need(0 <= max_tokens < 1 << 31, "max_tokens must be in [0, 2^31)")
    _need(1 <= page_size < 1 << 31, "page_size must be in [1, 2^31)")
    table, row, width = _table(block_table, requests, device)
    i32 = {"dtype": torch.int32, "device": lens.device}
    out = CachePlan(torch.empty(requests + 1, **i32), torch.empty(requests, **i32),
                    torch.empty(max_tokens, dtype=torch.int64, device=lens.device), torch.empty(max_tokens, **i32),
                    torch.empty(1, **i32))
    check(lib().fg_cache_plan(_vector(lens, None, torch.int32, device, "lens"),
                              _vector(new_lens, requests, torch.int32, device, "new_lens"), requests, table, row, width,
                              _vector(free_pages, None, torch.int32, device, "free_pages"), free_pages.shape[0],
                              page_size, max_tokens, out.q_starts.data_ptr(), out.kv_lens.data_ptr(),
                              out.slots.data_ptr(), out.positions.data_ptr(), out.used.data_ptr(), stream))
    return out


def cache_append(k: torch.Tensor, v: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor,
                 slots: torch.Tensor) -> None:
    """Writes rows k, v (tokens, heads_kv, dim) to the cache's slots (int64); a
    slot outside the cache, such as -1, is skipped."""
    device = k_cache.get_device()
    stream = _stream(device)
    cache, shape = _cache(k_cache, v_cache, device)
    tokens = slots.shape[0]
    want = (tokens, shape[2], shape[3])
    ks, vs = k.stride(), v.stride()
    _need(k.shape == want and v.shape == want, f"k and v must have shape {want}")
    _need(k.dtype == k_cache.dtype and v.dtype == k_cache.dtype, "k and v must have the cache's type")
    _need(k.get_device() == device and v.get_device() == device, "k and v must be on the same device")
    if tokens == 0:
        return
    _need(ks[2] == 1 and vs[2] == 1, "the last dimension of k and v must be contiguous")
    check(lib().fg_cache_append(cache, k.data_ptr(), v.data_ptr(), ks[0], ks[1], vs[0], vs[1],
                                _vector(slots, tokens, torch.int64, device, "slots"), tokens, stream))


def _attention(fn, q, k_cache, v_cache, block_table, q_starts, kv_lens, ids, max_q, scale, window, sinks, out, lse):
    device = q.get_device()
    stream = _stream(device)
    cache, shape = _cache(k_cache, v_cache, device)
    dim = shape[3]
    _need(q.ndim == 3 and q.shape[2] == dim and q.dtype == k_cache.dtype,
          f"q must have shape (tokens, heads, {dim}) and the cache's type")
    tokens, heads, _ = q.shape
    qs = q.stride()
    _need(qs[2] == 1 or tokens == 0, "the last dimension of q must be contiguous")
    requests = kv_lens.shape[0]
    if out is None:
        out = torch.empty((tokens, heads, dim), dtype=q.dtype, device=q.device)
    if lse is None:
        lse = torch.empty((tokens, heads), dtype=torch.float32, device=q.device)
    os_ = out.stride()
    _need(out.shape == q.shape and out.dtype == q.dtype and out.get_device() == device
          and (os_[2] == 1 or tokens == 0),
          "out must have q's shape and type, its last dimension contiguous, on the same device")
    _need(lse.shape == (tokens, heads) and lse.dtype == torch.float32 and lse.is_contiguous()
          and lse.get_device() == device, "lse must be contiguous float32 of shape (tokens, heads) on the same device")
    _need(0 <= sinks < 1 << 31 and -1 <= window < 1 << 31, "window and sinks must be in [0, 2^31)")
    table, row, width = _table(block_table, requests, device)
    starts = _vector(q_starts, requests + 1, torch.int32, device, "q_starts") if q_starts is not None else 0
    lists = nids = ids_ptr = 0
    if ids is not None:
        _need(ids.ndim == 3 and ids.shape[0] == requests and ids.dtype in _IDS and ids.is_contiguous()
              and ids.get_device() == device, f"ids must be contiguous int32 or uint32 of shape ({requests}, lists, K)")
        _, lists, nids = ids.shape
        ids_ptr = ids.data_ptr()
    need = lib().fg_attend_workspace_bytes(dim)
    work = torch.empty(need, dtype=torch.uint8, device=q.device)
    check(fn(cache, _ATTENTION.pack(q.data_ptr(), out.data_ptr(), lse.data_ptr(), qs[0], qs[1], os_[0], os_[1], table, row,
                                    starts, _vector(kv_lens, requests, torch.int32, device, "kv_lens"), ids_ptr,
                                    work.data_ptr(), need, width, requests, tokens, heads, max_q, window, sinks, lists,
                                    nids, scale if scale is not None else dim ** -0.5), stream))
    return out, lse


def attend(q: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor, block_table: torch.Tensor,
           q_starts: torch.Tensor, kv_lens: torch.Tensor, *, max_q: int, scale: float | None = None,
           window: int | None = None, sinks: int = 0, out: torch.Tensor | None = None,
           lse: torch.Tensor | None = None) -> tuple[torch.Tensor, torch.Tensor]:
    """Causal attention of each request's new tokens over its pages.

    q: (tokens, heads, dim), the requests' new tokens one after another;
    q_starts: (requests + 1,) int32, where each begins; kv_lens: (requests,)
    int32, tokens with the new ones, whose keys and values the cache already
    holds; max_q: the most new tokens of a request (a hint: results don't
    depend on it).  scale: dim ** -0.5 unless given.  window: the row at position
    p sees the tokens p - window + 1 .. p and the first `sinks`.
    Returns (out, lse): lse (tokens, heads) float32, the natural logarithm of the
    sum of exponentials.  A row that sees nothing gets 0 and -inf."""
    _need(window is None or window >= 1, "window must be at least 1, or None")
    _need(q_starts is not None, "q_starts is needed")
    _need(0 <= max_q < 1 << 31, "max_q must be in [0, 2^31)")
    return _attention(lib().fg_attend, q, k_cache, v_cache, block_table, q_starts, kv_lens, None, max_q, scale,
                      -1 if window is None else window, sinks, out, lse)


def attend_retrieved(q: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor, block_table: torch.Tensor,
                     kv_lens: torch.Tensor, ids: torch.Tensor, *, window: int, sinks: int = 0,
                     scale: float | None = None, out: torch.Tensor | None = None,
                     lse: torch.Tensor | None = None) -> tuple[torch.Tensor, torch.Tensor]:
    """Attention of one token a request over its first `sinks` tokens, its last
    `window` and the positions in a list, each token once.

    q: (requests, heads, dim), at position kv_lens - 1; ids: (requests, lists, K)
    int32 or uint32, lists a multiple of heads_kv that divides heads (one list for
    each query head, for each key/value head, or between).  An id past the
    request's tokens, among the first or last ones, or equal to the id before it
    adds nothing.  Returns (out, lse) as `attend` does."""
    _need(window >= 0, "window must be at least 0")
    _need(ids is not None, "ids are needed")
    return _attention(lib().fg_attend_retrieved, q, k_cache, v_cache, block_table, None, kv_lens, ids, 1, scale, window,
                      sinks, out, lse)
