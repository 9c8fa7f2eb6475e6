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
_ATTENTION = struct.Struct("3Q4qQq3Q5Ii3If")  # fg_attention


# the current stream's handle without a Stream object around it, a microsecond less a call
_raw_stream = getattr(torch._C, "_cuda_getCurrentRawStream", None) or (lambda d: torch.cuda.current_stream(d).cuda_stream)


class CachePlan(NamedTuple):
    """What `cache_plan` returns."""
    q_starts: torch.Tensor   # (requests + 1,) int32
    kv_lens: torch.Tensor    # (requests,) int32
    slots: torch.Tensor      # (max_tokens,) int64
    positions: torch.Tensor  # (max_tokens,) int32
    used: torch.Tensor       # (1,) int32


def _stream(device: int) -> int:
    if device < 0 or device != torch.cuda.current_device():
        raise ValueError("tensors must be on the current CUDA device")
    return _raw_stream(device)


def _vector(t: torch.Tensor, n: int, dtype: torch.dtype, device: int, name: str) -> int:
    if t.shape != (n,) or t.dtype != dtype or t.get_device() != device or not t.is_contiguous():
        raise ValueError(f"{name} must be a contiguous {dtype} vector of {n} on the same device")
    return t.data_ptr()


def _cache(k: torch.Tensor, v: torch.Tensor, device: int) -> tuple[bytes, torch.Size]:
    shape, dtype = k.shape, k.dtype
    if len(shape) != 4 or v.shape != shape:
        raise ValueError("k_cache and v_cache must have shape (pages, page_size, heads_kv, dim)")
    if dtype not in _DTYPES or v.dtype != dtype:
        raise ValueError("k_cache and v_cache must be bfloat16 or float16")
    if k.get_device() != device or v.get_device() != device:
        raise ValueError("k_cache and v_cache must be on the same device")
    k0, k1, k2, k3 = k.stride()
    v0, v1, v2, v3 = v.stride()
    if k3 != 1 or v3 != 1:
        raise ValueError("the last dimension of k_cache and v_cache must be contiguous")
    return _CACHE.pack(k.data_ptr(), v.data_ptr(), k0, k1, k2, v0, v1, v2, *shape, _DTYPES[dtype], 0), shape


def _table(t: torch.Tensor, requests: int, device: int) -> tuple[int, int, int]:
    shape, stride = t.shape, t.stride()
    if (t.dtype != torch.int32 or len(shape) != 2 or shape[0] != requests or t.get_device() != device
            or (stride[1] != 1 and shape[1] > 1) or stride[0] < 0):
        raise ValueError(f"block_table must be int32 of shape ({requests}, width), its rows contiguous, on the same device")
    return t.data_ptr(), stride[0], shape[1]


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
    stream = _stream(device)
    if lens.ndim != 1 or free_pages.ndim != 1:
        raise ValueError("lens and free_pages must be vectors")
    if not 0 <= max_tokens < 1 << 31 or not 1 <= page_size < 1 << 31:
        raise ValueError("page_size must be in [1, 2^31), max_tokens in [0, 2^31)")
    requests, nfree = lens.shape[0], free_pages.shape[0]
    table, row, width = _table(block_table, requests, device)
    # one allocation for the 32-bit outputs
    q_starts, kv_lens, positions, used = torch.empty(2 * requests + max_tokens + 2, dtype=torch.int32, device=lens.device).split(
        (requests + 1, requests, max_tokens, 1))
    slots = torch.empty(max_tokens, dtype=torch.int64, device=lens.device)
    check(lib().fg_cache_plan(_vector(lens, requests, torch.int32, device, "lens"),
                              _vector(new_lens, requests, torch.int32, device, "new_lens"), requests, table, row, width,
                              _vector(free_pages, nfree, torch.int32, device, "free_pages"), nfree, page_size, max_tokens,
                              q_starts.data_ptr(), kv_lens.data_ptr(), slots.data_ptr(), positions.data_ptr(),
                              used.data_ptr(), stream))
    return CachePlan(q_starts, kv_lens, slots, positions, used)


def cache_append(k: torch.Tensor, v: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor,
                 slots: torch.Tensor) -> None:
    """Writes rows k, v (tokens, heads_kv, dim) to the cache's slots (int64); a
    slot outside the cache, such as -1, is skipped."""
    device = k_cache.get_device()
    stream = _stream(device)
    cache, (_, _, heads_kv, dim) = _cache(k_cache, v_cache, device)
    tokens = slots.shape[0]
    if k.shape != (tokens, heads_kv, dim) or v.shape != k.shape:
        raise ValueError(f"k and v must have shape ({tokens}, {heads_kv}, {dim})")
    if k.dtype != k_cache.dtype or v.dtype != k_cache.dtype:
        raise ValueError("k and v must have the cache's type")
    if k.get_device() != device or v.get_device() != device:
        raise ValueError("k and v must be on the same device")
    if tokens == 0:
        return
    k0, k1, k2 = k.stride()
    v0, v1, v2 = v.stride()
    if k2 != 1 or v2 != 1:
        raise ValueError("the last dimension of k and v must be contiguous")
    check(lib().fg_cache_append(cache, k.data_ptr(), v.data_ptr(), k0, k1, v0, v1,
                                _vector(slots, tokens, torch.int64, device, "slots"), tokens, stream))


def _attention(fn, q, k_cache, v_cache, block_table, q_starts, kv_lens, ids, max_q, scale, window, sinks, out, lse):
    device = q.get_device()
    stream = _stream(device)
    cache, (_, _, _, dim) = _cache(k_cache, v_cache, device)
    shape, dtype, where = q.shape, q.dtype, q.device
    if len(shape) != 3 or shape[2] != dim or dtype != k_cache.dtype:
        raise ValueError(f"q must have shape (tokens, heads, {dim}) and the cache's type")
    tokens, heads, _ = shape
    q0, q1, q2 = q.stride()
    if q2 != 1 and tokens:
        raise ValueError("the last dimension of q must be contiguous")
    if out is None:
        out = torch.empty(tokens, heads, dim, dtype=dtype, device=where)
        o0, o1 = heads * dim, dim
    else:
        o0, o1, o2 = out.stride()
        if out.shape != shape or out.dtype != dtype or out.get_device() != device or (o2 != 1 and tokens):
            raise ValueError("out must have q's shape and type, its last dimension contiguous, on the same device")
    if lse is None:
        lse = torch.empty(tokens, heads, dtype=torch.float32, device=where)
    elif (lse.shape != (tokens, heads) or lse.dtype != torch.float32 or lse.get_device() != device
          or not lse.is_contiguous()):
        raise ValueError("lse must be contiguous float32 of shape (tokens, heads) on the same device")
    if not 0 <= sinks < 1 << 31 or not -1 <= window < 1 << 31:
        raise ValueError("window and sinks must be below 2^31, sinks not negative")
    if kv_lens.ndim != 1:
        raise ValueError("kv_lens must be a vector")
    requests = kv_lens.shape[0]
    table, row, width = _table(block_table, requests, device)
    starts = lists = nids = found = 0
    if ids is None:
        starts = _vector(q_starts, requests + 1, torch.int32, device, "q_starts")
    else:
        if (ids.ndim != 3 or ids.shape[0] != requests or ids.dtype not in _IDS or ids.get_device() != device
                or not ids.is_contiguous()):
            raise ValueError(f"ids must be contiguous int32 or uint32 of shape ({requests}, lists, K) on the same device")
        _, lists, nids = ids.shape
        found = ids.data_ptr()
    args = _ATTENTION.pack(q.data_ptr(), out.data_ptr(), lse.data_ptr(), q0, q1, o0, o1, table, row, starts,
                           _vector(kv_lens, requests, torch.int32, device, "kv_lens"), found, width, requests, tokens, heads,
                           max_q, window, sinks, lists, nids, dim ** -0.5 if scale is None else scale)
    need = lib().fg_attend_workspace_bytes(cache, args)
    work = torch.empty(need, dtype=torch.uint8, device=where).data_ptr() if need > 0 else 0
    check(fn(cache, args, work, need if need > 0 else 0, stream))
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
    if window is not None and window < 1:
        raise ValueError("window must be at least 1, or None")
    if q_starts is None or not 0 <= max_q < 1 << 31:
        raise ValueError("q_starts is needed, and max_q in [0, 2^31)")
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
    if window < 0 or ids is None:
        raise ValueError("ids are needed, and a window of at least 0")
    return _attention(lib().fg_attend_retrieved, q, k_cache, v_cache, block_table, None, kv_lens, ids, 1, scale, window,
                      sinks, out, lse)
