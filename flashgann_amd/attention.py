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
libflashgann.so; there is no fallback.  Wrong types, shapes or devices raise
ValueError, what the library refuses FlashGannError.  Nothing here has a gradient:
with autograd on, a tensor that requires one is refused (ValueError).
"""
from __future__ import annotations

import sys
from typing import NamedTuple

import torch

from . import _lib

_lib.lib()  # its message where the library is missing
try:
    from . import _attention  # (csrc/torch_attention.cpp)
except ImportError as e:
    raise ImportError(f"flashgann_amd._attention is not built for {sys.executable}: make -C flashgann_amd/csrc "
                      f"PYTHON={sys.executable} ({e})") from e

__all__ = ["CachePlan", "cache_plan", "cache_append", "attend", "attend_retrieved"]


class CachePlan(NamedTuple):
    """What `cache_plan` returns."""
    q_starts: torch.Tensor   # (requests + 1,) int32
    kv_lens: torch.Tensor    # (requests,) int32
    slots: torch.Tensor      # (max_tokens,) int64
    positions: torch.Tensor  # (max_tokens,) int32
    used: torch.Tensor       # (1,) int32


def cache_plan(lens: torch.Tensor, new_lens: torch.Tensor, block_table: torch.Tensor, free_pages: torch.Tensor, *,
               page_size: int, max_tokens: int) -> CachePlan:
    """Gives each request the pages that its new tokens need, in one launch.

    lens, new_lens: (requests,) int32, tokens held and tokens to come;
    block_table: (requests, width) int32, written in place where a request gets
    a page (-1 once free_pages is used up); free_pages: (n,) int32;
    max_tokens: the length of the slot map, at least the sum of new_lens for
    every token to have an entry.  Entries past the last token hold slot -1.
    `used` is the number of pages taken: drop so many from free_pages.  1 to 4,096
    requests a call."""
    return CachePlan(*_attention.cache_plan(lens, new_lens, block_table, free_pages, page_size, max_tokens))


def cache_append(k: torch.Tensor, v: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor,
                 slots: torch.Tensor) -> None:
    """Writes rows k, v (tokens, heads_kv, dim) to the cache's slots (int64); a
    slot outside the cache, such as -1, is skipped; no two rows may share a slot."""
    _attention.cache_append(k, v, k_cache, v_cache, slots)


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
    sum of exponentials.  A row that sees nothing gets 0 and -inf; rows outside every
    request, such as a padded batch's last ones, are left as they are, uninitialised
    unless out and lse are given.  0 to 65,536 requests a call.

    The host does not know the lengths: a block_table (and window) with room for up to 512
    tokens a request spares the call its second kernel, 3 to 6 us, and a workspace of up
    to 68 MB, so pass the columns in use, block_table[:, :n]."""
    return _attention.attend(q, k_cache, v_cache, block_table, q_starts, kv_lens, None, max_q, scale, window, sinks, out, lse)


def attend_retrieved(q: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor, block_table: torch.Tensor,
                     kv_lens: torch.Tensor, ids: torch.Tensor, *, window: int, sinks: int = 0,
                     scale: float | None = None, out: torch.Tensor | None = None,
                     lse: torch.Tensor | None = None) -> tuple[torch.Tensor, torch.Tensor]:
    """Attention of one token a request over its first `sinks` tokens, its last
    `window` and the positions in a list.

    q: (requests, heads, dim), at position kv_lens - 1; ids: (requests, lists, K)
    int32 or uint32, lists a multiple of heads_kv that divides heads (one list for
    each query head, for each key/value head, or between).  An id past the
    request's tokens, among the first or last ones, or equal to the id before it
    adds nothing; other repeats count again, so sort a list merged of several searches.
    Returns (out, lse) as `attend` does."""
    if ids is None:
        raise ValueError("ids are needed")
    return _attention.attend(q, k_cache, v_cache, block_table, None, kv_lens, ids, 1, scale, window, sinks, out, lse)
