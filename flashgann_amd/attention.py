"""A paged key/value cache on the GPU and the attention that reads it, for
programs that answer with what a search found.

  cache_plan        block tables and slot maps from request lengths
  cache_append      new keys and values into their slots
  attend            a chunk of new tokens (one to many a request) over the
                    cache, with or without a sliding window and first tokens
                    that stay visible
  attend_retrieved  one token a request over the first tokens, the last ones
                    and the ids that `Index.search_device` returned
  cache_bounds      bounds of the keys of each page that new tokens filled
  select_blocks     the pages whose bounds promise each query the most: the search
                    of a context that no index is built for
  attend_blocks     new tokens over the selected pages, the first and the last ones
  cache_weigh       the attention weight that each cached token has drawn
  cache_evict       requests back to a budget of tokens, the heaviest kept

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

__all__ = ["CacheEviction", "CachePlan", "attend", "attend_blocks", "attend_retrieved", "cache_append", "cache_bounds", "cache_evict",
           "cache_plan", "cache_weigh", "select_blocks"]


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


def cache_bounds(k_cache: torch.Tensor, slots: torch.Tensor, bounds: torch.Tensor, scales: torch.Tensor) -> None:
    """Bounds of the keys of each page whose last slot is among `slots` (int64), such as
    those that `cache_append` has just written: call it after with the same slots.

    bounds: (pages, heads_kv, 2, dim) int8, scales: (pages, heads_kv) float32, contiguous.
    bounds[p, h, 0] * scales[p, h] is no less than any key of the page, bounds[p, h, 1] *
    scales[p, h] no more; scales are powers of two, the least of which 127 reach the
    largest key.  A page with an infinity or NaN gets scale infinity.  Where keys are written
    again or moved (`cache_evict`), pass their pages' last slots once more."""
    _attention.cache_bounds(k_cache, slots, bounds, scales)


def select_blocks(q: torch.Tensor, bounds: torch.Tensor, scales: torch.Tensor, block_table: torch.Tensor, q_starts: torch.Tensor,
                  kv_lens: torch.Tensor, *, page_size: int, k: int, lists: int | None = None, first_blocks: int = 1,
                  last_blocks: int = 1) -> torch.Tensor:
    """The k pages that promise each row of q the most: (tokens, lists, k) int32, page
    numbers within the request (its block b holds tokens b * page_size and on), ascending,
    -1 behind them where fewer can be selected.

    q, q_starts and kv_lens as for `attend`.  The row at position p, in block c, selects
    from first_blocks <= b <= c - last_blocks, the blocks that `attend_blocks` does not
    read anyway.  lists: a multiple of heads_kv that divides heads, heads_kv unless given; the
    query heads of a list select together, by the sum over them of the most that the bounds
    leave for q . key, with the summed queries in 8 bits too.  Scores are exact, and equal
    ones go to the lower block.  Rows outside every request are left uninitialised.  1 to 4,096
    pages a list; up to 4,194,304 rows a call.

    Pass the columns in use, block_table[:, :n]: the call is run, and takes up to 1 GiB of
    workspace, by what the table has room for (4,096 rows over 1,000 pages 99 us, in a table of
    8,192 columns 297 us and 1 GiB)."""
    return _attention.select_blocks(q, bounds, scales, block_table, q_starts, kv_lens, page_size, k, lists, first_blocks, last_blocks)


def attend_blocks(q: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor, block_table: torch.Tensor, q_starts: torch.Tensor,
                  kv_lens: torch.Tensor, ids: torch.Tensor, *, first_blocks: int = 1, last_blocks: int = 1,
                  scale: float | None = None, out: torch.Tensor | None = None,
                  lse: torch.Tensor | None = None) -> tuple[torch.Tensor, torch.Tensor]:
    """Causal attention of each request's new tokens over the pages on a list, the
    first `first_blocks` of its context and the last `last_blocks` (the row's own among them).

    ids: (tokens, lists, k) int32 as `select_blocks` returns them, a list for each row; an
    id that is not above all before it in its list, or names one of the first or last blocks
    or one after them, adds nothing.  Everything else, and (out, lse), as for `attend`.  A
    block_table of more than 4,096 columns makes chunks take twice as long: pass those in use."""
    return _attention.attend_blocks(q, k_cache, v_cache, block_table, q_starts, kv_lens, ids, first_blocks, last_blocks, scale, out, lse)


def cache_weigh(q: torch.Tensor, k_cache: torch.Tensor, block_table: torch.Tensor, q_starts: torch.Tensor, kv_lens: torch.Tensor,
                lse: torch.Tensor, weights: torch.Tensor, known: torch.Tensor, *, scale: float | None = None) -> None:
    """Adds to each cached token's weight what these rows of q gave it: the sum over the
    rows that see it and the query heads of its key/value head of exp(scale q . k - lse).

    q, q_starts, kv_lens: as for `attend` (all new tokens, or a request's last ones only);
    lse: what `attend` returned for them, without a window, so that a row's weights sum to 1
    (with `attend_blocks`' they are shares of the selected pages, and a token outside those may
    count for more than 1).  weights: (pages, heads_kv,
    page_size) float32, contiguous, written in place.  known: (requests,) int32, the tokens
    that have a weight already (the length before this step, say): those from there on are
    set instead of added to.  Tokens that requests of the call share get all their sums if
    each knows them; one that has to be set may belong to one request only."""
    _attention.cache_weigh(q, k_cache, block_table, q_starts, kv_lens, lse, weights, known, scale)


class CacheEviction(NamedTuple):
    """What `cache_evict` returns."""
    kv_lens: torch.Tensor   # (requests,) int32
    freed: torch.Tensor     # (requests * width,) int32
    released: torch.Tensor  # (1,) int32


def cache_evict(k_cache: torch.Tensor, v_cache: torch.Tensor, weights: torch.Tensor, block_table: torch.Tensor, kv_lens: torch.Tensor,
                *, budget: int, window: int, sinks: int = 0) -> CacheEviction:
    """Takes each request of more than `budget` tokens back to it: its first `sinks` and last
    `window` tokens stay, and for each key/value head those of largest weight between them
    (equal ones: the earlier).

    Kept tokens below place budget - window stay where they are, those above it move into the
    places that became free there, the last `window` behind them: keys, values and
    weights, in place.  So a place's heads may hold different tokens, and the cache is for
    `attend` without a window from then on; keys hold their own positions.  Returns the
    new lengths, the pages that are free now (the first `released` entries of `freed`, -1
    behind them) and their number; block_table keeps its entries, which `cache_plan` writes
    over as the request grows.  A token whose place, or new place, has no page (cache_plan ran out
    of them: used > the free pages) is lost, and entries without one are among `freed` as they
    are: leave them out of the free pages.  No page may be named twice, and k_cache and v_cache may share
    no memory, with each other or between their own places.  1 to 4,096 requests a call.

    Kernels and workspace (8 bytes a request, head and token that the table names past the budget, or
    of the budget if that is less) follow what the table has room for: pass the columns in use,
    block_table[:, :n]."""
    return CacheEviction(*_attention.cache_evict(k_cache, v_cache, weights, block_table, kv_lens, budget, window, sinks))
