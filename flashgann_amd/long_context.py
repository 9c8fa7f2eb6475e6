"""Decoding over a long context whose keys an index holds: search and attention
together.

  python -m flashgann_amd.long_context [--tokens 20000] [--steps 8] [--heads 8]
         [--heads-kv 2] [--dim 128] [--k 128] [--beam 256] [--window 256] [--sinks 4]

One request with `tokens` tokens of synthetic keys and values.  Its prompt is
planned into pages and appended to the cache, and the keys of each key/value head
go into an index (inner product).  Every step then

  searches each head's index with the step's query heads   (Index.search_device),
  gives the new token a slot and appends its key and value (cache_plan, cache_append),
  attends to the first tokens, the last ones and what was found (attend_retrieved),

and compares with attention over the whole context (attend): the share of the
softmax's weight that the retrieved tokens carry, exp(lse - lse of all), and how
far the outputs lie apart.  Tokens newer than the index are the window's, so there
are as many steps as it has tokens at most: past them build the indexes again.

Trained keys cluster and their queries look for few of them; so do these: keys
around shared directions, queries near a key of the past.
"""
from __future__ import annotations

import argparse
import sys
from typing import NamedTuple

import torch

from . import Index, METRIC_IP, attention, builder, datasets
from .codebook import padded_dim_for

PAGE = 16


class Step(NamedTuple):
    """What one step computed, on the GPU."""
    ids: torch.Tensor       # (1, heads, k) what the searches found
    kv_lens: torch.Tensor   # (1,)
    q: torch.Tensor         # (1, heads, dim)
    out: torch.Tensor       # over the retrieved tokens
    lse: torch.Tensor
    all_out: torch.Tensor   # over all tokens
    all_lse: torch.Tensor


class LongContext:
    """The cache, its index per key/value head, and the decode step."""

    def __init__(self, tokens: int, steps: int, heads: int = 8, heads_kv: int = 2, dim: int = 128, k: int = 128,
                 beam: int = 256, window: int = 256, sinks: int = 4, dtype: torch.dtype = torch.bfloat16, seed: int = 1):
        if steps > window:  # a token would leave the window that no index holds
            raise ValueError(f"steps ({steps}) must be at most window ({window})")
        self.heads, self.heads_kv, self.dim, self.k, self.beam = heads, heads_kv, dim, k, beam
        self.steps_left = steps
        self.window, self.sinks, self.dtype = window, sinks, dtype
        self.g = torch.Generator(device="cuda")
        self.g.manual_seed(seed)
        pages = -(-(tokens + steps) // PAGE) + 1
        shape = (pages, PAGE, heads_kv, dim)
        self.k_cache, self.v_cache = (torch.zeros(shape, dtype=dtype, device="cuda") for _ in range(2))
        self.table = torch.full((1, pages), -1, dtype=torch.int32, device="cuda")
        self.free = torch.randperm(pages, generator=self.g, device="cuda").to(torch.int32)
        self.lens = torch.zeros(1, dtype=torch.int32, device="cuda")
        # the prompt's keys and values
        themes = torch.randn((64, heads_kv, dim), generator=self.g, device="cuda")
        pick = torch.randint(64, (tokens,), generator=self.g, device="cuda")
        keys = (themes[pick] + 0.6 * self._randn(tokens, heads_kv, dim)).to(dtype)
        values = self._randn(tokens, heads_kv, dim).to(dtype)
        self._append(keys, values)
        # an index of each head's keys: position p of the context is row p
        signs = datasets.signs_for(padded_dim_for(dim), 1)
        self.indexes = [Index.from_codebook(builder.build_codebook(keys[:, h].float().contiguous(), 32, signs, use_ip=True,
                                                                   device="cuda"), metric=METRIC_IP) for h in range(heads_kv)]
        self.keys = keys

    def close(self) -> None:
        for ix in self.indexes:
            ix.close()

    def _randn(self, *shape: int) -> torch.Tensor:
        return torch.randn(shape, generator=self.g, device="cuda")

    def _append(self, keys: torch.Tensor, values: torch.Tensor) -> attention.CachePlan:
        new = torch.full((1,), keys.shape[0], dtype=torch.int32, device="cuda")
        plan = attention.cache_plan(self.lens, new, self.table, self.free, page_size=PAGE, max_tokens=keys.shape[0])
        attention.cache_append(keys, values, self.k_cache, self.v_cache, plan.slots)
        # the pages handed out move to the list's end, where no later step reaches; on the GPU
        at = (torch.arange(self.free.shape[0], device="cuda") + plan.used) % self.free.shape[0]
        self.free, self.lens = self.free[at], plan.kv_lens
        return plan

    def step(self) -> Step:
        if self.steps_left == 0:
            raise RuntimeError("no step is left: the cache and the window are planned for `steps`")
        self.steps_left -= 1
        group = self.heads // self.heads_kv
        near = torch.randint(self.keys.shape[0], (self.heads,), generator=self.g, device="cuda")
        head = torch.arange(self.heads, device="cuda") // group
        q = (2.0 * self.keys[near, head].float() + self._randn(self.heads, self.dim))[None].to(self.dtype)
        ids = torch.empty((1, self.heads, self.k), dtype=torch.int32, device="cuda")
        queries = q[0].float()
        stream = torch.cuda.current_stream().cuda_stream
        for h, ix in enumerate(self.indexes):
            ix.search_device(queries[h * group:].data_ptr(), group, self.k, self.beam, ids[0, h * group:].data_ptr(), stream=stream)
        plan = self._append(self._randn(1, self.heads_kv, self.dim).to(self.dtype), self._randn(1, self.heads_kv, self.dim).to(self.dtype))
        out, lse = attention.attend_retrieved(q, self.k_cache, self.v_cache, self.table, plan.kv_lens, ids, window=self.window,
                                              sinks=self.sinks)
        all_out, all_lse = attention.attend(q, self.k_cache, self.v_cache, self.table, plan.q_starts, plan.kv_lens, max_q=1)
        return Step(ids, plan.kv_lens, q, out, lse, all_out, all_lse)


def main(argv: list[str] | None = None) -> int:
    ap = argparse.ArgumentParser(prog="python -m flashgann_amd.long_context", description=__doc__.splitlines()[0])
    for name, value in (("tokens", 20000), ("steps", 8), ("heads", 8), ("heads-kv", 2), ("dim", 128), ("k", 128), ("beam", 256),
                        ("window", 256), ("sinks", 4)):
        ap.add_argument("--" + name, type=int, default=value)
    args = vars(ap.parse_args(argv))
    if args["steps"] > args["window"]:
        ap.error("--steps must be at most --window")
    if not torch.cuda.is_available():
        raise SystemExit("no GPU is visible")
    ctx = LongContext(**args)
    try:
        for i in range(args["steps"]):
            s = ctx.step()
            share = torch.exp(s.lse - s.all_lse)
            off = (s.out.float() - s.all_out.float()).norm() / s.all_out.float().norm()
            print(f"step {i}: {int(s.kv_lens)} tokens, weight on the retrieved ones {share.mean():.4f} (least {share.min():.4f}), "
                  f"output off by {off:.4f}", flush=True)
    finally:
        ctx.close()
    return 0


if __name__ == "__main__":
    sys.exit(main())
