"""Prints, as JSON, the kernels that the batches of the tests of attention over selected pages
run: a program of its own, so that the profiler stays out of the tests' process."""
from __future__ import annotations

import json
import os
import re
import sys

import numpy as np
import torch
from torch.profiler import ProfilerActivity, profile

HERE = os.path.dirname(os.path.abspath(__file__))
sys.path[:0] = [HERE, os.path.dirname(HERE)]

from flashgann_amd import attention  # noqa: E402
from test_gpu_blocks import KV, MANY, case, ints, some_ids  # noqa: E402

FEW = ([1, 0, 3, 21, 17, 1], [9, 77, 3, 90, 217, 260])


def far(kv):
    return [5] + [2] * 7 + [9], [kv - 11 * r for r in range(9)]


# name: (new, kv), heads, heads_kv, lists, dim, page, k
BATCHES = {
    **{f"many {h} over {hk}, {lists} lists, dim {d}": ((MANY, KV), h, hk, lists, d, page, 3)
       for h, hk, lists, d, page in ((16, 8, 8, 128, 16), (24, 8, 8, 96, 24), (16, 2, 16, 64, 5), (32, 8, 8, 128, 4), (8, 8, 8, 96, 1), (16, 8, 8, 64, 8))},
    "many heads of a list": ((MANY * 2, KV * 2), 80, 2, 2, 64, 8, 4),
    **{f"many windows, pages of {page}": (far(kv), 16, 16, 16, 64, page, k) for page, kv, k in ((1, 2500, 20), (2, 4000, 5), (8, 9000, 3), (200, 5000, 2), (64, 3000, 4))},
    "few": (FEW, 8, 2, 2, 128, 16, 5),
    "few, dim 256": (FEW, 6, 1, 2, 256, 8, 5),
    "single tokens": (([1] * 60, [300] * 60), 8, 2, 2, 128, 16, 6),
    "one token, many pages": (([1], [9000]), 8, 2, 2, 128, 16, 200),
}


def main() -> None:
    names = {}
    for name, ((new, kv), heads, heads_kv, lists, dim, page, k) in BATCHES.items():
        q, kc, vc, table, starts = case(1, new, kv, heads, heads_kv, dim, page, torch.bfloat16)
        args = (q.cuda(), kc.cuda(), vc.cuda(), table.cuda(), ints(starts), ints(kv), some_ids(np.random.default_rng(2), new, kv, lists, k, page).cuda())
        torch.cuda.synchronize()
        with profile(activities=[ProfilerActivity.CUDA]) as p:
            attention.attend_blocks(*args)
            torch.cuda.synchronize()
        names[name] = [m.group(1) for e in p.events() if (m := re.search(r"\b(fg_blocks\w*_kernel)<", e.name))]
    print(json.dumps(names), flush=True)


if __name__ == "__main__":
    main()
