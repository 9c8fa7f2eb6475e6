"""The weights of attention over selected pages go into the product with the values in two
parts of the cache's type, so an output is off by its own rounding and little more: few
tokens with flat weights, whose values cancel; and infinite values, which no part may turn
into something else."""
from __future__ import annotations

import numpy as np
import pytest
import torch

import attention_oracle as A
import blocks_oracle as O
from test_gpu_blocks import KV, MANY, case, ints, some_ids

pytestmark = pytest.mark.gpu

BF, FP = torch.bfloat16, torch.float16
INF = float("inf")


@pytest.fixture(autouse=True)
def _gpu(gpu_available):
    torch.cuda.set_device(0)


class Oracle(O.Oracle):
    """Weights off by the second part's rounding alone: half a step of half a step, and, in float16,
    half of 2^-24 beside a largest weight of 2^15; 32-bit scores and sums; the output's own rounding."""

    def row(self, t, h, r, tokens):
        super().row(t, h, r, tokens)
        if len(tokens):
            j = np.asarray(tokens, np.int64)
            at, off = torch.from_numpy(self.table[r][j // self.page].astype(np.int64)), torch.from_numpy(j % self.page)
            kv_head = h // (self.q.shape[1] // self.heads_kv)
            k, v, q = self.k[at, off, kv_head].double().numpy(), np.abs(self.v[at, off, kv_head].double().numpy()), self.q[t, h].double().numpy()
            s = (k @ q) * self.scale
            w = np.exp(s - s.max())
            ds = float(((np.abs(k) @ np.abs(q)) * self.scale).max()) * (self.dim + 8) * 2.0 ** -24
            n, u = len(j), A.UNIT[self.q.dtype]
            with np.errstate(invalid="ignore"):
                self.out_tol[t, h] = ((u * u + 2 * ds + (n + 8) * 2.0 ** -22) * ((w / w.sum()) @ v) + u * np.abs(self.out[t, h]) * 1.01 +
                                      (n * 2.0 ** -40 * v.max(0) if self.q.dtype == FP else 0) + 2.0 ** -25)


def compare(new, kv, heads, heads_kv, dim, page, dtype, lists, k, seed=0, change=None):
    from flashgann_amd import attention
    q, kc, vc, table, starts = case(seed, new, kv, heads, heads_kv, dim, page, dtype)
    q *= 0.25
    ids = some_ids(np.random.default_rng(seed + 100), new, kv, lists, k, page)
    if change:
        change(q, kc, vc, table, ids)
    out, lse = attention.attend_blocks(q.cuda(), kc.cuda(), vc.cuda(), table.cuda(), ints(starts), ints(kv), ids.cuda())
    o = Oracle(q, kc, vc, table, dim ** -0.5)
    per = heads // lists
    for r, n in enumerate(kv):
        for i in range(new[r]):
            t = starts[r] + i
            for h in range(heads):
                o.row(t, h, r, O.seen_tokens(o.table, r, n, n - new[r] + i, page, o.pages, 1, 1, ids[t, h // per].tolist()))
    o.check(out, lse)


@pytest.mark.parametrize("dtype", (BF, FP))
@pytest.mark.parametrize("dim", (64, 96, 128, 256))
def test_weights_of_few_tokens(dtype, dim):
    """Single tokens, drafts and chunks of 16 rows a tile; 32 rows where there are many."""
    compare([1] * 24, list(range(2, 26)), 8, 2, dim, 4, dtype, 2, 2)
    compare([3, 1, 5, 9], [5, 2, 7, 12], 8, 2, dim, 4, dtype, 2, 2, 1)
    compare(MANY, [m + n % 9 for m, n in zip(MANY, KV)], 16, 8, dim, 4, dtype, 8, 2, 2)


@pytest.mark.parametrize("dtype", (BF, FP))
def test_weights_joined(dtype):
    """Parts of a row that several workgroups take."""
    compare([1], [3000], 8, 2, 128, 16, dtype, 2, 100)


@pytest.mark.parametrize("dtype", (BF, FP))
@pytest.mark.parametrize("new,kv,heads", (([1] * 3, [30, 17, 40], 8), ([6, 1, 2], [30, 17, 40], 8), (MANY, KV, 16)))
@pytest.mark.parametrize("what", (INF, -INF))
def test_infinite_values_under_any_weight(dtype, new, kv, heads, what):
    """An infinite value that a row sees makes its output's channel infinite, also under a weight
    that has no second part (a power of two: one of two equal keys) or a negative one."""
    def odd(q, kc, vc, table, ids):
        for r, n in enumerate(kv):
            for j in range(0, n, 3):
                vc[int(table[r, j // 4]), j % 4, :, j % 32] = what
            if n > 1:
                kc[int(table[r, 0]), 1] = kc[int(table[r, 0]), 0]
    compare(new, kv, heads, 2, 64, 4, dtype, 2, 3, 3, odd)
