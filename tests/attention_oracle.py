"""Attention over a paged cache in 64 bits, one row at a time on the CPU, and how
far a kernel that sums in 32 bits and rounds its weights once may be off it."""
from __future__ import annotations

import numpy as np
import torch

UNIT = {t: torch.finfo(t).eps / 2 for t in (torch.bfloat16, torch.float16)}  # half a step, relative: 2^-8, 2^-11


def make_cache(rng, pages, page, heads_kv, dim, dtype, layout="nhd"):
    shape = (pages, heads_kv, page, dim) if layout == "hnd" else (pages, page, heads_kv, dim)
    k, v = (torch.from_numpy(rng.standard_normal(shape).astype(np.float32)).to(dtype) for _ in range(2))
    return (k.permute(0, 2, 1, 3), v.permute(0, 2, 1, 3)) if layout == "hnd" else (k, v)


def make_table(rng, pages, lens, page, width=None):
    """Each request's pages, drawn without return; -1 past them."""
    need = [-(-n // page) for n in lens]
    width = max(need + [1]) if width is None else width
    order, at = rng.permutation(pages), 0
    table = np.full((len(lens), width), -1, np.int32)
    for r, n in enumerate(need):
        table[r, :min(n, width)] = order[at:at + n][:width]
        at += n
    assert at <= pages
    return torch.from_numpy(table)


def seen_tokens(table, r, kv, pos, page, pages, window, sinks):
    """Positions that the row at `pos` sees, by the definition."""
    out = []
    for j in range(min(kv, pos + 1)):
        if window is not None and not (j > pos - window or j < sinks):
            continue
        if j // page < table.shape[1] and 0 <= int(table[r, j // page]) < pages:
            out.append(j)
    return out


class Oracle:
    """Rows by the definition; `out` and `lse` with a bound on the error of each."""

    def __init__(self, q, k_cache, v_cache, table, scale):
        self.q, self.k, self.v, self.table, self.scale = q, k_cache, v_cache, table.numpy(), scale
        self.pages, self.page, self.heads_kv, self.dim = k_cache.shape
        T, H, D = q.shape
        self.out, self.lse = np.zeros((T, H, D)), np.full((T, H), -np.inf)
        self.out_tol, self.lse_tol = np.zeros((T, H, D)), np.zeros((T, H))
        self.rows = np.zeros(T, bool)

    def row(self, t, h, r, tokens):
        self.rows[t] = True
        if not len(tokens):
            return
        j = np.asarray(tokens, np.int64)
        at, off = torch.from_numpy(self.table[r][j // self.page].astype(np.int64)), torch.from_numpy(j % self.page)
        kv_head = h // (self.q.shape[1] // self.heads_kv)
        k = self.k[at, off, kv_head].double().numpy()
        v = self.v[at, off, kv_head].double().numpy()
        q = self.q[t, h].double().numpy()
        with np.errstate(all="ignore"):
            s = (k @ q) * self.scale
            m = s.max()
            w = np.exp(s - m)
            l = w.sum()
            self.out[t, h] = (w / l) @ v
            self.lse[t, h] = m + np.log(l)
            # 32-bit scores: D products and sums, each off by 2^-24 of the terms' size, and
            # the base-2 scaling of what they give
            ds = float(np.nanmax((np.abs(k) @ np.abs(q)) * self.scale)) * (self.dim + 8) * 2.0 ** -24
            n, u = len(j), UNIT[self.q.dtype]
            spread = (w / l) @ np.abs(v)
            self.lse_tol[t, h] = ds + (n + 8) * 2.0 ** -24 + 2.0 ** -21 * (1 + abs(self.lse[t, h]))
            # weights rounded once (u), the output once (u), 32-bit sums, and the 16-bit
            # floats' smallest weights
            self.out_tol[t, h] = (u + 2 * ds + (n + 8) * 2.0 ** -22) * spread + u * np.abs(self.out[t, h]) * 1.01
            self.out_tol[t, h] += (n * 2.0 ** -25 * np.abs(v).max() if self.q.dtype == torch.float16 else 0) + 2.0 ** -25

    def check(self, out, lse):
        out, lse = out.double().cpu().numpy(), lse.double().cpu().numpy()
        for name, got, want, tol in (("lse", lse, self.lse, self.lse_tol), ("out", out, self.out, self.out_tol)):
            got, want, tol = got[self.rows], want[self.rows], tol[self.rows]
            fine = np.isfinite(want)
            same = (got == want) | (np.isnan(got) & np.isnan(want))
            assert np.all(same[~fine]), (name, "non-finite values differ", np.argwhere(~fine & ~same)[:5])
            assert np.isfinite(got[fine]).all(), (name, "not finite", np.argwhere(fine & ~np.isfinite(got))[:5])
            off = np.abs(got[fine] - want[fine]) - tol[fine]
            assert (off <= 0).all(), (name, float(off.max()), np.argwhere(fine)[off > 0][:5])


def dense(q, k_cache, v_cache, table, q_starts, kv_lens, scale, window=None, sinks=0):
    o = Oracle(q, k_cache, v_cache, table, scale)
    for r, kv in enumerate(kv_lens):
        new = q_starts[r + 1] - q_starts[r]
        for i in range(new):
            tokens = seen_tokens(o.table, r, kv, kv - new + i, o.page, o.pages, window, sinks)
            for h in range(q.shape[1]):
                o.row(q_starts[r] + i, h, r, tokens)
    return o


def retrieved(q, k_cache, v_cache, table, kv_lens, ids, scale, window, sinks):
    o = Oracle(q, k_cache, v_cache, table, scale)
    B, L, K = ids.shape
    per = q.shape[1] // L
    for r, kv in enumerate(kv_lens):
        for h in range(q.shape[1]):
            tokens = [j for j in range(kv) if j < sinks or j >= kv - window]
            row = [int(x) for x in ids[r, h // per]]
            for i, j in enumerate(row):
                if 0 <= j < kv and sinks <= j < kv - window and (i == 0 or row[i - 1] != j):
                    tokens.append(j)
            tokens = [j for j in tokens if j // o.page < o.table.shape[1] and 0 <= int(o.table[r, j // o.page]) < o.pages]
            o.row(r, h, r, tokens)
    return o


def plan(lens, new, table, free, page, max_tokens):
    """cache_plan by its definition; returns (table, q_starts, kv_lens, slots, positions, used)."""
    table, width = table.copy(), table.shape[1]
    starts, slots, positions, used = [0], [], [], 0
    for r, (n, m) in enumerate(zip(lens, new)):
        n, m = max(n, 0), max(m, 0)
        for b in range(min(-(-n // page), width), min(-(-(n + m) // page), width)):
            table[r, b] = free[used] if used < len(free) else -1
            used += 1
        for p in range(n, n + m):
            at = table[r, p // page] if p // page < width else -1
            slots.append(int(at) * page + p % page if at >= 0 else -1)
            positions.append(p)
        starts.append(starts[-1] + m)
    fill = max(0, max_tokens - len(slots))
    return (table, starts, [max(n, 0) + max(m, 0) for n, m in zip(lens, new)], (slots + [-1] * fill)[:max_tokens],
            (positions + [0] * fill)[:max_tokens], used)
