"""Bounds of pages, selection by them, attention over selected pages, drawn weights and
eviction by their definitions, in 64 bits and whole numbers on the CPU."""
from __future__ import annotations

import math

import numpy as np
import torch

import attention_oracle as A


def power_for(most):
    """The least power of two, 2^-126 at least, of which 127 reach `most`."""
    s = -126
    while 127 * 2.0 ** s < most:
        s += 1
    return 2.0 ** s


def bounds(k_cache, pages):
    """{(page, head): (codes (2, dim), scale)} of the pages named."""
    out = {}
    for p in pages:
        for h in range(k_cache.shape[2]):
            k = k_cache[p, :, h].double().numpy()
            if not np.isfinite(k).all():
                out[p, h] = (np.zeros((2, k.shape[1]), np.int64), math.inf)
                continue
            scale = power_for(np.abs(k).max())
            out[p, h] = (np.stack([np.ceil(k.max(0) / scale), np.floor(k.min(0) / scale)]).astype(np.int64), scale)
    return out


def full_pages(slots, page, pages):
    return sorted({s // page for s in slots if 0 <= s < pages * page and s % page == page - 1})


def query_codes(q):
    """(group, dim) of one list -> 2 dim integers."""
    up, down = np.zeros(q.shape[1], np.float32), np.zeros(q.shape[1], np.float32)
    with np.errstate(all="ignore"):
        for row in q.float().numpy():  # in 32 bits, in order
            up = up + np.where(row < 0, np.float32(0), row)
            down = down + np.where(row > 0, np.float32(0), row)
    both = np.concatenate([up, down]).astype(np.float64)
    if not np.isfinite(both).all():
        return np.zeros(len(both), np.int64)
    return np.rint(both / power_for(np.abs(both).max())).astype(np.int64)


def select(q, codes, scales, table, q_starts, kv_lens, page, k, lists, first, last):
    """ids (tokens, lists, k); codes (pages, heads_kv, 2, dim), scales (pages, heads_kv)."""
    T, heads, _ = q.shape
    pages, heads_kv = scales.shape
    ids = np.full((T, lists, k), -1, np.int64)
    per, codes, scales = heads // lists, codes.long().numpy(), scales.numpy()
    for r, kv in enumerate(kv_lens):
        new = q_starts[r + 1] - q_starts[r]
        for i in range(new):
            pos = max(kv, 0) - new + i
            for lst in range(lists):
                h = lst // (lists // heads_kv)
                c = query_codes(q[q_starts[r] + i, lst * per:(lst + 1) * per])
                scored = []
                for b in range(first, min(pos // page - last + 1, table.shape[1]) if pos >= 0 else 0):
                    at = int(table[r, b])
                    if 0 <= at < pages:
                        whole = int((c * codes[at, h].reshape(-1)).sum())
                        assert abs(whole) < 2 ** 24
                        with np.errstate(over="ignore"):
                            score = np.float32(math.inf) if math.isinf(scales[at, h]) else np.float32(whole) * scales[at, h]
                        scored.append((-float(score), b))
                best = sorted(b for _, b in sorted(scored)[:k])
                ids[q_starts[r] + i, lst, :len(best)] = best
    return ids


def seen_tokens(table, r, kv, pos, page, pages, first, last, ids):
    out, c, most = [], pos // page, -1
    listed = set()
    for x in ids:
        if x > most:
            most = x
            if first <= x <= c - last:
                listed.add(int(x))
    for j in range(min(kv, pos + 1)):
        b = j // page
        if (b < first or b > c - last or b in listed) and b < table.shape[1] and 0 <= int(table[r, b]) < pages:
            out.append(j)
    return out


class Oracle(A.Oracle):
    """The same bounds, channel by channel: a channel's output is a sum of that channel's values
    alone, so what float16 loses of its weights (n tokens, 2^-25 each) is bounded by the largest
    value there, and an infinity or NaN in another channel takes no part in it."""

    def row(self, t, h, r, tokens):
        super().row(t, h, r, tokens)
        if len(tokens) and self.q.dtype == torch.float16:
            j = np.asarray(tokens, np.int64)
            at, off = torch.from_numpy(self.table[r][j // self.page].astype(np.int64)), torch.from_numpy(j % self.page)
            kv_head = h // (self.q.shape[1] // self.heads_kv)
            v = np.abs(self.v[at, off, kv_head].double().numpy())
            k, q = np.abs(self.k[at, off, kv_head].double().numpy()), self.q[t, h].double().numpy()
            with np.errstate(all="ignore"):
                s = (self.k[at, off, kv_head].double().numpy() @ q) * self.scale
                w = np.exp(s - s.max())
                ds = float(np.nanmax((k @ np.abs(q)) * self.scale)) * (self.dim + 8) * 2.0 ** -24
                n, u = len(j), A.UNIT[self.q.dtype]
                spread = (w / w.sum()) @ v
                self.out_tol[t, h] = ((u + 2 * ds + (n + 8) * 2.0 ** -22) * spread + u * np.abs(self.out[t, h]) * 1.01 +
                                      n * 2.0 ** -25 * v.max(0) + 2.0 ** -25)


def attend(q, k_cache, v_cache, table, q_starts, kv_lens, ids, scale, first, last):
    o = Oracle(q, k_cache, v_cache, table, scale)
    per = q.shape[1] // ids.shape[1]
    for r, kv in enumerate(kv_lens):
        new = q_starts[r + 1] - q_starts[r]
        for i in range(new):
            for h in range(q.shape[1]):
                t = q_starts[r] + i
                o.row(t, h, r, seen_tokens(o.table, r, kv, kv - new + i, o.page, o.pages, first, last, ids[t, h // per].tolist()))
    return o


def weigh(q, k_cache, table, q_starts, kv_lens, lse, weights, known, scale):
    """(weights, a bound on the error of each)."""
    pages, page, heads_kv, dim = k_cache.shape
    w, tol = weights.double().numpy().copy(), np.zeros(weights.shape)
    per = q.shape[1] // heads_kv
    set_already = np.zeros(weights.shape, bool)
    for r, kv in enumerate(kv_lens):
        new = q_starts[r + 1] - q_starts[r]
        for j in range(min(max(kv, 0), table.shape[1] * page)):
            p = int(table[r, j // page])
            if not 0 <= p < pages:
                continue
            for h in range(heads_kv):
                at = (p, h, j % page)
                total = off = 0.0
                rows = [i for i in range(new) if kv - new + i >= j]
                if rows:
                    t = torch.tensor([q_starts[r] + i for i in rows])
                    qs = q[t][:, h * per:(h + 1) * per].double().numpy().reshape(-1, dim)
                    z = lse[t][:, h * per:(h + 1) * per].double().numpy().reshape(-1)
                    k = k_cache[p, j % page, h].double().numpy()
                    qs, z = qs[z != -np.inf], z[z != -np.inf]
                    with np.errstate(all="ignore"):
                        s = qs @ k * scale
                        e = np.exp(s - z)
                        # the score's products and sums in 32 bits, the base-2 difference (two
                        # roundings of its terms), the exponential (an ulp), the sum over rows
                        d = (np.abs(qs) @ np.abs(k) * scale) * (dim + 8) * 2.0 ** -24 + (np.abs(s) + np.abs(z) + 2) * 2.0 ** -22
                        total = float(e.sum())
                        off = float((e * d).sum()) + total * (len(e) + 4) * 2.0 ** -24
                if j < known[r]:
                    w[at] += total
                    tol[at] += off + abs(w[at]) * 2.0 ** -23
                else:
                    assert not set_already[at]
                    set_already[at] = True
                    w[at], tol[at] = total, off
    return w, tol


def evict(k_cache, v_cache, weights, table, kv_lens, budget, window, sinks):
    """(k, v, weights, kv_lens, freed, released), by moving single rows."""
    pages, page, heads_kv, _ = k_cache.shape
    k, v, w = k_cache.clone(), v_cache.clone(), weights.clone()
    width = table.shape[1]
    lens, freed = [], []

    def slot(r, j):
        p = int(table[r, j // page])
        return (p, j % page) if 0 <= p < pages else None

    for r, n in enumerate(kv_lens):
        n = min(max(n, 0), width * page)
        lens.append(min(n, budget))
        freed += table[r, -(-lens[-1] // page):-(-n // page)].tolist()
        if n <= budget:
            continue
        keep, end = budget - window, n - window
        for h in range(heads_kv):
            def drawn(j):
                s = slot(r, j)
                if s is None:
                    return (1, 0.0)
                x = float(weights[s[0], h, s[1]])
                return (0, -(math.inf if math.isnan(x) else x))
            order = sorted(range(sinks, end), key=lambda j: (*drawn(j), j))
            stay = set(range(sinks)) | set(order[:keep - sinks])
            moves = list(zip(sorted(j for j in stay if j >= keep), (j for j in range(keep) if j not in stay)))
            moves += [(end + i, keep + i) for i in range(window)]
            for a, b in moves:
                a, b = slot(r, a), slot(r, b)
                if a is not None and b is not None:
                    k[b[0], b[1], h], v[b[0], b[1], h] = k[a[0], a[1], h], v[a[0], a[1], h]
                    w[b[0], h, b[1]] = w[a[0], h, a[1]]
    total = len(freed)
    return k, v, w, lens, freed + [-1] * (len(kv_lens) * width - total), total
