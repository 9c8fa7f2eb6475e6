"""How the attention kernels deal their items out, in whole numbers: what a test's
sizes make a workgroup do.  (The kernels cut in 32-bit floats, a unit off at most.)"""
from __future__ import annotations

from typing import NamedTuple

TILES = dict(item_tokens=256, unit=256, workgroups=256)  # fg_tiles_kernel, rows 256 (128 at dim 256)
FEW = dict(item_tokens=128, unit=128, workgroups=512)    # fg_rows_kernel, rows 16


class Piece(NamedTuple):
    request: int
    list: int
    block: int
    rows: int      # of the item
    t_lo: int      # tokens of the item's span
    t_hi: int
    whole: bool


def pieces(new, kv, group, lists, rows, item_tokens, unit, workgroups, window=None, sinks=0, ids=None):
    items = []  # (request, list, block, weight, rows, tokens)
    for r, (m, n) in enumerate(zip(new, kv)):
        m = 1 if ids is not None else m
        for l in range(lists):
            for b in range(-(-m * group // rows)):
                row0, row1 = b * rows, min((b + 1) * rows, m * group) - 1
                t0, t1 = row0 // group, row1 // group
                end = max(0, min(n - m + t1 + 1, n))
                total, weight = end, (item_tokens + max(n - m, 0)) * group + (b + 1) * rows
                if window is not None:
                    first = min(sinks, end)
                    total = first + max(0, end - max(first, n - m + t0 + 1 - window)) + (ids or 0)
                    weight = (item_tokens + min(n, sinks + window + rows // group) + (ids or 0)) * group
                items.append((r, l, b, weight, row1 - row0 + 1, total))
    share = max(-(-sum(i[3] for i in items) // workgroups), item_tokens * group)
    out, begin = [], 0
    for r, l, b, weight, n, total in items:
        units, x = max(-(-total // unit), 1), begin
        cuts = [0]
        while x < begin + weight:
            x = min((x // share + 1) * share, begin + weight)
            cuts.append(units if x == begin + weight else min((x - begin) * units // weight, units - 1))
        out += [Piece(r, l, b, n, u * unit, min(v * unit, total), (u, v) == (0, units)) for u, v in zip(cuts, cuts[1:]) if v > u]
        begin += weight
    return out


def joined_rows(ps):
    return sum(p.rows for p in ps if not p.whole and p.t_lo == 0)
