"""Plain CPU implementation, entry by entry with lists, of the life of cache pages: tables, counts of names, forks, compacted sequences."""
from __future__ import annotations

import collections

import torch


def free(refs, table, keep=None):
    """(refs, table) afterwards, lists."""
    refs, table = list(refs), [list(r) for r in table]
    for b, row in enumerate(table):
        for e in range(0 if keep is None else max(0, keep[b]), len(row)):
            if 0 <= row[e] < len(refs):
                refs[row[e]] -= 1
            row[e] = -1
    return refs, table


def alloc(refs, table, first, last):
    refs, table = list(refs), [list(r) for r in table]
    pages = [p for p, r in enumerate(refs) if r <= 0]
    for b, row in enumerate(table):
        for e in range(max(0, first[b]), min(last[b], len(row))):
            row[e] = pages.pop(0) if pages else -1
            if row[e] >= 0:
                refs[row[e]] = 1
    return refs, table


def fork(refs, table, source, target, lengths, page: int):
    """(refs, table, copies (from, to, tokens))"""
    refs, out = list(refs), [list(r) for r in table]
    pages, copies = [p for p, r in enumerate(refs) if r <= 0], []
    pairs = [(s, t) for s, t in zip(source, target) if 0 <= s < len(table) and 0 <= t < len(table) and s != t]
    sources, targets = {s for s, _ in pairs}, [t for _, t in pairs]
    twice = {t for t, n in collections.Counter(targets).items() if n > 1}
    for s, t in pairs:
        if t in sources or t in twice:
            continue
        n = max(0, lengths[s])
        whole, rest = n // page, n % page
        for e in range(len(out[t])):
            out[t][e] = table[s][e] if e < whole else -1
            if e < whole and 0 <= table[s][e] < len(refs):
                refs[table[s][e]] += 1
        if rest and whole < len(out[t]) and 0 <= table[s][whole] < len(refs) and pages:
            out[t][whole] = pages.pop(0)
            refs[out[t][whole]] = 1
            copies.append((table[s][whole], out[t][whole], rest))
    return refs, out, copies


def compact(pool, table, keep, out_table, counts=None, nothing=0):
    """A clone of pool [pages,heads,page,...] with the kept tokens in the pages of out_table."""
    out, (P, H, page) = pool.clone(), pool.shape[:3]

    def place(row, pos):
        return row[pos // page] if 0 <= pos < len(row) * page and 0 <= row[pos // page] < P else None

    for b in range(len(table)):
        for h in range(H):
            for i in range(keep.shape[2] if counts is None else max(0, min(keep.shape[2], counts[b]))):
                to, at = place(out_table[b], i), place(table[b], int(keep[b, h, i]))
                if to is not None:
                    out[to, h, i % page] = torch.full_like(pool[0, h, 0], nothing) if at is None else pool[at, h, int(keep[b, h, i]) % page]
    return out
