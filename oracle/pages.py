"""Pages that change hands, one sequence and one page at a time (kv_page_fork, kv_page_release, kv_page_compact of include/fp8_block.h)."""
import numpy as np


def _up(n, page):
    return -(-n // page)


def _ring(ring, head, count):
    n = len(ring)
    head, count = max(head, 0) % n, min(max(count, 0), n)
    return head, count, [int(ring[(head + i) % n]) for i in range(count)]


def _lengths(lens, table, page):
    return [min(max(int(n), 0), table.shape[1] * page) for n in lens]


def _has(j, n, gone, sinks, page):
    return j < _up(n, page) and (j < _up(sinks, page) or j >= gone)


def fork(lens, parent, keep, table, ring, head, count, shares, gone, page, sinks=0, window=0):
    table, shares, pages = table.copy(), shares.copy(), len(ring)
    head, count, free = _ring(ring, head, count)
    before, batch = _lengths(lens, table, page), len(lens)
    gone = [0] * batch if gone is None else [max(int(g), 0) for g in gone]
    lens_out, gone_out, taken, moves, asked = [int(n) for n in lens], list(gone), [0] * batch, [], 0
    for b, p in enumerate(parent):
        p = int(p)
        if not 0 <= p < batch or p == b or before[b]:
            continue
        n = before[p] if keep is None else min(before[p], max(int(keep[b]), 0))
        full, rest = divmod(n, page)
        # pages that hold a key which the next token, at place n, sees; without a window the one that is to be copied
        needs = [j for j in range(_up(n, page)) if (j + 1) * page > n + 1 - window] if window else [full] * (rest > 0)
        if not all(_has(j, n, gone[p], sinks, page) for j in needs):
            continue
        if rest:
            asked += 1
            if asked > count:
                continue
            moves.append((int(table[p, full]), free[asked - 1]))
            table[b, full] = free[asked - 1]
        for j in range(full):
            if _has(j, n, gone[p], sinks, page):
                table[b, j] = table[p, j]
                if 0 <= table[p, j] < pages:
                    shares[table[p, j]] += 1
        lens_out[b], taken[b], gone_out[b] = n, n, min(gone[p], full)
    used = len(moves)
    return dict(lens=lens_out, taken=taken, table=table, shares=shares, gone=gone_out, moves=moves, state=((head + used) % pages, count - used))


def release(lens, keep, table, ring, head, count, shares, gone, page, window=0, sinks=0):
    ring, shares, pages = ring.copy(), shares.copy(), len(ring)
    head, count, _ = _ring(ring, head, count)
    lens_out, gone_out = [], []
    for b, n in enumerate(_lengths(lens, table, page)):
        m = n if keep is None else min(n, max(int(keep[b]), 0))
        g = 0 if gone is None else max(int(gone[b]), 0)
        # pages that hold nothing from key m + 1 - window on
        passed = max(0, (m + 1 - window) // page) if window else 0
        left = min(max(g, passed), _up(m, page))
        for j in range(table.shape[1]):
            if _has(j, n, g, sinks, page) and not _has(j, m, left, sinks, page) and 0 <= table[b, j] < pages:
                shares[table[b, j]] -= 1
        lens_out.append(m)
        gone_out.append(left)
    for p in range(pages):
        if shares[p] < 0:
            shares[p] = 0
            if count < pages:
                ring[(head + count) % pages] = p
                count += 1
    return dict(lens=lens_out, gone=gone_out, shares=shares, ring=ring, state=(head, count))


def compact(lens, table, ring, head, count, shares, page):
    pages = len(ring)
    _, _, entries = _ring(ring, head, count)
    free = set(e for e in entries if 0 <= e < pages)
    used = pages - len(free)
    movers, holes = [p for p in range(used, pages) if p not in free], [p for p in range(used) if p in free]
    moved_to = [-1 if p in free else p for p in range(pages)]
    for a, b in zip(movers, holes):
        moved_to[a] = b
    out, shares_out = table.copy(), np.zeros_like(shares)
    for p in range(pages):
        if p not in free:
            shares_out[moved_to[p]] = shares[p]
    for b, n in enumerate(_lengths(lens, table, page)):
        for j in range(_up(n, page)):
            out[b, j] = moved_to[table[b, j]] if 0 <= table[b, j] < pages else -1
    return dict(table=out, ring=[used + i if used + i < pages else -1 for i in range(pages)], state=(0, pages - used), shares=shares_out, moved_to=moved_to,
                moves=list(zip(movers, holes)))
