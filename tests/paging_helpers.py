"""Plain forms of the page tables' operations, one number after the other, for the tests."""
from __future__ import annotations


def up(n, page):
    return -(-n // page)


def plan(lens, new, tables, free, counts, page, rows):
    """-> slots, positions, starts, lens, counts, tables (lists), and whether something was out of order."""
    tables = [list(t) for t in tables]
    width, odd = len(tables[0]), False
    n_free = min(max(counts[0], 0), len(free))
    odd |= n_free != counts[0]
    stack, missing = list(free[:n_free]), 0
    slots, positions, starts, out = [], [], [], []
    for b, (held, add) in enumerate(zip(lens, new)):
        h = min(max(held, 0), width * page)
        a = min(max(add, 0), width * page - h)
        odd |= h != held or a != add
        starts.append(len(slots))
        for i in range(up(h, page), up(h + a, page)):
            got = stack.pop() if stack else None
            if got is None:
                missing += 1
            ok = got is not None and 0 <= got < len(free)
            odd |= not ok
            tables[b][i] = got if ok else -1
        for p in range(h, h + a):
            e = tables[b][p // page]
            ok = 0 <= e < len(free)
            odd |= not ok
            slots.append(e * page + p % page if ok else -1)
            positions.append(p)
        out.append(h + a)
    odd |= len(slots) > rows
    starts = [min(s, rows) for s in starts + [len(slots)]]
    slots, positions = slots[:rows], positions[:rows]
    pad = rows - len(slots)
    return slots + [-1] * pad, positions + [0] * pad, starts, out, [len(stack), counts[1] + missing], tables, odd


def release(done, lens, tables, free, counts, page):
    """-> lens, counts, free"""
    width, free = len(tables[0]), list(free)
    n = min(max(counts[0], 0), len(free))
    out = []
    for b, held in enumerate(lens):
        h = min(max(held, 0), width * page)
        if done[b]:
            for i in range(up(h, page)):
                if counts[1] and not 0 <= tables[b][i] < len(free):
                    continue
                if n < len(free):
                    free[n] = tables[b][i]
                    n += 1
        out.append(0 if done[b] else h)
    return out, [n, counts[1]], free


def reorder(parents, lens, tables, free, counts, page, own=None):
    """parents (requests, beams) -> tables, lens, counts, src, dst, used, free"""
    beams, width, free = len(parents[0]), len(tables[0]), list(free)
    n = min(max(counts[0], 0), len(free))
    jobs = []
    for r, ps in enumerate(parents):
        old = [tables[r * beams + k] for k in range(beams)]
        held = [min(max(lens[r * beams + k], 0), width * page) for k in range(beams)]
        first = own[r] if own else 0
        live = sorted({p for p in ps if 0 <= p < beams})
        gone = []
        for i in range(max(first, 0), width):
            kept = {old[k][i] for k in live if i < up(held[k], page)}
            for k in range(beams):
                if i < up(held[k], page) and k not in live and old[k][i] not in kept and 0 <= old[k][i] < len(free):
                    gone.append(old[k][i])
                    kept.add(old[k][i])
        ends, copies = {}, []
        for j, p in enumerate(ps):
            if not 0 <= p < beams or held[p] % page == 0:
                continue
            e = old[p][held[p] // page]
            if e < 0:
                continue
            if held[p] // page < first or e in ends:
                copies.append(j)
            ends[e] = j
        jobs.append((r, ps, old, held, gone, copies))
    targets = {}
    for r, ps, old, held, gone, copies in jobs:                  # a request's own freed pages first
        for j, page_no in zip(copies, gone):
            targets[r, j] = page_no
        for page_no in gone[len(copies):]:
            free[n] = page_no
            n += 1
    missing = 0
    for r, ps, old, held, gone, copies in jobs:
        for j in copies[len(gone):]:
            if n > 0:
                n -= 1
                targets[r, j] = free[n]
            else:
                targets[r, j] = -1
                missing += 1
    t_out, l_out, src, dst, used = [], [], [], [], []
    for r, ps, old, held, gone, copies in jobs:
        for j, p in enumerate(ps):
            h = held[p] if 0 <= p < beams else 0
            row = [old[p][i] if i < up(h, page) else -1 for i in range(width)]
            s, d, u = -1, -1, 0
            if j in copies:
                s, d, u = row[h // page], targets[r, j], h % page
                row[h // page] = d
            t_out.append(row), l_out.append(h), src.append(s), dst.append(d), used.append(u)
    return t_out, l_out, [n, counts[1] + missing], src, dst, used, free
