"""The pages of a cache, one entry after the other: a table of page numbers (lists of lists), lens and refs, changed in place."""


def free(table, lens, refs, rows):
    P = len(refs)
    for r in rows:
        if not 0 <= r < len(table):
            continue
        for j, x in enumerate(table[r]):
            if 0 <= x < P:
                refs[x] -= 1
                table[r][j] = -1
        lens[r] = 0


def fork(table, lens, refs, src, dst):
    P, N = len(refs), len(table)
    before, lens0 = [list(r) for r in table], list(lens)
    last = {d: s for s, d in zip(src, dst) if 0 <= s < N and 0 <= d < N}
    for d, s in last.items():
        for x in table[d]:
            if 0 <= x < P:
                refs[x] -= 1
        for x in before[s]:
            if 0 <= x < P:
                refs[x] += 1
        table[d], lens[d] = list(before[s]), lens0[s]


def reserve(table, lens, refs, tokens, S):
    """(fits, copies as (from, to))."""
    P = len(refs)
    spare = [p for p in range(P) if refs[p] <= 0]
    fits, copies, over = [], [], False
    for row, n, t in zip(table, lens, tokens):
        n = max(n, 0)
        if t <= 0:
            fits.append(True)
            continue
        if (n + t - 1) // S >= len(row):
            fits.append(False)
            continue
        # as if one column after the other: an entry of the row that shares a page with another of it
        mine, want = {}, []
        for j in range(n // S, (n + t - 1) // S + 1):
            x = row[j]
            if not 0 <= x < P:
                want.append(j)
            elif refs[x] - mine.get(x, 0) > 1:
                want.append(j)
                mine[x] = mine.get(x, 0) + 1
        ok = not want or (not over and len(want) <= len(spare))
        over = over or not ok
        fits.append(ok)
        for j in want if ok else ():
            p = spare.pop(0)
            if 0 <= row[j] < P:
                copies.append((row[j], p))
                refs[row[j]] -= 1
            refs[p], row[j] = 1, p
    return fits, copies


def compact(table, refs):
    """(live, moved, copies)."""
    P = len(refs)
    live = sum(x > 0 for x in refs)
    holes = [p for p in range(live) if refs[p] <= 0]
    moved, copies = list(range(P)), []
    for p in range(live, P):
        if refs[p] > 0:
            h = holes.pop(0)
            moved[p] = h
            copies.append((p, h))
            refs[h], refs[p] = refs[p], 0
    for row in table:
        row[:] = [moved[x] if 0 <= x < P else x for x in row]
    return live, moved, copies
