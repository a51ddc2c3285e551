"""The pools' operators one entry after the other, on lists: what each does to
(table, lengths, counts), and None where it cannot be done."""
from __future__ import annotations


def counts(table, P, pinned=()):
    refs = [0] * P
    for row in table:
        for e in row:
            if 0 <= e < P:
                refs[e] += 1
    for p in pinned:
        refs[p] += 1
    return refs


def fork(table, lens, refs, parents, R, H, M):
    P = len(refs)
    B = len(table) // H
    if any(not -1 <= a < B for a in parents) or any(not 0 <= n <= M * R for n in lens):
        return None
    free = [p for p in range(P) if refs[p] == 0]
    new, new_len, copies, refs = [], [], [], list(refs)
    seen = set()
    for a in parents:
        for h in range(H):
            if a < 0:
                new.append([-1] * M)
                new_len.append(0)
                copies.append([-1, -1, 0])
                continue
            row, n = [e if 0 <= e < P else -1 for e in table[a * H + h]], lens[a * H + h]
            copy = [-1, -1, 0]
            if a in seen:
                full, part = divmod(n, R)
                kept = row[:full] + [-1] * (M - full)
                if part and row[full] >= 0:
                    if not free:
                        return None
                    copy = [row[full], free.pop(0), part]
                    kept[full] = copy[1]
                row = kept
            for e in row:
                if e >= 0:
                    refs[e] += 1
            new.append(row)
            new_len.append(n)
            copies.append(copy)
        seen.add(a)
    for row in table:
        for e in row:
            if 0 <= e < P:
                refs[e] -= 1
    return new, new_len, refs, copies


def reserve(table, lens, refs, R, tokens, view=None):
    """tokens: of each segment; view: (window, sinks) of each, or None."""
    P, M = len(refs), len(table[0]) if table else 0
    if any(not 0 <= n <= M * R for n in lens) or any(t < 0 for t in tokens) or (view and any(w < 0 or z < 0 for w, z in view)):
        return None
    if any(n + t > M * R for n, t in zip(lens, tokens)):
        return None
    free = [p for p in range(P) if refs[p] == 0]
    new, after = [], list(refs)
    for s, (row, n) in enumerate(zip(table, lens)):
        row = [e if 0 <= e < P else -1 for e in row]
        kept = list(row)
        for j, e in enumerate(row):
            if e < 0 and n // R <= j and j * R < n + tokens[s]:
                if not free:
                    return None
                kept[j] = free.pop(0)
                after[kept[j]] += 1
            elif e >= 0 and view:
                w, z = view[s]
                if j * R >= z and (j + 1) * R <= n + 1 - max(w, 1):
                    kept[j] = -1
                    after[e] -= 1
        new.append(kept)
    return new, after


def compact(table, refs, R):
    P = len(refs)
    used = [p for p in range(P) if refs[p] > 0]
    U = len(used)
    movers = [p for p in used if p >= U]
    holes = [p for p in range(U) if refs[p] == 0]
    place = dict(zip(movers, holes))
    new = [[-1 if not 0 <= e < P or (e >= U and e not in place) else place.get(e, e) for e in row] for row in table]
    after = list(refs)
    for a, b in place.items():
        after[b], after[a] = refs[a], 0
    moves = [[a, b, R] for a, b in place.items()] + [[-1, -1, 0]] * (P // 2 - len(place))
    return new, after, moves, U
