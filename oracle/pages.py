"""The plans of forks and compactions of paged rows in plain Python — TEST INFRASTRUCTURE ONLY (see the
package docstring).

Not in the reference; these restate the definitions of the calls on a cache's pages.  Pinned by the
invariants that define them (every row reads its tokens, pages to be written belong to one row, the lowest
free pages go first).

* ``fork``    -> (table, lens, free, copies) of rows that go on from ``parents``;
* ``compact`` -> (table, used, moves).
"""


def _pages(n, size):
    return -(-n // size)


def fork(table, lens, parents, num_pages, page, room=0, keep=()):
    """``table``: lists of page ids, ``lens``: tokens, ``parents``: rows to go on from, ``room``: a number or one per
    row, ``keep``: pages that others hold.  copies: (from, to) pairs."""
    width = len(table[0])
    parents = list(range(len(table))) if parents is None else parents
    rooms = [room] * len(parents) if isinstance(room, int) else list(room)
    valid = range(num_pages)
    rows = []
    for p in parents:
        n = min(max(lens[p], 0), width * page) if 0 <= p < len(table) else 0
        rows.append((n, list(table[p][:n // page]) if n else [], table[p][n // page] if n % page else None))
    taken = set(keep) | {x for _, whole, _ in rows for x in whole if x in valid}
    stays = []
    for _, _, last in rows:
        stays.append(last is None or last not in valid or last not in taken)
        if last is not None and last in valid:
            taken.add(last)
    free = [x for x in valid if x not in taken]
    left, out, copies = len(free), [], []

    def take():
        nonlocal left
        left -= 1
        return free.pop(0) if free else -1

    for (n, whole, last), mine, more in zip(rows, stays, rooms):
        row = list(whole)
        if last is not None:
            row.append(last if mine else take())
            if not mine and row[-1] >= 0:
                copies.append((last, row[-1]))
        while len(row) < _pages(min(n + max(more, 0), width * page), page):
            row.append(take())
        out.append(row + [-1] * (width - len(row)))
    return out, [n for n, _, _ in rows], left, copies


def compact(table, lens, num_pages, page, room=0, keep=()):
    """moves: (from, to) pairs."""
    width = len(table[0])
    wants = [_pages(min(min(max(n, 0), width * page) + room, width * page), page) for n in lens]
    rows = {x for row, w in zip(table, wants) for x in row[:w] if 0 <= x < num_pages}
    held = rows | set(keep)
    used = len(held)
    slots = [x for x in range(used) if x not in held]
    to = dict(zip(sorted(x for x in rows - set(keep) if x >= used), slots))
    out = [[to.get(x, x) if i < w else -1 for i, x in enumerate(row)] for row, w in zip(table, wants)]
    return out, used, sorted(to.items())
