"""The plans of forks and compactions (oracle/pages.py) by the invariants that define them (CPU)."""
import random

import pytest

from oracle import pages


def _rows(r, B, width, page, P):
    """Rows that share beginnings, on random pages."""
    ids = list(range(P))
    r.shuffle(ids)
    table, lens = [], []
    for b in range(B):
        n = r.randint(0, width * page)
        shared = r.randint(0, min(n // page, lens[-1] // page)) if table and r.random() < 0.5 else 0
        mine = -(-n // page) - shared
        if mine > len(ids):
            n, mine = shared * page, 0
        row = (table[-1][:shared] if shared else []) + [ids.pop() for _ in range(mine)]
        table.append(row + [-1] * (width - len(row)))
        lens.append(n)
    return table, lens


@pytest.mark.parametrize("seed", range(20))
def test_fork(seed):
    r = random.Random(seed)
    page, width, P, B, N = r.choice([32, 96]), r.randint(1, 9), r.randint(10, 80), r.randint(1, 9), r.randint(1, 12)
    table, lens = _rows(r, B, width, page, P)
    parents = [r.randint(-1, B) for _ in range(N)]
    keep = r.sample(range(P), P // 8)
    room = [r.randint(0, 2 * page) for _ in range(N)]
    out, n, free, copies = pages.fork(table, lens, parents, P, page, room, keep)
    content = dict(copies and [(d, s) for s, d in copies])  # what a fresh page holds
    written = []  # pages that a row goes on to write
    for b, p in enumerate(parents):
        want = lens[p] if 0 <= p < B else 0
        assert n[b] == want
        for i in range(-(-want // page)):
            if out[b][i] >= 0:
                assert content.get(out[b][i], out[b][i]) == table[p][i]  # the row reads its tokens
        written += [x for x in out[b][want // page:] if x >= 0]
    assert len(set(written)) == len(written)
    whole = {x for b, row in enumerate(out) for x in row[:n[b] // page]}
    assert not whole & set(written) and not set(keep) & set(written)
    if free >= 0:
        assert free == P - len(whole | set(written) | set(keep))
        assert all(-1 not in row[:-(-min(n[b] + room[b], width * page) // page)] for b, row in enumerate(out))
    assert not {d for _, d in copies} & ({s for s, _ in copies} | set(keep))


@pytest.mark.parametrize("seed", range(20))
def test_compact(seed):
    r = random.Random(seed)
    page, width, P, B = 32, r.randint(1, 9), r.randint(10, 80), r.randint(1, 9)
    table, lens = _rows(r, B, width, page, P)
    keep = r.sample(range(P), P // 8)
    out, used, moves = pages.compact(table, lens, P, page, 0, keep)
    held = {x for row, n in zip(table, lens) for x in row[:-(-n // page)]} | set(keep)
    assert used == len(held)
    to = dict(moves)
    assert not set(to.values()) & held and not set(to) & set(keep)
    for row, new, n in zip(table, out, lens):
        m = -(-n // page)
        assert new == [to.get(x, x) for x in row[:m]] + [-1] * (width - m)
        assert all(x < used or x in keep for x in new[:m])


def test_a_fork_by_hand():
    """Two beams of one row and one of another: the first keeps the last page, the second gets the lowest free one."""
    table, lens = [[7, 3, -1], [5, -1, -1]], [40, 32]
    assert pages.fork(table, lens, [0, 0, 1, -1], 8, 32, [1, 0, 1, 1], [0]) == (
        [[7, 3, -1], [7, 1, -1], [5, 2, -1], [4, -1, -1]], [40, 40, 32, 0], 1, [(3, 1)])
    assert pages.compact([[7, 0]], [64], 8, 32) == ([[1, 0]], 2, [(7, 1)])
    assert pages.compact(table, lens, 8, 32, 0, [0]) == ([[2, 3, -1], [1, -1, -1]], 4, [(5, 1), (7, 2)])
