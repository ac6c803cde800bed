"""copy_kv_pages, fork_kv_rows and compact_kv_pages on the GPU: tables, lengths and counts are whole numbers and equal
those of the plain restatement (oracle/pages.py); pages are equal byte for byte, and no other page changes."""
import random

import numpy as np
import pytest

pytestmark = pytest.mark.gpu

from oracle import pages  # noqa: E402
from tests.test_pages_oracle import _rows  # noqa: E402


def _caches(kind, P, page, layers=1, H=2, D=64, seed=0):
    import torch
    import pallas_flexattn as pf
    g = torch.Generator(device="cuda").manual_seed(seed)
    out = []
    for _ in range(layers):
        if kind == "latent":
            out.append(pf.LatentKVCache(torch.randn(P, page, 160, device="cuda", generator=g).bfloat16(), 128))
        elif kind == "fp8":
            c = [torch.randint(0, 256, (P, H, page, D), device="cuda", generator=g, dtype=torch.uint8).view(torch.float8_e4m3fn)
                 for _ in range(2)]
            out.append(pf.Fp8KVCache(*c, *[torch.randn(P, H, page // 32, device="cuda", generator=g) for _ in range(2)]))
        else:
            out.append(tuple(torch.randn(P, H, page, D, device="cuda", generator=g).bfloat16() for _ in range(2)))
    return out


def _host(caches):
    import torch
    return [x.reshape(x.shape[0], -1).view(torch.uint8).cpu().numpy() for c in caches for x in c if hasattr(x, "data_ptr")]


def _check_pages(before, caches, pairs):
    for x, y in zip(before, _host(caches)):
        want = x.copy()
        for s, d in pairs:
            want[d] = x[s]
        assert np.array_equal(want, y)


def _t(x, dtype=None):
    import torch
    return torch.tensor(x, device="cuda", dtype=dtype or torch.int32)


@pytest.mark.parametrize("kind,layers,H,page", [("bf16", 1, 2, 64), ("fp8", 3, 1, 32), ("latent", 2, 0, 96), ("fp8", 40, 2, 32),
                                                ("bf16", 1, 9, 256)])
def test_copy(kind, layers, H, page):
    import torch
    import pallas_flexattn as pf
    c = _caches(kind, 12, page, layers, H)
    before = _host(c)
    src, dst = [3, 3, -1, 5, 0, 12, 7], [1, 9, 2, -5, 0, 4, 2 ** 31 - 1]  # (twice from one page; the others are left out)
    versions = [x._version for k in c for x in k if hasattr(x, "data_ptr")]
    assert pf.copy_kv_pages(c, _t(src), _t(dst)) is None
    _check_pages(before, c, [(3, 1), (3, 9)])
    assert all(x._version > v for x, v in zip((x for k in c for x in k if hasattr(x, "data_ptr")), versions))
    pf.copy_kv_pages(c[0], _t([4, 2 ** 40], torch.int64), _t([6, 1], torch.int64))  # one cache, 64-bit ids
    _check_pages(before[:len(before) // layers], c[:1], [(3, 1), (3, 9), (4, 6)])
    pf.copy_kv_pages(c, _t([]), _t([]))
    pf.copy_kv_pages(c[0], [8], [11])
    _check_pages(before[:len(before) // layers], c[:1], [(3, 1), (3, 9), (4, 6), (8, 11)])


# rows, result rows, table width, page, pages; the plan of one workgroup and of several launches
FORKS = [(1, 8, 5, 32, 64), (9, 12, 7, 96, 200), (40, 33, 20, 32, 700), (3, 1, 1, 64, 5), (1, 1, 4, 32, 4),
         (5, 1100, 3, 32, 4000), (64, 64, 520, 32, 40000), (7, 9, 6, 32, 30000), (2, 3, 4, 64, 6)]


@pytest.mark.parametrize("case", FORKS, ids=[str(i) for i in range(len(FORKS))])
@pytest.mark.parametrize("kind", ["bf16", "fp8", "latent"])
def test_fork(case, kind):
    import pallas_flexattn as pf
    B, N, width, page, P = case
    r = random.Random(f"{case}{kind}")
    table, lens = _rows(r, B, width, page, P)
    if B > 1:
        table[0][0] = P + 7  # an id outside the cache stays
    lens[-1] = max(lens[-1], 0) if B > 2 else lens[-1]
    parents = [r.randint(-1, B) for _ in range(N)]
    keep = r.sample(range(P), P // 9)
    room = [r.choice([0, 1, page, 3 * page + 5]) for _ in range(N)]
    c = _caches(kind, P, page, 1, 1, 32)
    before = _host(c)
    import torch
    mask = torch.zeros(P, device="cuda", dtype=torch.bool)
    mask[keep] = True
    t, n, free = pf.fork_kv_rows(c, _t(table), _t(lens), _t(parents), room=_t(room), keep=mask)
    wt, wn, wf, copies = pages.fork(table, lens, parents, P, page, room, keep)
    assert t.tolist() == wt and n.tolist() == wn and int(free) == wf
    assert t.dtype == n.dtype == free.dtype == torch.int32 and free.shape == ()
    _check_pages(before, c, copies)
    # each row from itself, one room for all
    t2, n2, free2 = pf.fork_kv_rows(c, _t(table, torch.int64), _t(lens, torch.int64), room=1)
    wt, wn, wf, _ = pages.fork(table, lens, None, P, page, 1)
    assert t2.tolist() == wt and n2.tolist() == wn and int(free2) == wf


def test_too_few_pages():
    import pallas_flexattn as pf
    c = _caches("bf16", 3, 32)
    before = _host(c)
    table, lens = [[0, 2, -1]], [40]
    t, n, free = pf.fork_kv_rows(c, _t(table), _t(lens), _t([0, 0, 0]), room=0)
    assert t.tolist() == [[0, 2, -1], [0, 1, -1], [0, -1, -1]] and n.tolist() == [40] * 3 and int(free) == -1
    _check_pages(before, c, [(2, 1)])


def test_lengths_at_the_ends():
    """Lengths and rooms past the table, negative, and sums past 32 bits."""
    import pallas_flexattn as pf
    c = _caches("latent", 9, 32)
    table, lens, room = [[0, 1, 2]] * 4, [96, 2 ** 31 - 1, -5, 33], [2 ** 31 - 1, 2 ** 31 - 1, 2 ** 31 - 1, -7]
    t, n, free = pf.fork_kv_rows(c, _t(table), _t(lens), room=_t(room))
    wt, wn, wf, _ = pages.fork(table, lens, None, 9, 32, room)
    assert t.tolist() == wt and n.tolist() == wn and int(free) == wf
    t, used = pf.compact_kv_pages(c, _t(table), _t(lens), room=2 ** 31 - 1)
    assert t.tolist() == [[0, 1, 2]] * 4 and int(used) == 3


COMPACTS = [(1, 5, 32, 64), (9, 7, 96, 100), (40, 20, 32, 700), (64, 520, 32, 40000), (3, 4, 32, 30000), (1100, 3, 32, 4000), (2, 3, 64, 6)]


@pytest.mark.parametrize("case", COMPACTS, ids=[str(i) for i in range(len(COMPACTS))])
@pytest.mark.parametrize("kind", ["bf16", "fp8", "latent"])
def test_compact(case, kind):
    import torch
    import pallas_flexattn as pf
    B, width, page, P = case
    r = random.Random(f"{case}{kind}")
    table, lens = _rows(r, B, width, page, P)
    table[0][-1] = -9 if lens[0] > (width - 1) * page else table[0][-1]
    keep = r.sample(range(P), P // 9)
    c = _caches(kind, P, page, 1, 1, 32)
    before = _host(c)
    mask = torch.zeros(P, device="cuda", dtype=torch.bool)
    mask[keep] = True
    t, used = pf.compact_kv_pages(c, _t(table), _t(lens), keep=mask)
    wt, wu, moves = pages.compact(table, lens, P, page, 0, keep)
    assert t.tolist() == wt and int(used) == wu
    _check_pages(before, c, moves)
    t2, used2 = pf.compact_kv_pages(c, t, _t(lens), room=page)
    wt2, wu2, moves2 = pages.compact(wt, lens, P, page, page)
    assert t2.tolist() == wt2 and int(used2) == wu2


def test_replays_of_a_graph():
    """A captured fork and compaction take what their inputs hold at each replay."""
    import torch
    import pallas_flexattn as pf
    c = _caches("fp8", 300, 32, 2)
    table, lens, parents = _t([[-1] * 9] * 12), _t([0] * 12), _t([0] * 12)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        pf.fork_kv_rows(c, table, lens, parents, room=1)
        pf.compact_kv_pages(c, table, lens)
    torch.cuda.current_stream().wait_stream(s)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        t, n, free = pf.fork_kv_rows(c, table, lens, parents, room=1)
        t2, used = pf.compact_kv_pages(c, t, n, room=1)
    for seed in range(4):
        r = random.Random(seed)
        tab, ln = _rows(r, 12, 9, 32, 300)
        pa = [r.randint(-1, 12) for _ in range(12)]
        table.copy_(_t(tab)), lens.copy_(_t(ln)), parents.copy_(_t(pa))
        before = _host(c)
        g.replay()
        wt, wn, wf, copies = pages.fork(tab, ln, pa, 300, 32, 1)
        wt2, wu, moves = pages.compact(wt, wn, 300, 32, 1)
        assert t.tolist() == wt and n.tolist() == wn and int(free) == wf and t2.tolist() == wt2 and int(used) == wu
        now = _host(c)
        for x, y in zip(before, now):
            want = x.copy()
            for s_, d in copies:
                want[d] = x[s_]
            mid = want.copy()
            for s_, d in moves:
                want[d] = mid[s_]
            assert np.array_equal(want, y)


def test_another_stream_and_unaligned_scales():
    """On a stream of its own; scales that start 4 bytes off a 16-byte line are copied by words."""
    import torch
    import pallas_flexattn as pf
    c = _caches("fp8", 8, 96, 1, 1, 32)[0]
    raw = torch.randn(1 + c.key_scale.numel(), device="cuda")
    c = c._replace(key_scale=raw[1:].reshape(c.key_scale.shape))
    s = torch.cuda.Stream()
    with torch.cuda.stream(s):
        torch.cuda._sleep(1000)
        before = _host([c])
        pf.copy_kv_pages(c, _t([2, 5]), _t([3, 0]))
        _check_pages(before, [c], [(2, 3), (5, 0)])
