"""flex_prefill on the GPU against float64 attention over the cache's values (oracle/kv_cache.py).

Tolerance. Scores as in tests/test_gpu_decode_fp8.py: ds = (D + 2) 2^-24 sum |q||k| scale + 4 2^-24 |s| + cap 2^-20.
A weight is off by ds relative plus 2^-21 (exp2), its rounding to bf16 by half a step, 2^-8, and the sums of n weights
by n 2^-24: O is within half a step of its own (2^-8 |o|) plus c sum p |v|, c = 2 ds + 2^-8 + 2^-20 + 2 n 2^-24, and that
rounded once more (a factor 1 + 2^-8). LSE, from unrounded weights, is within ds + 2^-20 + n 2^-24 + 2^-22 |lse|."""
import numpy as np
import pytest

pytestmark = pytest.mark.gpu

from oracle import kv_cache  # noqa: E402
from tests.test_gpu_decode_fp8 import Cache as Fp8Cache  # noqa: E402
from tests.test_gpu_rotary import _np  # noqa: E402


class Bf16Cache:
    """Random rows of the given lengths in pages of random order; all that no row uses is NaN."""

    def __init__(self, lens, H, page, D, seed, per_row=None, spread=1.0):
        import torch
        B = len(lens)
        per_row = per_row or max(1, -(-max(lens) // page))
        g = torch.Generator(device="cuda").manual_seed(seed)
        n = B * per_row + 2
        self.table = torch.randperm(n, generator=g, device="cuda")[:B * per_row].reshape(B, per_row).to(torch.int32)
        self.lens = torch.tensor(lens, device="cuda", dtype=torch.int32)
        S = per_row * page
        used = (torch.arange(S, device="cuda") < self.lens[:, None])[:, None, :, None]
        self.rows, self.cache = [], []
        for _ in range(2):
            x = (torch.randn(B, H, S, D, device="cuda", generator=g) * spread).bfloat16()
            self.rows.append(torch.where(used, x.float(), 0.0))
            c = torch.full((n, H, page, D), float("nan"), device="cuda", dtype=torch.bfloat16)
            c[self.table.long().reshape(-1)] = torch.where(used, x, float("nan")).reshape(B, H, per_row, page, D).transpose(
                1, 2).reshape(-1, H, page, D)
            self.cache.append(c)
        self.cache = tuple(self.cache)


def _cache(kind, *a, **kw):
    return (Fp8Cache if kind == "fp8" else Bf16Cache)(*a, **kw)


def _check(o, lse, q, c, lens, ql=None, left=-1, right=-1, scale=None, slopes=None, cap=0.0):
    D = q.shape[3]
    qn, k, v = _np(q), _np(c.rows[0]), _np(c.rows[1])
    wo, wl, w = kv_cache.decode(qn, k, v, lens, ql, left, right, scale, slopes, cap)
    sc = D ** -0.5 if scale is None else scale
    qmax = np.abs(qn).sum(-1).max() * np.abs(k[np.isfinite(k)]).max() * sc  # an upper bound of sum |q||k| scale
    smax = qmax + (0 if slopes is None else float(np.max(np.abs(slopes))) * k.shape[2])
    ds = (D + 2) * 2.0 ** -24 * qmax + 4 * 2.0 ** -24 * smax + cap * 2.0 ** -20
    n = k.shape[2]
    c1 = (2 * ds + 2.0 ** -8 + 2.0 ** -20 + 2 * n * 2.0 ** -24) * (1 + 2.0 ** -8)
    go, gl = _np(o), _np(lse)
    for g, want in ((go, wo), (gl, wl)):
        assert np.array_equal(np.isnan(g), np.isnan(want))
        inf = np.isinf(want)
        assert np.array_equal(np.isinf(g), inf) and np.array_equal(g[inf], want[inf])
    dead = np.isneginf(wl)
    assert np.all(go[dead] == 0)
    fin = np.isfinite(wo)
    err, tol = np.abs(go - wo)[fin], (np.abs(wo) * 2.0 ** -8 + c1 * w + 1e-30)[fin]
    assert np.all(err <= tol), f"O off by {np.max(err / tol):.3g} times the tolerance"
    fin = np.isfinite(wl)
    el = np.abs(gl - wl)[fin]
    assert np.all(el <= ds + 2.0 ** -20 + n * 2.0 ** -24 + 2.0 ** -22 * np.abs(wl[fin])), f"LSE off by {el.max():.3g}"


def _q(B, Hq, T, D, seed, spread=1.0):
    import torch
    g = torch.Generator(device="cuda").manual_seed(seed)
    return (torch.randn(B, T, Hq, D, device="cuda", generator=g) * spread).bfloat16().transpose(1, 2)


CASES = [
    # keys (the queries' included), Hq, Hkv, T, D, page, mask (left, right), mods
    ([1], 1, 1, 1, 128, 32, None, 0), ([0, 5, 33, 64], 8, 2, 1, 128, 64, None, 0), ([40, 65], 4, 4, 33, 64, 32, (-1, 0), 0),
    # 32 and 33 rows of a kv head, 128 and 129
    ([200], 8, 1, 4, 128, 64, (-1, 0), 0), ([200, 77], 33, 1, 1, 64, 96, (-1, 0), 0), ([500], 4, 1, 32, 128, 128, (-1, 0), 1),
    ([500], 3, 1, 43, 128, 64, (-1, 0), 0), ([300, 64, 31], 14, 2, 20, 64, 32, (-1, 0), 1), ([700, 3, 129], 6, 2, 3, 128, 32, (-1, 0), 0),
    ([333, 0, 90], 4, 4, 20, 64, 64, (50, 0), 0), ([900, 350, 1700], 4, 2, 700, 64, 64, (-1, 0), 0), ([3001], 3, 1, 513, 128, 64, (200, 0), 1),
    ([400, 2], 2, 2, 301, 32, 32, (-1, 5), 0), ([100, 7], 2, 1, 70, 32, 32, (-1, 0), 1), ([90, 4000], 4, 1, 2, 64, 32, (1000, -1), 0),
    ([50, 60], 4, 2, 30, 128, 64, (0, 0), 0), ([130] * 70, 2, 2, 5, 32, 32, (-1, 0), 0), ([256, 255], 16, 2, 64, 128, 256, (63, 0), 0),
    ([5000, 30], 2, 1, 40, 128, 512, None, 1), ([64, 128], 1, 1, 128, 128, 32, (-1, 3), 0),
]


@pytest.mark.parametrize("kind", ["bf16", "fp8"])
@pytest.mark.parametrize("case", CASES, ids=[str(i) for i in range(len(CASES))])
def test_padded(case, kind):
    import pallas_flexattn as pf
    lens, Hq, Hkv, T, D, page, win, mods = case
    c = _cache(kind, lens, Hkv, page, D, 21)
    q = _q(len(lens), Hq, T, D, 22)
    left, right = win or (-1, -1)
    mask = None if win is None else pf.MaskSpec(left=left, right=right)
    score = pf.compose_score_mods(pf.alibi_score_mod(Hq), pf.softcap_score_mod(15.0)) if mods else None
    o, lse = pf.flex_prefill(q, c.cache, c.lens, c.table, mask_mod=mask, score_mod=score, enable_gqa=True, return_lse=True)
    assert o.stride() == q.stride()
    _check(o, lse, q, c, lens, None, left, right, None, pf.alibi_slopes(Hq) if mods else None, 15.0 if mods else 0.0)
    assert (pf.flex_prefill(q, c.cache, c.lens, c.table, mask_mod=mask, score_mod=score, enable_gqa=True) == o).all()


@pytest.mark.parametrize("kind", ["bf16", "fp8"])
@pytest.mark.parametrize("new", [[1], [40, 1, 1, 0, 129, 3], [0, 0, 7], [64] * 3, [1] * 130 + [300]], ids=range(5))
def test_packed(new, kind):
    """Tokens of all rows one behind another, rows without any among them, and tokens behind the last row's."""
    import torch
    import pallas_flexattn as pf
    D, Hq, Hkv = 64, 6, 2
    lens = [n + 37 * (i % 5) for i, n in enumerate(new)]
    c = _cache(kind, lens, Hkv, 32, D, 5)
    starts = np.concatenate([[0], np.cumsum(new)])
    tail = 75
    q = _q(1, Hq, int(starts[-1]) + tail, D, 6)
    q[:, :, starts[-1]:] = float("nan")
    for dtype in (torch.int32, torch.int64):
        o, lse = pf.flex_prefill(q, c.cache, c.lens, c.table, mask_mod=pf.causal_mask, enable_gqa=True, return_lse=True,
                                 query_starts=torch.tensor(starts, device="cuda", dtype=dtype))
        assert o.stride() == q.stride()
        assert (o[:, :, starts[-1]:] == 0).all() and torch.isneginf(lse[:, :, starts[-1]:]).all()
        T = max(new)
        pad = torch.zeros(len(new), Hq, T, D, device="cuda", dtype=torch.bfloat16)
        po, pl = torch.zeros_like(pad), torch.full((len(new), Hq, T), float("-inf"), device="cuda")
        for b, n in enumerate(new):
            pad[b, :, :n] = q[0, :, starts[b]:starts[b + 1]]
            po[b, :, :n], pl[b, :, :n] = o[0, :, starts[b]:starts[b + 1]], lse[0, :, starts[b]:starts[b + 1]]
        _check(po, pl, pad, c, lens, new, -1, 0)


@pytest.mark.parametrize("kind", ["bf16", "fp8"])
@pytest.mark.parametrize("packed", [False, True])
def test_items_of_unequal_ranges(kind, packed):
    """300 items (packed: 304, the first of single tokens) where 512 run at a time: some in one range of keys, whose results the join
    must leave, the others in two."""
    import torch
    import pallas_flexattn as pf
    D, Hq, Hkv = 128, 16, 4
    new = [1] * 5 + [33] + [800] * 3 if packed else [800] * 3
    lens = [n + x for n, x in zip(new, (300, 0, 64, 1, 500, 100, 0, 77, 200) if packed else (0, 77, 200))]
    c = _cache(kind, lens, Hkv, 64, D, 41)
    if not packed:
        q = _q(3, Hq, 800, D, 42)
        o, lse = pf.flex_prefill(q, c.cache, c.lens, c.table, mask_mod=pf.causal_mask, enable_gqa=True, return_lse=True)
        return _check(o, lse, q, c, lens, None, -1, 0)
    starts = [0, *np.cumsum(new).tolist()]
    q = _q(1, Hq, starts[-1] + 9, D, 42)
    o, lse = pf.flex_prefill(q, c.cache, c.lens, c.table, mask_mod=pf.causal_mask, enable_gqa=True, return_lse=True,
                             query_starts=torch.tensor(starts, device="cuda", dtype=torch.int32))
    assert (o[:, :, starts[-1]:] == 0).all() and torch.isneginf(lse[:, :, starts[-1]:]).all()
    for some in (range(6), range(6, 9)):
        T = max(new[b] for b in some)
        pad = torch.zeros(len(some), Hq, T, D, device="cuda", dtype=torch.bfloat16)
        po, pl = torch.zeros_like(pad), torch.full((len(some), Hq, T), float("-inf"), device="cuda")
        for i, b in enumerate(some):
            pad[i, :, :new[b]] = q[0, :, starts[b]:starts[b + 1]]
            po[i, :, :new[b]], pl[i, :, :new[b]] = o[0, :, starts[b]:starts[b + 1]], lse[0, :, starts[b]:starts[b + 1]]
        part = type("Rows", (), {"rows": [x[some.start:some.stop] for x in c.rows]})
        _check(po, pl, pad, part, [lens[b] for b in some], [new[b] for b in some], -1, 0)


@pytest.mark.parametrize("kind", ["bf16", "fp8"])
def test_query_lens(kind):
    """Padded rows of every length, to none, whose padding is NaN; lengths past the sizes and below zero."""
    import torch
    import pallas_flexattn as pf
    lens, ql = [300, 12, 50, 200, 90], [150, 0, 33, 200, -4]
    c = _cache(kind, lens, 2, 64, 64, 7)
    q = _q(5, 4, 150, 64, 8)
    for b, n in enumerate(ql):
        q[b, :, max(n, 0):] = float("nan")
    o, lse = pf.flex_prefill(q, c.cache, c.lens, c.table, mask_mod=pf.causal_mask, enable_gqa=True, return_lse=True, query_lens=ql)
    clean = torch.nan_to_num(q)
    _check(o, lse, clean, c, lens, [150, 0, 33, 150, 0], -1, 0)


@pytest.mark.parametrize("kind", ["bf16", "fp8"])
def test_what_is_not_there(kind):
    """Lengths past the table and below zero, page ids outside the cache (zero keys), no lengths, no table, kv_len."""
    import torch
    import pallas_flexattn as pf
    c = _cache(kind, [192, 192, 192], 2, 64, 128, 9)
    q = _q(3, 4, 40, 128, 10)

    def run(**kw):
        return pf.flex_prefill(q, c.cache, mask_mod=pf.causal_mask, enable_gqa=True, return_lse=True, **kw)

    o, lse = run(kv_lens=[10 ** 6, -3, 2 ** 40], page_table=c.table)
    _check(o, lse, q, c, [192, 0, 192], None, -1, 0)
    o, lse = run(page_table=c.table.long())
    _check(o, lse, q, c, [192] * 3, None, -1, 0)
    o, lse = run(kv_lens=c.lens, page_table=c.table, kv_len=100)
    _check(o, lse, q, c, [100] * 3, None, -1, 0)
    bad = c.table.clone()
    bad[0, 1], bad[1, 0], bad[2, 2] = -1, 10 ** 6, 2 ** 31 - 1
    rows = [r.clone() for r in c.rows]
    for r in c.rows:
        r[0, :, 64:128], r[1, :, :64], r[2, :, 128:] = 0, 0, 0
    o, lse = run(kv_lens=c.lens, page_table=bad)
    _check(o, lse, q, c, [192] * 3, None, -1, 0)
    c.rows = rows
    one = _cache(kind, [50, 64], 2, 64, 128, 11)  # without a table page b is row b's
    order = one.table[:, 0].long()
    parts = [t[order] if t.dtype != torch.float8_e4m3fn else t.view(torch.uint8)[order].view(t.dtype) for t in one.cache]
    cache = pf.Fp8KVCache(*parts) if kind == "fp8" else tuple(parts)
    o, lse = pf.flex_prefill(q[:2], cache, one.lens, enable_gqa=True, return_lse=True)
    _check(o, lse, q[:2], one, [50, 64])


@pytest.mark.parametrize("T", [3, 90])  # items of at most 32 rows, and larger ones
@pytest.mark.parametrize("kind", ["bf16", "fp8"])
def test_values_that_are_not_finite(kind, T):
    """NaN and infinities in keys and values reach the queries that see them, and no others: causal, so that the
    queries of a tile differ; behind a window nobody sees them."""
    import torch
    import pallas_flexattn as pf
    lens, D = [400, 260], 64
    c = _cache(kind, lens, 2, 32, D, 13)
    q = _q(2, 4, T, D, 14)

    def put(which, b, h, key, d, x):
        page, row = int(c.table[b, key // 32]), key % 32
        t = c.cache[which]
        if kind == "fp8":
            t.view(torch.uint8)[page, h, row, d] = 0x7f
            x = float("nan")
        else:
            t[page, h, row, d] = x
        c.rows[which][b, h, key, d] = x

    inf = float("inf")
    put(1, 0, 0, 399, 3, inf)          # the last key: the last query alone
    put(1, 0, 1, 398, 5, float("nan"))
    put(1, 1, 0, 259, 9, -inf)
    put(1, 1, 0, 258, 9, inf)          # both: NaN for the last, inf for the one before
    put(0, 1, 1, 259, 7, float("nan"))  # a key: the whole row
    put(1, 0, 0, 20, 0, float("nan"))   # long before: behind the window
    put(0, 0, 0, 21, 0, float("nan"))
    put(1, 1, 1, 100, 1, inf)
    with np.errstate(invalid="ignore"):
        o, lse = pf.flex_prefill(q, c.cache, c.lens, c.table, mask_mod=pf.MaskSpec(left=60, right=0), enable_gqa=True, return_lse=True)
        _check(o, lse, q, c, lens, None, 60, 0)
        o, lse = pf.flex_prefill(q, c.cache, c.lens, c.table, mask_mod=pf.causal_mask, enable_gqa=True, return_lse=True)
        _check(o, lse, q, c, lens, None, -1, 0)


def test_large_scores_and_scale():
    """Scores that change by hundreds from key to key (the reference maximum moves all the time), a scale of one's own."""
    import pallas_flexattn as pf
    for kind in ("bf16", "fp8"):
        lens = [900, 450]
        c = _cache(kind, lens, 2, 64, 64, 31, spread=4.0)
        q = _q(2, 4, 60, 64, 32, spread=6.0)
        o, lse = pf.flex_prefill(q, c.cache, c.lens, c.table, scale=0.7, enable_gqa=True, return_lse=True)
        _check(o, lse, q, c, lens, scale=0.7)


def test_strides():
    """Queries that are a slice of a larger projection, that start off a 16-byte line, and that are expanded."""
    import torch
    import pallas_flexattn as pf
    c = _cache("bf16", [130, 70], 2, 64, 64, 41)
    wide = torch.randn(2, 50, 3, 4, 64, device="cuda").bfloat16()
    raw = torch.randn(2 * 4 * 50 * 64 + 1, device="cuda").bfloat16()
    for q in (wide[:, :, 1].transpose(1, 2), wide[:, ::2, 2].transpose(1, 2), raw[1:].reshape(2, 4, 50, 64),
              wide[:1, :, 0, :1].transpose(1, 2).expand(2, 4, 50, 64), wide[:, :, 0].permute(0, 2, 1, 3).flip(1)):
        o, lse = pf.flex_prefill(q, c.cache, c.lens, c.table, mask_mod=pf.causal_mask, enable_gqa=True, return_lse=True)
        _check(o, lse, q, c, [130, 70], None, -1, 0)


def test_splits_and_empty_calls():
    """A page table far wider than the rows (keys in many ranges, most of them empty); no tokens, no rows."""
    import torch
    import pallas_flexattn as pf
    for kind in ("bf16", "fp8"):
        lens = [70, 1, 3000]
        c = _cache(kind, lens, 1, 128, 128, 51, per_row=300)
        q = _q(3, 2, 50, 128, 52)
        o, lse = pf.flex_prefill(q, c.cache, c.lens, c.table, mask_mod=pf.causal_mask, enable_gqa=True, return_lse=True)
        c.rows = [r[:, :, :3008] for r in c.rows]
        _check(o, lse, q, c, lens, None, -1, 0)
        for z in (q[:, :, :0], q[:0]):
            o, lse = pf.flex_prefill(z, c.cache, c.lens[:z.shape[0]], c.table[:z.shape[0]], enable_gqa=True, return_lse=True)
            assert o.shape == z.shape and lse.shape == z.shape[:3]
    none = pf.flex_prefill(q[:1, :, :0], c.cache, c.lens, c.table, enable_gqa=True,
                           query_starts=torch.zeros(4, device="cuda", dtype=torch.int32))
    assert none.shape == (1, 2, 0, 128)


@pytest.mark.parametrize("kind", ["bf16", "fp8"])
def test_replays_of_a_graph(kind):
    """A captured call takes lengths, starts, tables and cache as they are at each replay, on another stream too."""
    import torch
    import pallas_flexattn as pf
    c = _cache(kind, [500, 40, 320], 2, 64, 64, 61)
    starts = torch.tensor([0, 100, 101, 140], device="cuda", dtype=torch.int32)
    q = _q(1, 4, 140, 64, 62).clone()
    lens = c.lens.clone()

    def run():
        return pf.flex_prefill(q, c.cache, lens, c.table, mask_mod=pf.causal_mask, enable_gqa=True, return_lse=True, query_starts=starts)

    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        run()
    torch.cuda.current_stream().wait_stream(s)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        o, lse = run()
    for st, ln in (([0, 100, 101, 140], [500, 40, 320]), ([0, 0, 2, 2], [100, 40, 64]), ([0, 1, 140, 140], [1, 40, 0])):
        starts.copy_(torch.tensor(st)), lens.copy_(torch.tensor(ln)), q.copy_(torch.randn_like(q.float()))
        g.replay()
        eo, el = run()
        assert torch.equal(o, eo) and torch.equal(lse, el)


def test_a_stream_of_its_own():
    import torch
    import pallas_flexattn as pf
    c = _cache("bf16", [500, 40], 2, 64, 64, 61)
    q = _q(2, 4, 40, 64, 62)
    want = pf.flex_prefill(q, c.cache, c.lens, c.table, mask_mod=pf.causal_mask, enable_gqa=True)
    torch.cuda.synchronize()
    s = torch.cuda.Stream()
    with torch.cuda.stream(s):
        later = torch.zeros_like(q)
        torch.cuda._sleep(10000000)
        later.copy_(q)
        got = pf.flex_prefill(later, c.cache, c.lens, c.table, mask_mod=pf.causal_mask, enable_gqa=True)
    s.synchronize()
    assert torch.equal(got, want)


def test_agrees_with_decode():
    """The same rows through flex_decode_fp8: both within rounding of one another."""
    import torch
    import pallas_flexattn as pf
    c = _cache("fp8", [900, 31, 64], 2, 64, 128, 71)
    q = _q(3, 8, 4, 128, 72)
    a, la = pf.flex_prefill(q, c.cache, c.lens, c.table, mask_mod=pf.causal_mask, enable_gqa=True, return_lse=True)
    b, lb = pf.flex_decode_fp8(q, c.cache, c.lens, c.table, mask_mod=pf.causal_mask, enable_gqa=True, return_lse=True)
    assert torch.allclose(a.float(), b.float(), atol=2 ** -7, rtol=2 ** -6)
    assert torch.allclose(la, lb, atol=1e-4) or torch.equal(torch.isinf(la), torch.isinf(lb))
