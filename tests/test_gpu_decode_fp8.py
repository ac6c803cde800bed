"""flex_decode_fp8 on the GPU against float64 attention over the dequantised cache (oracle/kv_cache.py).

Tolerance. Scores: sums of D products of exact bf16 operands in fp32, off by at most (D + 2) 2^-24 sum |q||k|
scale, the scale and log2 factors 3 2^-24 |s| more; the soft-cap's tanh (exp2 and rcp, each within 2^-22) adds
cap 2^-20, ALiBi's term rounds with the sum. A weight is then off by ds relative plus 2^-21 (exp2), its two bf16
pieces by 2^-16, and the sums of n weights by n 2^-24 at most: O is within half a bf16 step (2^-8 |o|) plus
c sum p |v|, c = 2 ds + 2^-16 + 2^-20 + 2 n 2^-24; LSE within ds + 2^-20 + n 2^-24 + 2^-22 |lse|."""
import numpy as np
import pytest

pytestmark = pytest.mark.gpu

from oracle import kv_cache  # noqa: E402
from tests.test_gpu_rotary import _np  # noqa: E402


class Cache:
    """Random rows of the given lengths in pages of random order; all that no row uses is NaN codes, with NaN scales."""

    def __init__(self, lens, H, page, D, seed, per_row=None, spread=1.0):
        import torch
        import pallas_flexattn as pf
        B = len(lens)
        per_row = per_row or max(1, -(-max(lens) // page))
        g = torch.Generator(device="cuda").manual_seed(seed)
        n = B * per_row + 2
        self.table = torch.randperm(n, generator=g, device="cuda")[:B * per_row].reshape(B, per_row).to(torch.int32)
        self.lens = torch.tensor(lens, device="cuda", dtype=torch.int32)
        S = per_row * page
        codes, scales, self.rows = [], [], []
        used = (torch.arange(S, device="cuda") < self.lens[:, None])  # (B, S)
        for _ in range(2):
            x = torch.randn(B, H, S, D, device="cuda", generator=g) * spread
            e = torch.randint(0, 5, (B, H, S // 32), device="cuda", generator=g)  # (448 2^-6 = 7: no code overflows)
            s = torch.exp2(e.float() - 6) * spread
            c = (x / s.repeat_interleave(32, 2)[..., None]).to(torch.float8_e4m3fn)
            val = c.float() * s.repeat_interleave(32, 2)[..., None]
            self.rows.append(torch.where(used[:, None, :, None], val, 0.0))
            c = torch.where(used[:, None, :, None], c.view(torch.uint8), 0x7f)
            s = torch.where(used.reshape(B, 1, -1, 32).any(-1), s, float("nan"))
            pc = torch.full((n, H, page, D), 0x7f, device="cuda", dtype=torch.uint8)
            ps = torch.full((n, H, page // 32), float("nan"), device="cuda")
            ids = self.table.long().reshape(-1)
            pc[ids] = c.reshape(B, H, per_row, page, D).transpose(1, 2).reshape(-1, H, page, D)
            ps[ids] = s.reshape(B, H, per_row, -1).transpose(1, 2).reshape(B * per_row, H, -1)
            codes.append(pc.view(torch.float8_e4m3fn))
            scales.append(ps)
        self.cache = pf.Fp8KVCache(*codes, *scales)


def _check(o, lse, q, c, lens, ql=None, left=-1, right=-1, scale=None, slopes=None, cap=0.0):
    D = q.shape[3]
    qn, k, v = _np(q), _np(c.rows[0]), _np(c.rows[1])
    wo, wl, w = kv_cache.decode(qn, k, v, lens, ql, left, right, scale, slopes, cap)
    sc = D ** -0.5 if scale is None else scale
    qmax = np.abs(qn).sum(-1).max() * np.abs(k).max() * sc  # an upper bound of sum |q||k| scale
    smax = qmax + (0 if slopes is None else float(np.max(np.abs(slopes))) * k.shape[2])
    ds = (D + 2) * 2.0 ** -24 * qmax + 4 * 2.0 ** -24 * smax + cap * 2.0 ** -20
    n = k.shape[2]
    c1 = 2 * ds + 2.0 ** -16 + 2.0 ** -20 + 2 * n * 2.0 ** -24
    go, gl = _np(o), _np(lse)
    assert np.all(np.isneginf(gl) == np.isneginf(wl))
    dead = np.isneginf(wl)
    assert np.all(go[dead] == 0)
    err = np.abs(go - wo)
    tol = np.abs(wo) * 2.0 ** -8 + c1 * w + 1e-30
    assert np.all(err <= tol), f"O off by {np.max(err / tol):.3g} times the tolerance"
    el = np.abs(gl[~dead] - wl[~dead])
    assert np.all(el <= ds + 2.0 ** -20 + n * 2.0 ** -24 + 2.0 ** -22 * np.abs(wl[~dead])), f"LSE off by {el.max():.3g}"


def _q(B, Hq, Sq, D, seed, spread=1.0):
    import torch
    g = torch.Generator(device="cuda").manual_seed(seed)
    return (torch.randn(B, Hq, Sq, D, device="cuda", generator=g) * spread).bfloat16()


CASES = [
    # lens, Hq, Hkv, Sq, D, page, mask (left, right), mods
    ([1], 1, 1, 1, 128, 32, None, 0), ([0, 5, 33, 64], 8, 2, 1, 128, 64, None, 0), ([1000, 31, 32], 4, 4, 1, 64, 128, None, 0),
    ([700, 3, 129], 6, 2, 3, 128, 32, (-1, 0), 0), ([513], 8, 1, 4, 32, 96, (-1, 0), 0), ([300, 64], 14, 2, 1, 64, 64, None, 1),
    ([2000, 40], 8, 2, 5, 128, 256, (100, 0), 1), ([333, 0, 90], 4, 4, 20, 64, 64, (50, 0), 0), ([640], 16, 2, 9, 128, 64, (-1, 0), 0),
    ([100, 7], 2, 1, 70, 32, 32, (-1, 0), 1), ([5000], 8, 8, 1, 128, 512, None, 0), ([90, 4000], 4, 1, 2, 64, 32, (1000, -1), 0),
    ([50, 60], 4, 2, 3, 128, 64, (-1, 2), 0), ([65] * 70, 2, 2, 1, 32, 32, None, 0), ([17, 450] * 140, 2, 1, 1, 32, 32, None, 0),
    # chunks of a prompt: hundreds of rows per kv head, more queries than keys in a row, odd row counts
    ([900, 350, 1700], 4, 2, 700, 64, 64, (-1, 0), 0), ([3001], 3, 1, 513, 128, 64, (200, 0), 1), ([400, 2], 2, 2, 301, 32, 32, (-1, 5), 0),
]


@pytest.mark.parametrize("case", CASES, ids=[str(i) for i in range(len(CASES))])
def test_decode(case):
    import pallas_flexattn as pf
    lens, Hq, Hkv, Sq, D, page, win, mods = case
    c = Cache(lens, Hkv, page, D, 21)
    q = _q(len(lens), Hq, Sq, D, 22)
    left, right = win or (-1, -1)
    mask = None if win is None else pf.MaskSpec(left=left, right=right)
    score = pf.compose_score_mods(pf.alibi_score_mod(Hq), pf.softcap_score_mod(15.0)) if mods else None
    o, lse = pf.flex_decode_fp8(q, c.cache, c.lens, c.table, mask_mod=mask, score_mod=score, enable_gqa=True, return_lse=True)
    _check(o, lse, q, c, lens, None, left, right, None, pf.alibi_slopes(Hq) if mods else None, 15.0 if mods else 0.0)
    assert (pf.flex_decode_fp8(q, c.cache, c.lens, c.table, mask_mod=mask, score_mod=score, enable_gqa=True) == o).all()


LARGE = [
    # lens, Hq, Hkv, Sq, D, pages per row of 512 tokens, mask, mods: page tables long enough that 32-row items (more than
    # 16 rows) and reads past the caches are chosen
    ([900, 40], 16, 2, 3, 128, 200, (-1, 0), 0), ([33, 2000], 8, 2, 5, 64, 200, None, 1), ([700, 0], 14, 2, 5, 32, 300, (300, 0), 0),
    ([1500, 1], 4, 2, 1, 128, 400, None, 0), ([3000, 100], 4, 2, 2, 64, 600, (-1, 0), 1), ([600, 64], 32, 2, 1, 32, 800, None, 0),
]


@pytest.mark.parametrize("case", LARGE, ids=[str(i) for i in range(len(LARGE))])
def test_large_tables(case):
    import pallas_flexattn as pf
    lens, Hq, Hkv, Sq, D, pages, win, mods = case
    c = Cache(lens, Hkv, 512, D, 23, per_row=pages)
    q = _q(len(lens), Hq, Sq, D, 24)
    left, right = win or (-1, -1)
    mask = None if win is None else pf.MaskSpec(left=left, right=right)
    score = pf.compose_score_mods(pf.alibi_score_mod(Hq), pf.softcap_score_mod(15.0)) if mods else None
    o, lse = pf.flex_decode_fp8(q, c.cache, c.lens, c.table, mask_mod=mask, score_mod=score, enable_gqa=True, return_lse=True)
    keep = -(-max(lens) // 32) * 32
    c.rows = [r[:, :, :keep] for r in c.rows]
    _check(o, lse, q, c, lens, None, left, right, None, pf.alibi_slopes(Hq) if mods else None, 15.0 if mods else 0.0)


def test_large_scores_and_scale():
    """Scores that change by hundreds from key to key (the running maximum moves all the time), a scale of one's own."""
    import pallas_flexattn as pf
    lens = [900, 450]
    c = Cache(lens, 2, 64, 64, 31, spread=4.0)
    q = _q(2, 4, 2, 64, 32, spread=6.0)
    o, lse = pf.flex_decode_fp8(q, c.cache, c.lens, c.table, scale=0.7, enable_gqa=True, return_lse=True)
    _check(o, lse, q, c, lens, scale=0.7)


def test_many_rows():
    """Row counts around and past what a wave's lanes hold, with items cut in pieces: short rows beside long ones."""
    import torch
    import pallas_flexattn as pf
    for B in (63, 64, 65, 129, 256, 257):
        lens = [(37 * i) % 90 for i in range(B)]
        lens[B // 2], lens[B - 1] = 2500, 1700
        c = Cache(lens, 1, 512, 32, 33, per_row=9)  # (long enough tables to be cut in pieces)
        q = _q(B, 2, 1, 32, 34)
        o, lse = pf.flex_decode_fp8(q, c.cache, c.lens, c.table, enable_gqa=True, return_lse=True)
        _check(o, lse, q, c, lens)


@pytest.mark.parametrize("B", [258, 319, 1023, 1024, 1025])
def test_hundreds_of_rows(B):
    """More rows than a wave's lanes hold four each of, up to sixteen each and past that."""
    import pallas_flexattn as pf
    lens = [(37 * i) % 90 for i in range(B)]
    lens[B // 3], lens[B - 1] = 2500, 1700
    c = Cache(lens, 1, 512, 32, 37, per_row=9)
    q = _q(B, 2, 1, 32, 38)
    o, lse = pf.flex_decode_fp8(q, c.cache, c.lens, c.table, enable_gqa=True, return_lse=True)
    _check(o, lse, q, c, lens)


def test_kv_len_bounds_the_keys():
    """A bound on the keys under the table's width: same results, longer rows cut, rows without lengths that long."""
    import pallas_flexattn as pf
    lens = [70, 33, 0, 512]
    c = Cache(lens, 2, 64, 64, 38, per_row=60)
    q = _q(4, 4, 2, 64, 39)
    kw = dict(mask_mod=pf.causal_mask, enable_gqa=True, return_lse=True)
    for bound in (512, 513, 3839, 3840):
        o, lse = pf.flex_decode_fp8(q, c.cache, c.lens, c.table, kv_len=bound, **kw)
        _check(o, lse, q, c, lens, None, -1, 0)
    o, lse = pf.flex_decode_fp8(q, c.cache, c.lens, c.table, kv_len=50, **kw)
    _check(o, lse, q, c, [min(n, 50) for n in lens], None, -1, 0)
    o, lse = pf.flex_decode_fp8(q, c.cache, None, c.table, kv_len=33, **kw)
    want, wl = pf.flex_decode_fp8(q, c.cache, [33] * 4, c.table, kv_len=33, **kw)
    assert (o[:2] == want[:2]).all() and (lse[:2] == wl[:2]).all()


def test_window_without_an_end():
    """Window sides past every key, at the largest 32-bit number and above it."""
    import pallas_flexattn as pf
    c = Cache([70, 3], 1, 32, 64, 35)
    q = _q(2, 2, 2, 64, 36)
    want, wl = pf.flex_decode_fp8(q, c.cache, c.lens, c.table, mask_mod=pf.causal_mask, enable_gqa=True, return_lse=True)
    _check(want, wl, q, c, [70, 3], None, -1, 0)
    for left in (96, 2 ** 31 - 1, 2 ** 40):
        got = pf.flex_decode_fp8(q, c.cache, c.lens, c.table, mask_mod=pf.sliding_window_mask(left, 0), enable_gqa=True)
        assert (got == want).all()
    both = pf.flex_decode_fp8(q, c.cache, c.lens, c.table, mask_mod=pf.sliding_window_mask(2 ** 40, 2 ** 40), enable_gqa=True)
    assert (both == pf.flex_decode_fp8(q, c.cache, c.lens, c.table, enable_gqa=True)).all()


def test_padded_queries():
    import torch
    import pallas_flexattn as pf
    lens, ql = [200, 33, 5, 64], [3, 0, 5, 1]
    c = Cache(lens, 2, 32, 128, 41)
    q = _q(4, 8, 5, 128, 42)
    o, lse = pf.flex_decode_fp8(q, c.cache, c.lens, c.table, mask_mod=pf.sliding_window_mask(40, 0), enable_gqa=True,
                                return_lse=True, query_lens=torch.tensor(ql, device="cuda"))
    spec = pf.sliding_window_mask(40, 0)
    _check(o, lse, q, c, lens, ql, spec.left, spec.right)


def test_pages_before_the_window_may_be_anything():
    """A sliding window's old pages given back: table entries of them and all they hold are garbage."""
    import torch
    import pallas_flexattn as pf
    lens, left = [300, 170], 60
    c = Cache(lens, 2, 32, 64, 48)
    q = _q(2, 4, 2, 64, 49)
    first = [n - 2 - left for n in lens]  # the first key that the first query sees
    codes = [t.view(torch.uint8) for t in c.cache[:2]]
    table = c.table.clone()
    for b, n in enumerate(first):
        for t in codes:
            t[c.table[b, n // 32].long(), :, :n % 32] = 0xff
        table[b, :n // 32] = -5
    o, lse = pf.flex_decode_fp8(q, c.cache, c.lens, table, mask_mod=pf.sliding_window_mask(left, 0), enable_gqa=True,
                                return_lse=True)
    _check(o, lse, q, c, lens, None, left, 0)


@pytest.mark.parametrize("D,Hq,Sq,left", [(128, 4, 4, -1), (64, 2, 40, 37), (32, 12, 5, 70)])
def test_nan_reaches_the_queries_that_see_it(D, Hq, Sq, left):
    """NaN in single elements of keys and values that some queries see and others, masked, do not."""
    import torch
    import pallas_flexattn as pf
    lens = [150, 97]
    c = Cache(lens, 1, 32, D, 50)
    q = _q(2, Hq, Sq, D, 55)
    dims = {0: (0, D - 1), 1: (3, D // 2)}  # of the values, per row
    codes = [t.view(torch.uint8) for t in c.cache[:2]]
    hit = np.zeros((2, Hq, Sq, D), bool)
    for b, n in enumerate(lens):
        # a value of the newest key, of the one before the last query's, and of one that a window ends on; a key's element
        for pos, what in ((n - 1, "v"), (n - 2, "k"), (max(n - Sq - max(left, 0), 0), "v")):
            page = c.table[b, pos // 32].long()
            for i in range(Sq):
                at = n - Sq + i
                if pos <= at and (left < 0 or at - pos <= left):
                    hit[b, :, i, list(dims[b]) if what == "v" else slice(None)] = True
            if what == "v":
                for d in dims[b]:
                    codes[1][page, :, pos % 32, d] = 0x7f if d else 0xff
            else:
                codes[0][page, :, pos % 32, 1] = 0x7f
    o, lse = pf.flex_decode_fp8(q, c.cache, c.lens, c.table, mask_mod=pf.sliding_window_mask(left, 0), enable_gqa=True,
                                return_lse=True)
    assert np.array_equal(np.isnan(_np(o)), hit)
    wo, wl, _ = kv_cache.decode(_np(q), _np(c.rows[0]), _np(c.rows[1]), lens, None, left, 0)
    clean = ~hit.any(-1)
    np.testing.assert_allclose(_np(o)[~hit & clean[..., None]], wo[~hit & clean[..., None]], rtol=2.0 ** -7, atol=1e-3)


@pytest.mark.parametrize("masked", [False, True])
@pytest.mark.parametrize("n", [70, 2000])  # in one workgroup per item, in pieces
def test_padded_queries_are_zero_beside_nan(n, masked):
    """Padded queries give 0 and -inf also where every value that the others see is NaN."""
    import torch
    import pallas_flexattn as pf
    c = Cache([n, n, n], 1, 32, 64, 51)
    q = _q(3, 4, 3, 64, 52)
    c.cache[1].view(torch.uint8).fill_(0x7f)
    ql = torch.tensor([0, 1, 3], device="cuda")
    o, lse = pf.flex_decode_fp8(q, c.cache, c.lens, c.table, mask_mod=pf.causal_mask if masked else None, enable_gqa=True,
                                return_lse=True, query_lens=ql)
    for b, m in enumerate((0, 1, 3)):
        assert torch.isnan(o[b, :, :m]).all() and torch.isfinite(lse[b, :, :m]).all()
        assert (o[b, :, m:] == 0).all() and (lse[b, :, m:] == float("-inf")).all()


def test_more_queries_than_keys():
    """Queries before the first position see nothing (a row of 2 keys, 4 causal queries)."""
    import pallas_flexattn as pf
    c = Cache([2, 40], 1, 32, 64, 43)
    q = _q(2, 2, 4, 64, 44)
    o, lse = pf.flex_decode_fp8(q, c.cache, c.lens, c.table, mask_mod=pf.causal_mask, enable_gqa=True, return_lse=True)
    _check(o, lse, q, c, [2, 40], None, -1, 0)


def test_bad_pages_are_zero_keys_and_lengths_are_clamped():
    import torch
    import pallas_flexattn as pf
    lens = [130, 64]
    c = Cache(lens, 2, 32, 64, 45)
    q = _q(2, 4, 1, 64, 46)
    table = c.table.clone()
    table[0, 1], table[0, 3], table[1, 0] = -1, 10 ** 8, 2 ** 31 - 1
    for r in c.rows:
        r[0, :, 32:64], r[0, :, 96:128], r[1, :, :32] = 0, 0, 0
    o, lse = pf.flex_decode_fp8(q, c.cache, c.lens, table, enable_gqa=True, return_lse=True)
    _check(o, lse, q, c, lens)
    c = Cache([64, 64], 2, 32, 64, 47)
    o, lse = pf.flex_decode_fp8(q, c.cache, torch.tensor([10 ** 6, -4], device="cuda"), c.table, enable_gqa=True, return_lse=True)
    _check(o, lse, q, c, [64, 0])


def test_whole_table_strides_and_no_table():
    import pallas_flexattn as pf
    c = Cache([96, 96, 96], 2, 96, 128, 51)
    q = _q(3, 6, 2, 128, 52)
    want, wl = pf.flex_decode_fp8(q, c.cache, None, c.table, enable_gqa=True, return_lse=True)
    _check(want, wl, q, c, [96] * 3)
    v = q.transpose(1, 2).contiguous().transpose(1, 2)
    got = pf.flex_decode_fp8(v, c.cache, c.lens.long(), c.table.long(), enable_gqa=True)
    assert (got == want).all()
    odd = q.new_zeros(3, 6, 2, 129)[..., 1:]  # rows that are not 16-byte aligned
    assert (pf.flex_decode_fp8(odd.copy_(q), c.cache, c.lens, c.table, enable_gqa=True) == want).all()
    rows = [t[c.table[:, 0].long()].contiguous() for t in c.cache]
    assert (pf.flex_decode_fp8(q, pf.Fp8KVCache(*rows), [96] * 3, enable_gqa=True) == want).all()
    # slots of nobody's pages and of unused rows do not matter: garbage elsewhere changes nothing
    assert pf.flex_decode_fp8(q[:0], c.cache, c.lens[:0], c.table[:0], enable_gqa=True).shape == (0, 6, 2, 128)
    assert pf.flex_decode_fp8(q[:, :, :0], c.cache, c.lens, c.table, enable_gqa=True).numel() == 0


def test_two_threads_at_once():
    """The launcher from two threads, each on a stream of its own."""
    import threading
    import torch
    import pallas_flexattn as pf
    c = Cache([3000, 500], 2, 64, 64, 63)
    q = _q(2, 8, 1, 64, 64)
    want = pf.flex_decode_fp8(q, c.cache, c.lens, c.table, enable_gqa=True)
    torch.cuda.synchronize()
    got = [None, None]

    def work(i):
        s = torch.cuda.Stream()
        with torch.cuda.stream(s):
            got[i] = [pf.flex_decode_fp8(q, c.cache, c.lens, c.table, enable_gqa=True) for _ in range(20)]
        s.synchronize()

    ts = [threading.Thread(target=work, args=(i,)) for i in range(2)]
    for t in ts:
        t.start()
    for t in ts:
        t.join()
    assert all(torch.equal(o, want) for g in got for o in g)


def test_same_results_alone_and_in_a_batch_order():
    """A row's result does not depend on its neighbours beyond the order in which its pieces are added."""
    import torch
    import pallas_flexattn as pf
    lens = [3000, 17, 1200, 800]
    c = Cache(lens, 2, 64, 128, 61)
    q = _q(4, 8, 1, 128, 62)
    a, la = pf.flex_decode_fp8(q, c.cache, c.lens, c.table, enable_gqa=True, return_lse=True)
    b, lb = pf.flex_decode_fp8(q, c.cache, c.lens, c.table, enable_gqa=True, return_lse=True)
    assert torch.equal(a, b) and torch.equal(la, lb)
    for i in range(4):
        o, l = pf.flex_decode_fp8(q[i:i + 1], c.cache, c.lens[i:i + 1], c.table[i:i + 1], enable_gqa=True, return_lse=True)
        np.testing.assert_allclose(_np(o), _np(a[i:i + 1]), rtol=2.0 ** -7, atol=1e-4)
        np.testing.assert_allclose(_np(l), _np(la[i:i + 1]), rtol=1e-5, atol=1e-5)


def test_serving_run_eager_graph_and_streams():
    """Prompt, then token by token: append and decode together, eager and as a captured graph replayed with new
    contents, against attention over the cache that the appends left; two streams at once."""
    import torch
    import pallas_flexattn as pf
    B, Hq, Hkv, D, page, T = 3, 8, 2, 128, 64, 70
    rot = pf.rotary_embedding(D)
    cache = pf.create_fp8_kv_cache(B * 2, Hkv, page, D)
    cache.key.view(torch.uint8).fill_(0x7f), cache.value.view(torch.uint8).fill_(0x7f)
    table = torch.randperm(B * 2, device="cuda").reshape(B, 2).to(torch.int32)
    lens = torch.zeros(B, device="cuda", dtype=torch.int32)
    new = torch.tensor([70, 33, 1], device="cuda", dtype=torch.int32)
    mk = lambda h, t: torch.randn(B, t, h, D, device="cuda").bfloat16().transpose(1, 2)  # noqa: E731

    class View:
        def __init__(self):
            k, v = cache.dequantize()
            self.rows = [torch.nan_to_num(x[table.long()].transpose(1, 2).reshape(B, Hkv, -1, D)) for x in (k, v)]

    q, k, v = mk(Hq, T), mk(Hkv, T), mk(Hkv, T)
    q2 = pf.append_kv_cache(cache, k, v, lens, table, new_lens=new, rotary=rot, query=q)
    lens = lens + new
    o, lse = pf.flex_decode_fp8(q2, cache, lens, table, mask_mod=pf.causal_mask, enable_gqa=True, return_lse=True, query_lens=new)
    _check(o, lse, q2, View(), lens.tolist(), new.tolist(), -1, 0)

    q, k, v = mk(Hq, 1), mk(Hkv, 1), mk(Hkv, 1)
    after = lens + 1

    def step():
        q2 = pf.append_kv_cache(cache, k, v, lens, table, rotary=rot, query=q)
        return (q2,) + pf.flex_decode_fp8(q2, cache, after, table, mask_mod=pf.causal_mask, enable_gqa=True, return_lse=True)

    want = step()
    _check(want[1], want[2], want[0], View(), after.tolist(), None, -1, 0)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = step()
    for i in range(3):
        for t, h in ((q, Hq), (k, Hkv), (v, Hkv)):
            t.copy_(mk(h, 1))
        lens.copy_(after), after.add_(1)
        graph.replay()
        torch.cuda.synchronize()
        _check(got[1], got[2], got[0], View(), after.tolist(), None, -1, 0)
        want = step()  # the same tokens again, eagerly: the run's scale stays, the codes are the same
        assert all(torch.equal(a, b) for a, b in zip(got, want))
    s = [torch.cuda.Stream() for _ in range(2)]
    outs = []
    for x in s:
        x.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(x):
            outs.append([pf.flex_decode_fp8(got[0], cache, after, table, enable_gqa=True) for _ in range(4)])
    for x in s:
        torch.cuda.current_stream().wait_stream(x)
    ref = pf.flex_decode_fp8(got[0], cache, after, table, enable_gqa=True)
    assert all(torch.equal(o, ref) for os in outs for o in os)


def test_bf16_cache_filled_by_append_serves_flex_decode():
    import torch
    import pallas_flexattn as pf
    B, Hq, Hkv, D, page = 2, 4, 2, 64, 64
    rot = pf.rotary_embedding(D)
    caches = tuple(torch.zeros(B * 3, Hkv, page, D, device="cuda", dtype=torch.bfloat16) for _ in range(2))
    table = torch.randperm(B * 3, device="cuda").reshape(B, 3).to(torch.int32)
    new = [150, 90]
    mk = lambda h: torch.randn(B, 150, h, D, device="cuda").bfloat16().transpose(1, 2)  # noqa: E731
    q, k, v = mk(Hq), mk(Hkv), mk(Hkv)
    pf.append_kv_cache(caches, k, v, [0, 0], table, new_lens=new, rotary=rot, query=q)
    k2 = pf.apply_rotary(k, None, rot)
    o = pf.flex_decode(q[:, :, :1], caches[0], caches[1], enable_gqa=True, kv_lens=torch.tensor(new, device="cuda"), page_table=table)
    for b in range(B):
        want = pf.flex_attention(q[b:b + 1, :, :1], k2[b:b + 1, :, :new[b]], v[b:b + 1, :, :new[b]], enable_gqa=True)
        np.testing.assert_allclose(_np(o[b:b + 1]), _np(want), rtol=2e-2, atol=2e-2)


def test_offsets_past_32_bits():
    """Pages past the 4 GiB of a cache's bytes: the last pages of a large pool."""
    import torch
    import pallas_flexattn as pf
    H, page, D, n = 8, 512, 128, 8300  # 4.35e9 bytes per tensor
    small = Cache([700], H, page, D, 71)
    cache = pf.create_fp8_kv_cache(n, H, page, D)
    ids = torch.tensor([[n - 1, n - 2]], device="cuda", dtype=torch.int32)
    for big, few in zip(cache, small.cache):
        a, b = (t.view(torch.uint8) if t.dtype == torch.float8_e4m3fn else t for t in (big, few))
        a[ids.long()[0]] = b[small.table.long()[0]]
    q = _q(1, 16, 1, D, 72)
    want = pf.flex_decode_fp8(q, small.cache, [700], small.table, enable_gqa=True)
    assert torch.equal(pf.flex_decode_fp8(q, cache, [700], ids, enable_gqa=True), want)
    k = torch.randn(1, H, 3, D, device="cuda").bfloat16()
    for c, t in ((cache, ids), (small.cache, small.table)):
        pf.append_kv_cache(c, k, k, [700], t)
    want = pf.flex_decode_fp8(q, small.cache, [703], small.table, enable_gqa=True)
    assert torch.equal(pf.flex_decode_fp8(q, cache, [703], ids, enable_gqa=True), want)
