"""flex_decode_fp8 where an item takes 32 query rows, and where few rows of D = 32 are cut in pieces: every form of those
kernels (head dim, masks that differ between rows or not, reads past the caches or not, one workgroup per item or
pieces), against the float64 attention and its tolerances of test_gpu_decode_fp8.

The host decides by the page table's width, so the tables are wide: past the rows' pages, entries outside the cache."""
import ctypes

import numpy as np
import pytest

pytestmark = pytest.mark.gpu

from oracle import kv_cache  # noqa: E402
from tests.test_gpu_decode_fp8 import Cache, _check, _q  # noqa: E402
from tests.test_gpu_rotary import _np  # noqa: E402

# lens, Hq, Hkv, Sq, D, tiles of 32 keys that the table holds, mask (left, right), mods, 16-row blocks per item, pieces, stream
PIECES = [
    ([2500, 40], 48, 2, 1, 128, 6000, None, 0, 2, True, True), ([1900], 120, 3, 1, 128, 4000, None, 0, 2, True, False),
    ([2100, 0], 34, 2, 1, 64, 6000, None, 0, 2, True, False), ([33, 1800], 76, 2, 1, 64, 8000, None, 0, 2, True, True),
    ([1700, 31], 66, 2, 1, 32, 3500, None, 0, 2, True, False), ([2049, 600], 46, 2, 1, 32, 16000, None, 0, 2, True, True),
    ([2200, 300], 14, 2, 3, 128, 6000, (-1, 0), 0, 2, True, True), ([1500], 3, 3, 37, 128, 4100, (-1, 0), 0, 2, True, False),
    ([3, 1300], 10, 2, 5, 64, 6100, (-1, 1), 1, 2, True, False), ([1999, 64], 40, 2, 1, 64, 8000, None, 1, 2, True, True),
    ([2500, 100], 22, 2, 3, 32, 6000, (-1, 0), 0, 2, True, False), ([1600, 18], 62, 2, 1, 32, 15000, None, 1, 2, True, True),
    # a long window, many rows
    ([(97 * i) % 700 for i in range(126)] + [3500], 18, 2, 2, 32, 200, (3000, 0), 0, 2, True, False),
    # up to 16 rows, score mods, cut in pieces
    ([3000, 5], 30, 2, 1, 32, 200, None, 1, 1, True, False), ([2600], 5, 1, 3, 32, 40000, (-1, 0), 1, 1, True, False),
    ([2600, 2], 8, 2, 2, 32, 20000, (-1, 0), 0, 1, True, True),
]
BY_ITEM = [
    ([(53 * i) % 300 for i in range(63)] + [3000], 24 * h // 4, h, 3, D, 94, None, m, 2, False, D == 128)
    for D, h, m in ((128, 4, 0), (64, 4, 0), (32, 4, 0), (128, 4, 1))
] + [
    ([(31 * i) % 200 for i in range(64)], 28, 4, 3, 64, 94, (-1, 0), 1, 2, False, False),
    ([(31 * i) % 200 for i in range(64)], 20, 4, 5, 32, 94, (-1, 0), 0, 2, False, False),
    ([(71 * i) % 1500 for i in range(16)], 16 * 17, 16, 2, 64, 47, (-1, 0), 0, 2, False, False),  # (short walks)
]
CASES = PIECES + BY_ITEM


def _workspace(B, Hq, Hkv, Sq, D, tiles, left, right):
    """What the library asks for, and what it would with 1 or 2 blocks of rows per item cut in pieces: each piece's slot
    holds 16 rows of D + 2 floats per block."""
    import torch
    from pallas_flexattn import _lib
    p = _lib.FaParams()
    p.abi_version, p.dtype = _lib.ABI_VERSION, _lib.DTYPE_FP8_E4M3
    p.B, p.Hq, p.Hkv, p.Sq, p.Skv, p.D, p.window_left, p.window_right = B, Hq, Hkv, Sq, 32 * tiles, D, left, right
    got = _lib.load().fa_fwd_kvcache_fp8_workspace_bytes(
        ctypes.byref(p), ctypes.byref(_lib.FaFp8Cache(16, 16, 16, 16, 16, 32, tiles, 8, 16, None)))
    rows, pieces = Hq // Hkv * Sq, 4 * torch.cuda.get_device_properties(0).multi_processor_count
    walk = tiles if left < 0 else min(tiles, (left + Sq + 30) // 32 + 1)
    want = {}
    for nq in (1, 2):
        items = B * Hkv * -(-rows // (16 * nq))
        grid = min(items * -(-walk // (8 if walk <= 128 else 16)), items + pieces)
        want[nq] = -(-(8 * B + 8) // 256) * 256 + min(grid, 2 * pieces) * 16 * nq * (D + 2) * 4
    return got, want


def _table(c, tiles):
    import torch
    B, n = c.table.shape
    wide = torch.full((B, tiles), -1, device="cuda", dtype=torch.int32)
    wide[:, :n] = c.table
    return wide


def _call(case, seed, query_lens=None, cache=None):
    import pallas_flexattn as pf
    lens, Hq, Hkv, Sq, D, tiles, win, mods = case[:8]
    c = cache or Cache(lens, Hkv, 32, D, seed)
    q = _q(len(lens), Hq, Sq, D, seed + 1)
    left, right = win or (-1, -1)
    mask = None if win is None else pf.MaskSpec(left=left, right=right)
    score = pf.compose_score_mods(pf.alibi_score_mod(Hq), pf.softcap_score_mod(15.0)) if mods else None
    o, lse = pf.flex_decode_fp8(q, c.cache, c.lens, _table(c, tiles), mask_mod=mask, score_mod=score, enable_gqa=True,
                                return_lse=True, query_lens=query_lens)
    return c, q, o, lse, left, right


@pytest.mark.parametrize("case", CASES, ids=[str(i) for i in range(len(CASES))])
def test_blocks(case):
    import pallas_flexattn as pf
    lens, Hq, Hkv, Sq, D, tiles, win, mods, nq, pieces, _ = case
    need, with_blocks = _workspace(len(lens), Hq, Hkv, Sq, D, tiles, *(win or (-1, -1)))
    assert need == (with_blocks[nq] if pieces else 0), "not the form that this case is for"
    c, q, o, lse, left, right = _call(case, 71)
    _check(o, lse, q, c, lens, None, left, right, None, pf.alibi_slopes(Hq) if mods else None, 15.0 if mods else 0.0)
    again = _call(case, 71, cache=c)
    assert (again[2] == o).all() and (again[3] == lse).all()


PADDED = [PIECES[6], PIECES[8], PIECES[10], BY_ITEM[5]]


@pytest.mark.parametrize("case", PADDED, ids=[str(i) for i in range(len(PADDED))])
def test_padded_queries(case):
    import torch
    import pallas_flexattn as pf
    lens, Hq, Hkv, Sq, D, tiles, win, mods = case[:8]
    ql = [(i + 1) % (Sq + 1) for i in range(len(lens))]
    c, q, o, lse, left, right = _call(case, 73, torch.tensor(ql, device="cuda"))
    _check(o, lse, q, c, lens, ql, left, right, None, pf.alibi_slopes(Hq) if mods else None, 15.0 if mods else 0.0)


@pytest.mark.parametrize("D", [128, 64, 32])
@pytest.mark.parametrize("short", [False, True])  # (pieces, or one workgroup per item)
def test_nan_reaches_the_queries_that_see_it(D, short):
    """In both blocks of an item: causal queries, a NaN value of the newest key and of the one before, a NaN key."""
    import torch
    B, Sq, g = (64, 9, 3) if short else (2, 9, 3)
    Hkv, tiles = (4, 94) if short else (1, 12000)
    lens = [70 + (i * 13) % 50 for i in range(B - 1)] + [2000]
    case = (lens, g * Hkv, Hkv, Sq, D, tiles, (-1, 0), 0)
    c = Cache(lens, Hkv, 32, D, 75)
    hit = np.zeros((B, g * Hkv, Sq, D), bool)
    codes = [t.view(torch.uint8) for t in c.cache[:2]]
    for b in (0, B - 1):
        n = lens[b]
        for pos, what, d in ((n - 1, 1, D - 1), (n - 4, 1, 0), (n - 2, 0, 3)):
            codes[what][c.table[b, pos // 32].long(), :, pos % 32, d] = 0x7f
            hit[b, :, Sq - (n - pos):, d if what else slice(None)] = True
    need, with_blocks = _workspace(B, g * Hkv, Hkv, Sq, D, tiles, -1, 0)
    assert need == (0 if short else with_blocks[2])
    _, q, o, lse, left, right = _call(case, 75, cache=c)
    assert np.array_equal(np.isnan(_np(o)), hit)
    wo, _, _ = kv_cache.decode(_np(q), _np(c.rows[0]), _np(c.rows[1]), lens, None, left, right)
    clean = ~hit.any(-1)
    np.testing.assert_allclose(_np(o)[clean], wo[clean], rtol=2.0 ** -7, atol=1e-3)
