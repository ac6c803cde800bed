"""flex_decode_latent over values that are not finite, in tiles that only some of the queries see: their scores are those of the
values as they are, whichever wave of the workgroup comes first.  (A wave takes the scores of 16 of a tile's 64 keys; the
tile's values belong to all waves in pieces of 1 KB.)"""
import numpy as np
import pytest

pytestmark = pytest.mark.gpu

from tests.test_gpu_latent import Latent, _check, _q  # noqa: E402

VALUES = (float("nan"), float("inf"), -float("inf"))


def _run(L, R, H, T, part, left):
    """A batch row per value, element and place of the key among its tile's: the newest keys (some queries stand before them), or
    those that a window leaves to the first queries only."""
    import pallas_flexattn as pf
    elements = (0, 7, L // 2 + 3, L - 1) if part == "latent" else (L, L + R // 2 + 1, L + R - 1)
    rows = [(x, d, at) for x in VALUES for d in elements for at in (2, 18, 35, 51, 63)]
    lens = [256 + at + 1 for _, _, at in rows]  # the newest key is number `at` of a tile of 64, in one wave's keys or another's
    c = Latent(lens, L, R, 64, 17)
    q, qr = _q(len(rows), H, T, L, R, 18)
    for b, (x, d, _) in enumerate(rows):
        # seen by the last query, or the last two; behind a window: by the first, or the first two
        key = lens[b] - 1 - b % 2 if left < 0 else lens[b] - T - left + b % 2
        c.cache.data[int(c.table[b, key // 64]), key % 64, d] = x
        c.rows[b, key, d] = x

    def call():
        return pf.flex_decode_latent(q, qr, c.cache, 0.1, c.lens, c.table, mask_mod=pf.MaskSpec(left=left, right=0), return_lse=True)

    with np.errstate(invalid="ignore"):
        o, lse = call()
        _check(o, lse, q, qr, c, lens, 0.1, None, left, 0)
    for _ in range(5):
        for got, want in zip(call(), (o, lse)):
            assert ((got == want) | (got.isnan() & want.isnan())).all()


# one to four blocks of 16 rows, and two work items of 48
@pytest.mark.parametrize("H", [5, 10, 16, 21, 30])
@pytest.mark.parametrize("part", ["latent", "rotary"])
@pytest.mark.parametrize("left", [-1, 40])
def test_some_queries_see_them(H, part, left):
    _run(512, 64, H, 3, part, left)


@pytest.mark.parametrize("L,R", [(256, 32), (128, 64), (128, 32), (256, 64), (512, 32)])
@pytest.mark.parametrize("part", ["latent", "rotary"])
def test_other_lengths(L, R, part):
    _run(L, R, 16, 3, part, -1)
    _run(L, R, 4, 4, part, 70)
