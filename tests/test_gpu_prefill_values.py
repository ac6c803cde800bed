"""flex_prefill over e4m3 values that their scale takes past bf16: infinite, as in a tile that every query sees, for the queries
that see their key, and for no others."""
import numpy as np
import pytest

pytestmark = pytest.mark.gpu

from tests.test_gpu_decode_fp8 import Cache  # noqa: E402
from tests.test_gpu_prefill import _check, _q  # noqa: E402


@pytest.mark.parametrize("T", [3, 90])  # items of at most 32 rows, and larger ones
@pytest.mark.parametrize("D", [32, 64, 128])
@pytest.mark.parametrize("left", [-1, 120])
def test_codes_past_bf16(T, D, left):
    import torch
    import pallas_flexattn as pf
    lens, page = [400, 260, 330], 32
    c = Cache(lens, 2, page, D, 13)
    q = _q(3, 4, T, D, 14)
    codes, scales = c.cache.value.view(torch.uint8), c.cache.value_scale

    def put(b, h, key, d, code):  # the key's run: zeros but for what is put
        at = int(c.table[b, key // page]), h
        if float(scales[at]) != 2.0 ** 125:
            scales[at] = 2.0 ** 125
            codes[at] = 0
            c.rows[1][b, h, key // page * page:(key // page + 1) * page] = 0
        codes[at[0], h, key % page, d] = code
        x = float(torch.tensor([code], dtype=torch.uint8).view(torch.float8_e4m3fn).float()) * 2.0 ** 125
        c.rows[1][b, h, key, d] = x if x != x or abs(x) < 3.39e38 else np.copysign(np.inf, x)

    put(0, 0, 399, 3, 0x7e)   # 448 2^125: the last query alone
    put(0, 0, 398, 5, 0xfe)
    put(0, 1, 398, D - 1, 0x08)   # 2^119 is finite, in sums too
    put(0, 1, 399, D - 1, 0x7f)   # NaN all the same
    put(1, 0, 258, 9, 0x50)   # 8 2^125, just past bf16
    put(1, 0, 259, 9, 0xd0)   # both: NaN for the last, an infinity for the one before
    put(1, 1, 257, 0, 0x01)   # 2^116
    put(2, 0, 330 - T - left if left >= 0 else 328, 7, 0x7e)  # behind a window: the first query alone
    with np.errstate(invalid="ignore"):
        o, lse = pf.flex_prefill(q, c.cache, c.lens, c.table, mask_mod=pf.MaskSpec(left=left, right=0), enable_gqa=True, return_lse=True)
        _check(o, lse, q, c, lens, None, left, 0)
