"""flex_prefill's packed rows whose starts fall: they count as the highest start before them, and every result is written."""
import numpy as np
import pytest

from tests.test_decode_limits import _native


def test_every_token_in_one_row(tmp_path):
    assert _native("packed_rows_check.cpp", tmp_path).strip() == "ok"


@pytest.mark.gpu
@pytest.mark.parametrize("starts", [[0, 40, 10, 60, 50, 100], [90, 0, 0, 200, 5, 100], [0, 300, -7, 2 ** 31 - 1, 20, 9], [130, 100, 0, 0, 0, 0]],
                         ids=range(4))
@pytest.mark.parametrize("kind", ["bf16", "fp8"])
@pytest.mark.parametrize("times", [1, 20])  # more rows than a wave has lanes
def test_starts_that_fall(starts, kind, times):
    import torch
    import pallas_flexattn as pf
    from tests.test_gpu_prefill import _cache, _q
    B, tokens = 5 * times, 150
    rows = [*starts, *starts[1:] * (times - 1)]
    high = np.maximum.accumulate(np.clip(rows, 0, tokens)).tolist()
    c = _cache(kind, [200 + 7 * (b % 9) for b in range(B)], 2, 32, 64, 5)
    q = _q(1, 4, tokens, 64, 6)

    def call(s):
        torch.full((1, 4, tokens, 64), float("nan"), device="cuda", dtype=torch.bfloat16)  # (what a call leaves out may show)
        return pf.flex_prefill(q, c.cache, c.lens, c.table, mask_mod=pf.causal_mask, enable_gqa=True, return_lse=True,
                               query_starts=torch.tensor(s, device="cuda"))

    for got, want in zip(call(rows), call(high)):
        assert torch.equal(got, want)
    o, lse = call(rows)
    for some in (slice(0, high[0]), slice(high[-1], tokens)):
        assert (o[:, :, some] == 0).all() and torch.isneginf(lse[:, :, some]).all()
