"""flex_decode_latent with many blocks of 64 rows: short prompts, whose blocks go over all XCDs (csrc/latent_plan.h)."""
import pytest

pytestmark = pytest.mark.gpu

from tests.test_gpu_latent import test_decode as decode  # noqa: E402


@pytest.mark.parametrize("case", [
    # keys (the queries' included), H, T, L, R, page, mask: 9 blocks and more, in one piece of keys, in several and whole; 8 blocks
    ([700], 16, 36, 128, 32, 32, (-1, 0)), ([300], 16, 130, 128, 64, 64, (-1, 0)), ([90, 200, 64], 16, 64, 256, 32, 32, (-1, 0)),
    ([900, 130, 40], 30, 30, 128, 32, 64, (-1, 0)), ([400] * 9, 32, 24, 128, 32, 64, (200, 0)), ([1200, 60], 64, 8, 512, 64, 64, (-1, 0)),
    ([260], 128, 20, 512, 64, 128, (-1, 0)),
], ids=range(7))
def test_many_blocks(case):
    decode(case)
