"""Which workgroup of latent attention takes which block of rows (CPU: the host-and-device arithmetic, with sanitizers)."""
from tests.test_decode_limits import _native


def test_every_block_once_and_no_xcd_left_idle(tmp_path):
    assert _native("latent_plan_check.cpp", tmp_path).strip() == "ok"
