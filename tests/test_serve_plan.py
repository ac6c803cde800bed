"""The host-and-device arithmetic of chunks and page plans, built for the CPU with sanitizers."""
from tests.test_decode_limits import _native


def test_partition_and_rows(tmp_path):
    assert _native("serve_plan_check.cpp", tmp_path).strip() == "ok"
