"""Decode calls at the ends of the sizes that the C ABI takes (CPU: argument checks and the plan; nothing is launched)."""
import ctypes

import pytest

from pallas_flexattn import _lib
from tests.test_cache_refusals import _decode_cache, _decode_params


def _plan(**kw):
    """(what the call returns without a query tensor: nothing is launched, bytes of workspace)"""
    p, c = _decode_params(Skv=1 << 12, **kw), _decode_cache(max_pages=1 << 6)
    lib = _lib.load()
    rc = lib.fa_fwd_kvcache_fp8(ctypes.byref(p), ctypes.byref(c), None, 16, 16, 16, 1 << 40, None)
    return rc, lib.fa_fwd_kvcache_fp8_workspace_bytes(ctypes.byref(p), ctypes.byref(c))


@pytest.mark.parametrize("kw", [dict(B=1, Hq=1, Hkv=1, Sq=(1 << 26) - 3, D=32), dict(B=1, Hq=1, Hkv=1, Sq=1 << 26, D=32),
                                dict(B=1, Hq=4, Hkv=1, Sq=1 << 24, D=64)])
def test_as_many_rows_as_a_launch_has_threads(kw):
    """Joining pieces takes a wave per query row: past 2^26 - 4 rows more threads than a launch can have, so such a call is
    not cut (its items fill the units many times over anyway)."""
    assert _plan(**kw) == (-1, 0)


def test_fewer_rows_are_cut():
    rc, need = _plan(B=1, Hq=1, Hkv=1, Sq=(1 << 26) - 4, D=32)
    assert rc == -1 and need > 0


def _native(name, tmp_path):
    import os
    import shutil
    import subprocess
    cxx = shutil.which("g++")
    if cxx is None:
        pytest.skip("no C++ compiler")
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    exe = tmp_path / "check"
    subprocess.run([cxx, "-std=c++17", "-O1", "-g", "-fsanitize=address,undefined", "-fno-sanitize-recover=all",
                    "-I" + os.path.join(root, "pallas-flexattn_amd", "csrc"),
                    os.path.join(root, "tests", "native", name), "-o", str(exe)], check=True)
    out = subprocess.run([str(exe)], capture_output=True, text=True)
    assert out.returncode == 0, out.stderr
    return out.stdout


def test_windows_at_the_ends_of_32_bits(tmp_path):
    assert _native("decode_window_check.cpp", tmp_path).startswith("ok 80")
