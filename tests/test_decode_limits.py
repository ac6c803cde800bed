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


def _native(name, tmp_path, *args):
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
    out = subprocess.run([str(exe), *map(str, args)], capture_output=True, text=True)
    assert out.returncode == 0, out.stderr
    return out.stdout


def test_windows_at_the_ends_of_32_bits(tmp_path):
    assert _native("decode_window_check.cpp", tmp_path).startswith("ok 80")


def test_blocks_of_the_gpu_tests_cases(tmp_path):
    """The cases of test_gpu_decode_blocks take the blocks of rows per item that they are there for (where items are cut in
    pieces, the workspace shows it there as well)."""
    from tests.test_gpu_decode_blocks import CASES
    args, want = [], []
    for lens, Hq, Hkv, Sq, D, tiles, win, mods, nq, pieces, stream in CASES:
        left = -1 if win is None else win[0]
        walk = tiles if left < 0 else min(tiles, (left + Sq + 30) // 32 + 1)
        args += [Hq // Hkv * Sq, len(lens) * Hkv, walk]
        want.append(nq)
        assert stream == (2 * len(lens) * Hkv * walk * 32 * D > 112 << 20)
        assert pieces == (walk > 48 and (len(lens) * Hkv < 256 or walk > 128))
    assert [int(x) for x in _native("decode_plan.cpp", tmp_path, *args).split()] == want
    assert {(c[4], bool(c[7] or c[6]), c[9]) for c in CASES if c[8] == 2} == {(D, g, p) for D in (32, 64, 128) for g in (False, True)
                                                                            for p in (False, True)}


def test_every_workgroup_finds_its_work(tmp_path):
    assert _native("decode_unit_check.cpp", tmp_path).startswith("ok 1500 ")
