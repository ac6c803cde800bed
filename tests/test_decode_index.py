"""The work partition of decode over a paged cache (csrc/decode_index.h), enumerated on the CPU under
AddressSanitizer and UndefinedBehaviorSanitizer (tests/native/decode_index_check.cpp)."""
import os
import shutil
import subprocess

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def test_every_tile_once_and_every_piece_found(tmp_path):
    cxx = shutil.which("g++")
    if cxx is None:
        pytest.skip("no C++ compiler")
    exe = tmp_path / "check"
    subprocess.run([cxx, "-std=c++17", "-O1", "-g", "-fsanitize=address,undefined", "-fno-sanitize-recover=all",
                    "-I" + os.path.join(ROOT, "pallas-flexattn_amd", "csrc"),
                    os.path.join(ROOT, "tests", "native", "decode_index_check.cpp"), "-o", str(exe)], check=True)
    out = subprocess.run([str(exe)], capture_output=True, text=True)
    assert out.returncode == 0, out.stderr
    assert out.stdout.startswith("ok 4000 ")
