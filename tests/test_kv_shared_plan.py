"""Plans of steps whose sequences share pages (tests/native/kv_shared_check.cpp),
built with AddressSanitizer and UndefinedBehaviorSanitizer; and the setting's host
side."""
import os
import shutil
import subprocess

import pytest

from test_kv_runtime import CSRC, NATIVE, SAN


def test_shared_pages_are_read_once_and_joined(tmp_path):
    cxx = shutil.which("g++")
    if not cxx:
        pytest.skip("no C++ compiler")
    exe = str(tmp_path / "kv_shared_check")
    subprocess.run([cxx, "-std=c++17", "-O1", "-g", "-Wall", "-Wextra", *SAN, "-I", CSRC, os.path.join(NATIVE, "kv_shared_check.cpp"),
                    os.path.join(CSRC, "kv_pages.cpp"), "-o", exe], check=True)
    r = subprocess.run([exe], capture_output=True, text=True, timeout=300)
    assert r.returncode == 0, r.stderr[-3000:]
