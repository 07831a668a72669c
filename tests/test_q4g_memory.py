"""The device memory of 4-bit matrices on the CPU (tests/native/q4g_memory_check.cpp): the host pass of
hale-token_amd/csrc/step_ops.hip, built with AddressSanitizer and UndefinedBehaviorSanitizer over a
HIP runtime in host memory."""
import os
import shutil
import subprocess

import pytest

from test_kv_runtime import CSRC, HOST_SAN, NATIVE, SAN


def test_matrices_hold_little_more_than_their_bytes(tmp_path):
    hipcc = os.environ.get("HIPCC", "/opt/rocm/bin/hipcc")
    clang = "/opt/rocm/lib/llvm/bin/clang++"
    if not (os.path.exists(hipcc) or shutil.which("hipcc")) or not os.path.exists(clang):
        pytest.skip("no hipcc to compile the host side with")
    objs = []
    for src in (os.path.join(CSRC, "step_ops.hip"), os.path.join(NATIVE, "q4g_memory_check.cpp")):
        objs.append(str(tmp_path / (os.path.basename(src) + ".o")))
        subprocess.run([hipcc, "-x", "hip", "--cuda-host-only", "-std=c++17", "-O1", "-g", *HOST_SAN, "-I", CSRC, "-c", src,
                        "-o", objs[-1]], check=True)
    exe = str(tmp_path / "q4g_memory_check")
    subprocess.run([clang, "-std=c++17", "-O1", "-g", *SAN, *objs, "-o", exe], check=True)
    r = subprocess.run([exe], capture_output=True, text=True, timeout=120)
    assert r.returncode == 0, r.stderr[-3000:]
