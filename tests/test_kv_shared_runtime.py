"""The host side of attention over shared prefixes (hale-token_amd/csrc/kv.hip) on the CPU: its
host pass, built with AddressSanitizer and UndefinedBehaviorSanitizer over a HIP runtime in host
memory (tests/native/kv_fake_hip.h)."""
import os
import shutil
import subprocess

import pytest

from test_kv_runtime import CSRC, HOST_SAN, NATIVE, SAN


@pytest.fixture(scope="module")
def check(tmp_path_factory):
    hipcc = os.environ.get("HIPCC", "/opt/rocm/bin/hipcc")
    clang = "/opt/rocm/lib/llvm/bin/clang++"
    if not (os.path.exists(hipcc) or shutil.which("hipcc")) or not os.path.exists(clang):
        pytest.skip("no hipcc to compile the host side with")
    tmp = tmp_path_factory.mktemp("kv_shared_runtime")
    objs = []
    for src in (os.path.join(CSRC, "kv.hip"), os.path.join(NATIVE, "kv_shared_runtime_check.cpp")):
        objs.append(str(tmp / (os.path.basename(src) + ".o")))
        subprocess.run([hipcc, "-x", "hip", "--cuda-host-only", "-std=c++17", "-O1", "-g", *HOST_SAN, "-I", CSRC, "-c", src,
                        "-o", objs[-1]], check=True)
    exe = str(tmp / "kv_shared_runtime_check")
    subprocess.run([clang, "-std=c++17", "-O1", "-g", *SAN, "-I", CSRC, *objs,
                    *(os.path.join(CSRC, f) for f in ("kv_pages.cpp", "rope_freq.cpp")), "-o", exe], check=True)

    def run(what):
        r = subprocess.run([exe, what], capture_output=True, text=True, timeout=120)
        assert r.returncode == 0, r.stderr[-3000:]

    return run


def test_a_step_of_one_sequence_is_launched_as_without_sharing(check):
    check("one_sequence")


def test_steps_of_many_rows_launch_nothing_for_few(check):
    check("many_rows")
