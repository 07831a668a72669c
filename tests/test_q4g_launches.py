"""The launches of the 4-bit products on the CPU (tests/native/q4g_launch_check.cpp): the host pass of
hale-token_amd/csrc/kernels_q4g.hip over a HIP runtime that only notes them."""
import os
import shutil
import subprocess

import pytest

from test_kv_runtime import CSRC, HOST_SAN, NATIVE, SAN


def test_launches_keep_to_limits_that_no_other_call_changes(tmp_path):
    hipcc = os.environ.get("HIPCC", "/opt/rocm/bin/hipcc")
    clang = "/opt/rocm/lib/llvm/bin/clang++"
    if not (os.path.exists(hipcc) or shutil.which("hipcc")) or not os.path.exists(clang) or not shutil.which("nm"):
        pytest.skip("no hipcc to compile the host side with")
    objs = []
    for src in (os.path.join(CSRC, "kernels_q4g.hip"), os.path.join(NATIVE, "q4g_launch_check.cpp")):
        objs.append(str(tmp_path / (os.path.basename(src) + ".o")))
        subprocess.run([hipcc, "-x", "hip", "--cuda-host-only", "-std=c++17", "-O1", "-g", *HOST_SAN, "-I", CSRC, "-c", src,
                        "-o", objs[-1]], check=True)
    exe = str(tmp_path / "q4g_launch_check")
    # the device code, which a host pass has not: a name of the object's own
    nm = subprocess.run(["nm", "-u", objs[0]], check=True, capture_output=True, text=True)
    absent = [f"-Wl,--defsym={n}=no_device_code" for n in nm.stdout.split() if n.startswith("__hip_fatbin")]
    subprocess.run([clang, "-std=c++17", "-O1", "-g", *SAN, *objs, *absent, "-o", exe], check=True)
    r = subprocess.run([exe], capture_output=True, text=True, timeout=120)
    assert r.returncode == 0, r.stderr[-3000:]
