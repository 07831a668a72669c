"""The host side of norms that hand on 8 bits, 4-bit products and logit rules
(hale-token_amd/csrc/step_ops.hip) on the CPU: its host pass, built with
AddressSanitizer and UndefinedBehaviorSanitizer over a HIP runtime in host
memory; and the kernels' resources."""
import os
import shutil
import subprocess

import pytest

from test_kernel_resources import PKG, parse
from test_kv_runtime import CSRC, HOST_SAN, NATIVE, SAN

UNITS = ["kernels_norm_q8", "kernels_q4g", "kernels_logits"]


@pytest.fixture(scope="module")
def check(tmp_path_factory):
    hipcc = os.environ.get("HIPCC", "/opt/rocm/bin/hipcc")
    clang = "/opt/rocm/lib/llvm/bin/clang++"
    if not (os.path.exists(hipcc) or shutil.which("hipcc")) or not os.path.exists(clang):
        pytest.skip("no hipcc to compile the host side with")
    tmp = tmp_path_factory.mktemp("step_ops")
    objs = []
    for src in (os.path.join(CSRC, "step_ops.hip"), os.path.join(NATIVE, "step_ops_check.cpp")):
        objs.append(str(tmp / (os.path.basename(src) + ".o")))
        subprocess.run([hipcc, "-x", "hip", "--cuda-host-only", "-std=c++17", "-O1", "-g", *HOST_SAN, "-I", CSRC, "-c", src,
                        "-o", objs[-1]], check=True)
    exe = str(tmp / "step_ops_check")
    subprocess.run([clang, "-std=c++17", "-O1", "-g", *SAN, *objs, "-o", exe], check=True)

    def run(what):
        r = subprocess.run([exe, what], capture_output=True, text=True, timeout=120)
        assert r.returncode == 0, r.stderr[-3000:]

    return run


def test_arguments_of_the_norm(check):
    check("norm_arguments")


def test_matrices_and_the_arguments_of_their_products(check):
    check("matrices")


def test_arguments_of_the_rules_on_logits(check):
    check("logit_arguments")


def test_no_kernel_uses_scratch():
    hipcc = os.environ.get("HIPCC", "/opt/rocm/bin/hipcc")
    if not (os.path.exists(hipcc) or shutil.which("hipcc")) or not shutil.which("make"):
        pytest.skip("no hipcc to compile the kernels with")
    p = subprocess.run(["make", "-C", PKG, "-j4", "resources"], capture_output=True, text=True, timeout=900)
    assert p.returncode == 0, p.stderr[-3000:]
    report = {u: parse(open(os.path.join(PKG, "_build", u + ".res")).read()) for u in UNITS}
    names = [k for u in UNITS for k in report[u]]
    for kernel in ("k_norm_q8", "k_q4g_pack", "k_q4g_unpack", "k_q4g_few", "k_logits"):
        assert any(kernel in n for n in names), kernel
    bad = [(u, k) for u in UNITS for k, r in report[u].items()
           if int(r.get("ScratchSize [bytes/lane]", "0")) or r.get("Dynamic Stack") == "True"]
    assert not bad, bad
