"""The rotary and key/value cache kernels use no scratch memory (nothing is
spilled), from the compiler's own resource report; see
test_kernel_resources.py for how it is made."""
import os
import shutil
import subprocess

import pytest

from test_kernel_resources import PKG, parse

UNITS = ["kernels_kv", "kernels_kv_attn"]


@pytest.fixture(scope="module")
def report():
    hipcc = os.environ.get("HIPCC", "/opt/rocm/bin/hipcc")
    if not (os.path.exists(hipcc) or shutil.which("hipcc")) or not shutil.which("make"):
        pytest.skip("no hipcc to compile the kernels with")
    p = subprocess.run(["make", "-C", PKG, "-j4", "resources"], capture_output=True, text=True, timeout=900)
    assert p.returncode == 0, p.stderr[-3000:]
    return {u: parse(open(os.path.join(PKG, "_build", u + ".res")).read()) for u in UNITS}


def test_every_kernel_is_reported(report):
    names = [k for u in UNITS for k in report[u]]
    for kernel in ("k_rope", "k_kv_upload", "k_kv_append", "k_kv_read", "k_kv_attend", "k_kv_join"):
        assert any(kernel in n for n in names), kernel


def test_no_kernel_uses_scratch(report):
    bad = [(u, k) for u in UNITS for k, r in report[u].items()
           if int(r.get("ScratchSize [bytes/lane]", "0")) or r.get("Dynamic Stack") == "True"]
    assert not bad, bad
