"""The key/value cache's page bookkeeping and step plans, and the rotary
frequencies, on the CPU: the host code behind hale_kv_* and hale_rope_*
(hale-token_amd/csrc/kv_pages.cpp, rope_freq.cpp) built with AddressSanitizer and
UndefinedBehaviorSanitizer and run by small native programs, and the refusals
that need no device."""
import math
import os
import subprocess

import numpy as np
import pytest

import hale_moe

HERE = os.path.dirname(os.path.abspath(__file__))
CSRC = os.path.join(os.path.dirname(HERE), "hale-token_amd", "csrc")
SAN = ["-fsanitize=address,undefined", "-fno-sanitize-recover=all", "-fno-omit-frame-pointer", "-g"]


def build(tmp, name, source):
    exe = tmp / name
    subprocess.run(["g++", "-std=c++17", "-O1", *SAN, "-I", CSRC, os.path.join(CSRC, source),
                    os.path.join(HERE, "native", name + ".cpp"), "-o", str(exe)], check=True)
    return exe


def test_pages_and_plans_under_asan_ubsan(tmp_path):
    exe = build(tmp_path, "kv_pages_check", "kv_pages.cpp")
    r = subprocess.run([str(exe)], capture_output=True, text=True, timeout=300)
    assert r.returncode == 0, r.stderr[-2000:]
    ops, refused = map(int, r.stdout.split())
    assert ops == 18000 and refused > 500


@pytest.fixture(scope="module")
def rope(tmp_path_factory):
    exe = build(tmp_path_factory.mktemp("rope"), "rope_freq_check", "rope_freq.cpp")

    def run(layout=0, scaling=0, hd=128, r=128, base=1e4, factor=1.0, original=0.0, low=1.0, high=32.0, att=1.0):
        out = subprocess.run([str(exe), *map(str, (layout, scaling, hd, r, base, factor, original, low, high, att))],
                             capture_output=True, text=True, timeout=60)
        assert out.returncode == 0, out.stderr[-2000:]
        return out.stdout.strip() if out.stdout.startswith("refused") else np.array(list(map(float, out.stdout.split())))

    return run


def test_rope_frequencies(rope):
    i = np.arange(64)
    plain = 1e6 ** (-i / 64.0)
    # pow() is good to an ulp or two of its result; the scalings add three roundings
    tol = 8 * 2.0 ** -53
    assert np.allclose(rope(base=1e6), plain, rtol=tol, atol=0)
    assert np.allclose(rope(base=1e6, scaling=1, factor=4.0), plain / 4, rtol=tol, atol=0)
    ntk = (1e6 * 8.0 ** (128 / 126)) ** (-i / 64.0)
    # the base's error of a few ulps enters with a power of up to 1
    assert np.allclose(rope(base=1e6, scaling=2, factor=8.0), ntk, rtol=4 * tol, atol=0)
    got = rope(base=1e6, scaling=3, factor=8.0, original=8192.0, low=1.0, high=32.0)
    turns = 8192.0 * plain / (2 * math.pi)
    keep = np.clip((turns - 1) / 31, 0, 1)
    assert np.allclose(got, plain * keep + plain / 8 * (1 - keep), rtol=4 * tol, atol=0)
    assert (got[turns >= 32] == rope(base=1e6)[turns >= 32]).all()
    assert np.allclose(got[turns <= 1], plain[turns <= 1] / 8, rtol=tol, atol=0)
    assert rope(hd=128, r=32).size == 16 and rope(hd=2, r=2).size == 1


@pytest.mark.parametrize("bad", [
    dict(layout=2), dict(layout=-1), dict(scaling=4), dict(scaling=-1), dict(hd=0), dict(hd=2000), dict(r=0), dict(r=3),
    dict(r=130), dict(base=1.0), dict(base="inf"), dict(base="nan"), dict(scaling=1, factor=0.5),
    dict(scaling=1, factor="nan"), dict(scaling=2, factor=2.0, r=2), dict(scaling=3, factor=2.0, original=0.0),
    dict(scaling=3, factor=2.0, original=100.0, low=4.0, high=4.0),
    dict(scaling=3, factor=2.0, original=100.0, low=-1.0), dict(att=0.0), dict(att="inf")])
def test_rope_refusals(rope, bad):
    assert isinstance(rope(**bad), str), bad


def test_null_arguments_are_refused_without_a_device():
    L, E = hale_moe.lib(), hale_moe.EINVAL
    assert L.hale_rope_create(None, None, None) == E
    assert L.hale_rope_frequencies(None, None, 0) == E
    assert L.hale_rope_device(None, 0, 1, None, None, 1, 1, None, 1, None, 0, 0, None, 0) == E
    assert L.hale_kv_create(None, 1, 1, 1, 64, 1, 1, 1, None) == E
    assert L.hale_kv_seq_create(None, None) == E
    assert L.hale_kv_seq_free(None, 0) == E
    assert L.hale_kv_seq_fork(None, 0, 1, None) == E
    assert L.hale_kv_seq_copy(None, 0, None) == E
    assert L.hale_kv_seq_truncate(None, 0, 0) == E
    assert L.hale_kv_seq_len(None, 0, None) == E
    assert L.hale_kv_pages(None, None, None) == E
    assert L.hale_kv_compact(None, None) == E
    assert L.hale_kv_resize(None, 1) == E
    assert L.hale_kv_step(None, 0, None, None) == E
    assert L.hale_kv_reserve(None, 1) == E
    assert L.hale_kv_positions(None, None) == E
    assert L.hale_kv_append_device(None, 0, 0, 1, None, 1, None, 1) == E
    assert L.hale_kv_attention_device(None, 0, 0, 1, None, 1, 1.0, 0, None, 1) == E
    assert L.hale_kv_read_device(None, 0, 0, 0, 1, None, None) == E
    L.hale_rope_destroy(None)
    L.hale_kv_destroy(None)
