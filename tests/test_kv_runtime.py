"""The key/value cache's host side (hale-token_amd/csrc/kv.hip) on the CPU: its
host pass, built with AddressSanitizer and UndefinedBehaviorSanitizer over a
HIP runtime in host memory (tests/native/kv_fake_hip.h)."""
import os
import shutil
import subprocess

import pytest

HERE = os.path.dirname(os.path.abspath(__file__))
CSRC = os.path.join(os.path.dirname(HERE), "hale-token_amd", "csrc")
NATIVE = os.path.join(HERE, "native")
SAN = ["-fsanitize=address,undefined", "-fno-sanitize-recover=all"]
HOST_SAN = [x for flag in SAN for x in ("-Xarch_host", flag)]


@pytest.fixture(scope="module")
def check(tmp_path_factory):
    hipcc = os.environ.get("HIPCC", "/opt/rocm/bin/hipcc")
    clang = "/opt/rocm/lib/llvm/bin/clang++"
    if not (os.path.exists(hipcc) or shutil.which("hipcc")) or not os.path.exists(clang):
        pytest.skip("no hipcc to compile the host side with")
    tmp = tmp_path_factory.mktemp("kv_runtime")
    objs = []
    for src in (os.path.join(CSRC, "kv.hip"), os.path.join(NATIVE, "kv_runtime_check.cpp")):
        objs.append(str(tmp / (os.path.basename(src) + ".o")))
        subprocess.run([hipcc, "-x", "hip", "--cuda-host-only", "-std=c++17", "-O1", "-g", *HOST_SAN, "-I", CSRC, "-c", src,
                        "-o", objs[-1]], check=True)
    exe = str(tmp / "kv_runtime_check")
    subprocess.run([clang, "-std=c++17", "-O1", "-g", *SAN, "-I", CSRC, *objs,
                    *(os.path.join(CSRC, f) for f in ("kv_pages.cpp", "rope_freq.cpp")), "-o", exe], check=True)

    def run(what):
        r = subprocess.run([exe, what], capture_output=True, text=True, timeout=120)
        assert r.returncode == 0, r.stderr[-3000:]

    return run


def test_every_list_of_every_view_in_one_step(check):
    check("every_view")


def test_a_plan_that_was_outgrown_stays_while_graphs_exist(check):
    check("plan_behind_a_graph")


def test_a_captured_rotation_of_positions_that_moved_is_refused(check):
    check("rotation_in_a_graph")


def test_a_step_that_finds_no_memory_changes_nothing(check):
    check("step_without_memory")


def test_a_copy_that_finds_no_memory_makes_no_sequence(check):
    check("copy_without_memory")


def test_a_compaction_that_finds_no_memory_moves_nothing(check):
    check("compact_without_memory")


def test_other_calls_that_find_no_memory_change_nothing(check):
    check("others_without_memory")


def test_a_graph_of_a_cache_is_not_launched_inside_a_capture(check):
    check("launch_in_a_capture")


def test_reads_of_any_length_fit_their_launches(check):
    check("long_reads")
