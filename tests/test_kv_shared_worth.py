"""Plans of steps whose sequences share pages read no more of them than plans of each sequence by
itself (tests/native/kv_shared_worth_check.cpp), built with AddressSanitizer and
UndefinedBehaviorSanitizer."""
import os
import shutil
import subprocess

import pytest

from test_kv_runtime import CSRC, NATIVE, SAN


@pytest.fixture(scope="module")
def check(tmp_path_factory):
    cxx = shutil.which("g++")
    if not cxx:
        pytest.skip("no C++ compiler")
    exe = str(tmp_path_factory.mktemp("kv_worth") / "kv_shared_worth_check")
    subprocess.run([cxx, "-std=c++17", "-O1", "-g", "-Wall", "-Wextra", *SAN, "-I", CSRC, os.path.join(NATIVE, "kv_shared_worth_check.cpp"),
                    os.path.join(CSRC, "kv_pages.cpp"), "-o", exe], check=True)

    def run(what):
        r = subprocess.run([exe, what], capture_output=True, text=True, timeout=300)
        assert r.returncode == 0, r.stderr[-3000:]

    return run


def test_sharing_reads_no_more_pages(check):
    check("no_more_pages")


def test_sequences_of_many_rows(check):
    check("many_rows")


def test_plans_that_share_nothing_say_so(check):
    check("nothing_shared")


def test_as_much_is_shared_as_there_is_room_for(check):
    check("as_much_as_there_is_room_for")


def test_steps_whose_many_rows_come_from_sharing(check):
    check("many_rows_by_sharing")


def test_steps_of_short_sequences_stay_apart(check):
    check("short_steps")


def test_rows_of_many_parts(check):
    check("many_parts")
