"""The student operators through the C++20 host layer (tinytensor_amd/host/tt_amd.h): tests/cpp/test_student_amd.cpp, a plain
g++ program over the C ABI, built by __graft_entry__.build() (or on demand here) and run on a GPU."""
import os
import subprocess

import pytest

CPP = os.path.join(os.path.dirname(os.path.abspath(__file__)), "cpp")
BINARY = os.path.join(CPP, "test_student_amd")


def ensure_built():
    if not os.path.exists(BINARY):
        subprocess.run(["make", "-C", CPP, "test_student_amd"], check=True, capture_output=True)


def test_program_builds_and_lists():
    ensure_built()
    out = subprocess.run([BINARY, "--list"], check=True, capture_output=True, text=True).stdout
    assert len(out.strip().splitlines()) == 3


@pytest.mark.gpu
def test_student_operators_through_the_cpp_host_layer():
    ensure_built()
    proc = subprocess.run([BINARY], capture_output=True, text=True, timeout=110)
    print(proc.stdout[-3000:], proc.stderr[-2000:])
    assert proc.returncode == 0, proc.stdout[-3000:]
    assert "0 failure(s)" in proc.stdout
