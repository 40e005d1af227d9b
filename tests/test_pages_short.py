"""Serving from a pool of pages that runs out, without a GPU: csrc/pages.hip's kernels on the CPU (tests/cpp/pages_short_cpu.cpp)."""
import os
import subprocess

from conftest import ROOT

CPP = os.path.join(ROOT, "tests", "cpp")


def test_on_the_cpu():
    subprocess.run(["make", "-s", "-C", CPP, "bin/pages_short_cpu"], check=True)
    r = subprocess.run([os.path.join(CPP, "bin", "pages_short_cpu")], capture_output=True, text=True, timeout=600)
    assert r.returncode == 0 and "all passed" in r.stdout, r.stdout + r.stderr
