"""The cache's row kernels run on the CPU (tests/cpp/cache_rows_cpu.cpp): no index leaves its arrays and every list ends as a
sort on the host says, at list lengths and budgets around the blocks that the kernels take a long list in."""
import os
import subprocess

from conftest import ROOT

CPP = os.path.join(ROOT, "tests", "cpp")


def test_rows_kernels_on_the_cpu():
    subprocess.run(["make", "-s", "-C", CPP, "bin/cache_rows_cpu"], check=True)
    r = subprocess.run([os.path.join(CPP, "bin", "cache_rows_cpu")], capture_output=True, text=True, timeout=600)
    assert r.returncode == 0 and "all passed" in r.stdout, r.stdout + r.stderr
