"""Without a GPU: the cache's row kernels run on the CPU (tests/cpp/cache_rows_cpu.cpp), where no index leaves its arrays and
every list ends as a sort on the host says, at list lengths and budgets around the blocks that the kernels take a long list
in; and what TransformerRuntime's cache calls pass on (tests/cpp/cache_host_cpu.cpp)."""
import os
import subprocess

import pytest

from conftest import ROOT

CPP = os.path.join(ROOT, "tests", "cpp")


@pytest.mark.parametrize("name", ["cache_rows_cpu", "cache_host_cpu"])
def test_on_the_cpu(name):
    subprocess.run(["make", "-s", "-C", CPP, f"bin/{name}"], check=True)
    r = subprocess.run([os.path.join(CPP, "bin", name)], capture_output=True, text=True, timeout=600)
    assert r.returncode == 0 and "all passed" in r.stdout, r.stdout + r.stderr
