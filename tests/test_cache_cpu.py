"""Without a GPU: the cache's row kernels run on the CPU (tests/cpp/cache_rows_cpu.cpp), where no index leaves its arrays and
every list ends as a sort on the host says, at list lengths and budgets around the blocks that the kernels take a long list
in; what TransformerRuntime's cache calls pass on (tests/cpp/cache_host_cpu.cpp); and which sizes are refused before any
launch, with a HIP runtime that records launches and runs nothing."""
import os
import subprocess

import pytest

pytest.importorskip("torch")

import mako_attn as M  # noqa: E402
from conftest import ROOT  # noqa: E402
from test_cache_host import F, I, X, evict_call, space, tree_call, weights_call  # noqa: E402
from test_host_paths import hip, launches  # noqa: E402, F401

CPP = os.path.join(ROOT, "tests", "cpp")


@pytest.mark.parametrize("name", ["cache_rows_cpu", "cache_host_cpu"])
def test_on_the_cpu(name):
    subprocess.run(["make", "-s", "-C", CPP, f"bin/{name}"], check=True)
    r = subprocess.run([os.path.join(CPP, "bin", name)], capture_output=True, text=True, timeout=600)
    assert r.returncode == 0 and "all passed" in r.stdout, r.stdout + r.stderr


def append_call(a, ws):
    M.cache_append(a, X, X, X, X, I, I, stream=0x71000)


# calls with a launch of 2^32 threads (which HIP refuses) and the largest of the same kind below
GRIDS = {
    "evict": (evict_call, M.cache_evict_workspace,
              lambda n: M.evict_args(batch=n, kv_heads=8, dim=64, cap=2, max_ctx=2, budget=1), 1 << 20),
    "evict, long": (evict_call, M.cache_evict_workspace,
                    lambda n: M.evict_args(batch=n, kv_heads=8, dim=64, cap=5000, max_ctx=5000, budget=5000), 1 << 19),
    "evict, move": (evict_call, M.cache_evict_workspace,
                    lambda n: M.evict_args(batch=n, kv_heads=8, dim=64, cap=4096, max_ctx=4096, budget=2048), 1 << 14),
    "append": (append_call, lambda a: 0,
               lambda n: M.append_args(batch=n, n_draft=1, kv_heads=1, dim=64, cap=2), 1 << 22),
    "weights": (weights_call, M.cache_weights_workspace,
                lambda n: M.weights_args(batch=n, n_q=65, heads=8, kv_heads=8, dim=64, cap=2, max_ctx=2), 1 << 21),
    "tree": (tree_call, lambda a: 0,
             lambda n: M.tree_args(batch=n, n_draft=64, heads=64, kv_heads=1, dim=64, cap=2, max_ctx=2), 1 << 18),
    "tree, split": (tree_call, M.attn_tree_workspace,
                    lambda n: M.tree_args(batch=n, n_draft=64, heads=64, kv_heads=1, dim=64, cap=9000, max_ctx=9000), 1 << 14),
}


@pytest.mark.parametrize("name", GRIDS)
def test_launches_past_the_grid_are_refused_before_any(hip, name):  # noqa: F811
    call, query, args, over = GRIDS[name]
    with pytest.raises(M.MakoError, match="exceed the grid"):
        call(args(over), space(query(args(over))))
    assert launches(hip) == []
    a = args(over - 8)
    call(a, space(query(a)))
    assert launches(hip) != []
