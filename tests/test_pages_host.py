"""The host side of a cache kept in pages without a GPU: TransformerRuntime's calls (tests/cpp/pages_host_cpu); and with a HIP
runtime that runs nothing, the library's workspaces, launches and empty calls."""
import os
import re
import subprocess

import pytest

torch = pytest.importorskip("torch")

import mako_attn as M  # noqa: E402
from conftest import ROOT  # noqa: E402
from test_cache_host import F, I, X, space  # noqa: E402
from test_host_paths import events, hip, launches, tensor  # noqa: E402, F401


def test_cpp_host_side():
    path = os.path.join(ROOT, "tests", "cpp", "bin", "pages_host_cpu")
    assert os.path.exists(path), f"{path} is not built (build() makes it)"
    r = subprocess.run([path], capture_output=True, text=True, timeout=120)
    print(r.stdout)
    assert r.returncode == 0 and "all passed" in r.stdout, r.stdout + r.stderr


S = 0x71000
PAGES = dict(batch=70, pages=5000, page=64, max_pages=80, rows=70, kv_heads=8, dim=128, layers=2)
PAGED = dict(batch=3, rows=200, heads=32, kv_heads=8, dim=128, pages=5000, page=64, max_pages=200, max_new=150, max_ctx=9000)


def attn(a, ws):
    M.attn_paged(a, X, X, X, I, I, X, ws, starts=I, lse=F, stream=S)


def reserve(a, ws):
    M.pages_reserve(a, X, X, I, I, I, I, I, I, ws, starts=I, stream=S)


def fork(a, ws):
    M.pages_fork(a, I, I, I, I, I, I, ws, parent=I, keep=I, stream=S)


def compact(a, ws):
    M.pages_compact(a, X, X, I, I, I, I, I, ws, map_out=I, stream=S)


CALLS = {
    "attn": (attn, M.attn_paged_workspace, M.paged_args(**PAGED), ["paged_rows", "paged_merge"]),
    "attn_256": (attn, M.attn_paged_workspace, M.paged_args(**dict(PAGED, dim=256, heads=16)), ["paged_rows", "paged_merge"]),
    "reserve": (reserve, M.pages_reserve_workspace, M.pages_args(**PAGES), None),
    "fork": (fork, M.pages_fork_workspace, M.pages_args(**PAGES), None),
    "compact": (compact, M.pages_compact_workspace, M.pages_args(**PAGES), None),
}


@pytest.mark.parametrize("name", CALLS)
def test_workspaces(hip, name):  # noqa: F811
    """The bytes that the query names are enough and all are needed; the library allocates nothing of its own, and what it
    launches is kernels on the caller's stream."""
    call, query, a, kernels = CALLS[name]
    need = query(a)
    assert need > 0
    for ws in (None, space(need - 1), space(need, 0x200008), space(0)):
        with pytest.raises(M.MakoError, match="workspace"):
            call(a, ws)
    assert launches(hip) == []
    call(a, space(need))
    got = launches(hip)
    if kernels:
        assert len(got) == len(kernels) and all(k in x for k, x in zip(kernels, got)), got
    assert got and len(got) == len(events(hip)), events(hip)


def test_calls_that_need_no_workspace(hip):  # noqa: F811
    """Short contexts' attention is one launch; forks into other arrays and writes take none."""
    a = M.paged_args(**dict(PAGED, max_ctx=700, max_new=1, rows=3, batch=3))
    assert M.attn_paged_workspace(a) == 0
    attn(a, None)
    assert len(launches(hip)) == 1 and "paged_rows" in launches(hip)[0]
    J = tensor(torch.int32, 0x300000)
    p = M.pages_args(**PAGES)
    M.pages_fork(p, I, I, I, J, J, J, None, parent=I, stream=S)
    M.pages_write(p, X, X, X, X, I, I, stream=S)
    assert events(hip, "alloc", "free") == []


def test_empty_calls_launch_nothing(hip):  # noqa: F811
    for kw in (dict(batch=0), dict(max_new=0), dict(max_ctx=0)):
        a = M.paged_args(**dict(PAGED, **kw))
        assert M.attn_paged_workspace(a) == 0 or not kw.get("max_ctx", 1)
        attn(a, None)
    for kw in (dict(batch=0), dict(rows=0), dict(kv_heads=0)):
        if "kv_heads" not in kw:
            M.pages_write(M.pages_args(**dict(PAGES, **kw)), X, X, X, X, I, I, starts=I, stream=S)
    assert launches(hip) == []


@pytest.mark.parametrize("dim", [64, 128, 256])
@pytest.mark.parametrize("heads,kv", [(1, 1), (32, 8), (32, 4), (48, 2), (24, 8), (64, 1)])
def test_ranges_fill_the_chip_once(hip, dim, heads, kv):  # noqa: F811
    """One workgroup a CU at most (unless the column blocks are more than that), grouped by XCD, whatever the batch; with short
    contexts and few rows, a workgroup for each sequence, kv head and column block."""
    group = heads // kv
    hq = next(h for h in (8, 4, 2, 1) if group % h == 0)
    ncb = group // hq
    for batch, max_new, max_ctx in ((1, 1, 100), (1, 1, 100000), (64, 1, 4000), (3, 500, 9000), (300, 7, 500)):
        rows = batch * max_new
        a = M.paged_args(batch=batch, rows=rows, heads=heads, kv_heads=kv, dim=dim, pages=5000, page=64, max_pages=2000,
                         max_new=max_new, max_ctx=max_ctx)
        hip.fake_clear()
        attn(a, space(max(16, M.attn_paged_workspace(a))))
        grid = events(hip, "launch")[0][2]
        x, y, z = (int(i) for i in re.findall(r"\d+", grid)[:3])
        assert y == ncb and ncb <= x * y * z <= max(256, ncb)
        if max_ctx == 100 and kv * ncb <= 248:
            assert (x, z) == (kv, batch)
        else:
            assert x in (1, 8) and x * y * z > 256 - 8 * ncb
