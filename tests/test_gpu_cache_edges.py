"""The cache operators where their kernels change course: lists of several blocks, budgets at a block's end; the bits that
f16 output keeps; cached values that are not finite; the append of a prompt; and a prompt's padded tiles through the C++ host side (tests/cpp/cache_prompt_test)."""
import os
import subprocess

import numpy as np
import pytest

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

import cache_ref as R  # noqa: E402
import mako_attn as M  # noqa: E402
from conftest import ROOT  # noqa: E402
import test_gpu_cache as T  # noqa: E402
from test_gpu_cache import BF16, F16, F32, as_i64, gen, i32, randn, random_masks  # noqa: E402

GUARD = 1 << 18  # bytes on either side of a workspace


@pytest.fixture
def guarded(monkeypatch):
    """Workspaces between guard bytes, which are as they were when the test ends."""
    made = []

    def buffer(n):
        whole = torch.full((max(n, 16) + 2 * GUARD,), 0xA5, dtype=torch.uint8, device="cuda")
        made.append((whole, max(n, 16)))
        return whole[GUARD:GUARD + max(n, 16)]

    monkeypatch.setattr(T, "buffer", buffer)
    yield
    torch.cuda.synchronize()
    assert made
    for whole, n in made:
        assert torch.all(whole[:GUARD] == 0xA5) and torch.all(whole[GUARD + n:] == 0xA5), "a byte outside a workspace changed"


def few_values(w, rng):
    w[:] = rng.integers(0, 700, w.shape)


LONG = [
    dict(ctx=[40000], budget=32767),
    dict(ctx=[40000], budget=32768),
    dict(ctx=[40000, 36000], budget=32769, recent=300, sinks=4, moved=True),
    dict(ctx=[33000, 40000], budget=33000, recent=100),
    dict(ctx=[40000], budget=33000, weigh=few_values),
    dict(ctx=[70001], budget=40000, sinks=2),
    dict(ctx=[70001, 9], budget=65536, moved=True),
    dict(ctx=[100000], budget=70000, recent=1000, max_ctx=98000),
]


@pytest.mark.parametrize("case", LONG, ids=lambda c: f"n{max(c['ctx'])}to{c['budget']}")
@pytest.mark.parametrize("in_place", [False, True])
def test_evict_lists_of_several_blocks(guarded, case, in_place):
    """Distinct weights, so that the selection ends without a tie, and the budget past the first block's rows."""
    T.run_evict(dt=F16 if in_place else BF16, dim=64, kv=2, seed=70, in_place=in_place,
                **dict(dict(weigh=lambda w, rng: w.__setitem__(..., rng.permutation(w.size).reshape(w.shape))), **case))


@pytest.mark.parametrize("dim,heads,kv,ctx,n", [(64, 4, 2, [40, 3], 7), (128, 8, 2, [30, 12], 6), (128, 8, 1, [60, 20], 20),
                                               (128, 4, 2, [9000, 5000], 16), (256, 8, 2, [33, 31], 9),
                                               (256, 4, 1, [6000], 40)])
def test_tree_f16_output_is_rounded_once(dim, heads, kv, ctx, n):
    """f16 tiles and f16 output: what the output's own rounding (2^-11 of the value, 2^-25 below f16's normal range) does not
    explain is within the bound of f32 output, that is, the probabilities hold twice f16's bits: where p and v cancel, one
    f16 value of p would show."""
    B, cap, g, rng = len(ctx), max(ctx) + 3, gen(80), np.random.default_rng(80)
    q = randn(g, (heads, B * n, dim), F16, 2.0 ** -4)  # (small scores, so that their own bound is small)
    k, v = (randn(g, (B, kv, cap, dim), F16) for _ in range(2))
    kd, vd = (randn(g, (kv, B * n, dim), F16) for _ in range(2))
    m = random_masks(rng, B, n)
    a = M.tree_args(batch=B, n_draft=n, heads=heads, kv_heads=kv, dim=dim, cap=cap, max_ctx=cap)
    o = torch.zeros((B * n, heads * dim), dtype=F16, device="cuda")
    M.attn_tree(a, q, k, v, kd, vd, i32(ctx), o, T.buffer(M.attn_tree_workspace(a)), mask=as_i64(m))
    torch.cuda.synchronize()
    want, _, tol, _ = R.tree(*[R.f64(t) for t in (q, k, v, kd, vd)], ctx, [n] * B, m, n=n, scale=a.scale, out=F32,
                             in_dtype=F16)
    T.check(o, want, tol + 2.0 ** -11 * np.abs(want) + 2.0 ** -25, "o")


def test_cpp_prompt_of_padded_tiles():
    path = os.path.join(ROOT, "tests", "cpp", "bin", "cache_prompt_test")
    assert os.path.exists(path), f"{path} is not built (build() makes it)"
    r = subprocess.run([path], capture_output=True, text=True, timeout=120)
    print(r.stdout)
    assert r.returncode == 0 and "all passed" in r.stdout, r.stdout + r.stderr


@pytest.mark.parametrize("bad", [float("nan"), float("inf"), -float("inf")])
@pytest.mark.parametrize("dt,out,dim,ctx", [(F16, F16, 128, 70), (BF16, F32, 64, 5000), (BF16, BF16, 256, 9000)])
def test_tree_cached_values_that_are_not_finite(dt, out, dim, ctx, bad):
    """Such a value in a row of the cache: its head dim of the rows that see it is not finite, and no other output changes."""
    heads, kv, n, g = 4, 2, 6, gen(90)
    q = randn(g, (heads, 2 * n, dim), dt)
    k, v = (randn(g, (2, kv, ctx, dim), dt) for _ in range(2))
    kd, vd = (randn(g, (kv, 2 * n, dim), dt) for _ in range(2))
    a = M.tree_args(batch=2, n_draft=n, heads=heads, kv_heads=kv, dim=dim, cap=ctx, max_ctx=ctx)
    ws, outs = T.buffer(M.attn_tree_workspace(a)), []
    for step in range(2):
        if step:
            v[1, 1, [3, ctx // 2, ctx - 1], [5, 7, dim - 1]] = bad
        o, lse = torch.zeros((2 * n, heads * dim), dtype=out, device="cuda"), torch.zeros((heads, 2 * n), device="cuda")
        M.attn_tree(a, q, k, v, kd, vd, i32([ctx, ctx]), o, ws, lse=lse)
        torch.cuda.synchronize()
        outs.append((o.view(2, n, heads, dim), lse))
    (o0, l0), (o1, l1) = outs
    hit = torch.zeros_like(o0, dtype=torch.bool)
    hit[1, :, heads // kv:, [5, 7, dim - 1]] = True
    assert not torch.isfinite(o1[hit]).any()
    assert torch.equal(o1[~hit], o0[~hit]) and torch.equal(l1, l0)


@pytest.mark.parametrize("case", [(F16, 128, 8, 4096, [0], [4096], 4100), (BF16, 64, 3, 513, [5, 700, 0], [513, 300, 600], 1000),
                                  (BF16, 256, 1, 2000, [37], [1999], 1500)], ids=lambda c: f"d{c[1]}kv{c[2]}n{c[3]}")
@pytest.mark.parametrize("in_place", [False, True])
def test_append_of_a_prompt(case, in_place):
    """Thousands of rows a sequence, some lists at their cap, tiles with padded heads."""
    T.test_append(case, in_place)
