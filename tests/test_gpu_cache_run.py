"""The cache operators together, as a serving loop uses them: drafts from mako_heads, attention over the tree, the append of
the accepted path, its weights, the eviction; eager against a simulation in 64 bits, captured into a graph and replayed, on
two streams at once, over a cache past 32-bit offsets; and through the C++ host side (tests/cpp/cache_test)."""
import os
import subprocess

import numpy as np
import pytest

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

import cache_ref as R  # noqa: E402
import mako_attn as M  # noqa: E402
from conftest import ROOT  # noqa: E402
from test_gpu_cache import as_i64, buffer, check, gen, i32, random_masks, randn  # noqa: E402

F16, BF16, F32 = torch.float16, torch.bfloat16, torch.float32


def test_cpp_host_side():
    path = os.path.join(ROOT, "tests", "cpp", "bin", "cache_test")
    assert os.path.exists(path), f"{path} is not built (build() makes it)"
    r = subprocess.run([path], capture_output=True, text=True, timeout=120)
    print(r.stdout)
    assert r.returncode == 0 and "all passed" in r.stdout, r.stdout + r.stderr


def angles(positions, dim):
    inv = 1e6 ** (-torch.arange(0, dim, 2, dtype=torch.float64) / dim)
    a = torch.as_tensor(positions, dtype=torch.float64)[:, None] * inv
    return torch.stack([a.cos(), a.sin()], -1).float().cuda().contiguous()


def test_serving_loop():
    """Two sequences of other lengths, twenty rounds: tiles from fp32 rows with their norms and rotations (each draft at its
    own position), tree, append, weights, eviction once over the budget. The simulation holds each list's rows, weights and
    positions in 64 bits and takes the same accepted paths; eviction is decided by the device's weights."""
    B, n, heads, kv, D, cap, budget, recent, sinks = 2, 6, 4, 2, 128, 160, 96, 12, 2
    dt, rng, g = BF16, np.random.default_rng(3), gen(3)
    k, v = (randn(g, (B, kv, cap, D), dt) for _ in range(2))
    w, pos = torch.zeros((B, kv, cap), device="cuda"), torch.zeros((B, kv, cap), dtype=torch.int32, device="cuda")
    ctx, seen = i32([80, 7]), i32([80, 7])
    pos[:] = torch.arange(cap, dtype=torch.int32, device="cuda")
    wq, wk = (torch.rand(D, generator=g, device="cuda") + 0.5 for _ in range(2))
    sim = [[dict(k=R.f64(k)[b, h, :c].copy(), v=R.f64(v)[b, h, :c].copy(), pos=list(range(c))) for h in range(kv)]
           for b, c in enumerate((80, 7))]
    tokens = [80, 7]
    ta = M.tree_args(batch=B, n_draft=n, heads=heads, kv_heads=kv, dim=D, cap=cap, max_ctx=cap)
    aa = M.append_args(batch=B, n_draft=n, kv_heads=kv, dim=D, cap=cap)
    wa = M.weights_args(batch=B, n_q=n, heads=heads, kv_heads=kv, dim=D, cap=cap, max_ctx=cap, decay=0.9)
    ea = M.evict_args(batch=B, kv_heads=kv, dim=D, cap=cap, max_ctx=cap, budget=budget, recent=recent, sinks=sinks)
    tws, wws, ews = (buffer(x) for x in (M.attn_tree_workspace(ta), M.cache_weights_workspace(wa),
                                         M.cache_evict_workspace(ea)))
    o = torch.zeros((B * n, heads * D), device="cuda")
    lse = torch.zeros((heads, B * n), device="cuda")
    q, kd, vd = (torch.zeros((x, B * n, D), dtype=dt, device="cuda") for x in (heads, kv, kv))
    for step in range(20):
        masks = random_masks(rng, B, n)
        nodes = [n, int(rng.integers(2, n + 1))]
        depth = [[bin(m).count("1") - 1 for m in ms] for ms in masks]
        cs = angles([tokens[b] + depth[b][r] for b in range(B) for r in range(n)], D)
        xq, xk, xv = (randn(g, (B * n, x * D), F32) for x in (heads, kv, kv))
        kw = dict(rows=B * n, col0=0, stride=D, dim=D, n_pad=B * n)
        M.heads(xq, q, ld=heads * D, heads=heads, rope=1, rot=D, eps=1e-6, cs=cs, w=wq, **kw)
        M.heads(xk, kd, ld=kv * D, heads=kv, rope=1, rot=D, eps=1e-6, cs=cs, w=wk, **kw)
        M.heads(xv, vd, ld=kv * D, heads=kv, **kw)
        M.attn_tree(ta, q, k, v, kd, vd, ctx, o, tws, n_nodes=i32(nodes), mask=as_i64(masks), lse=lse)
        torch.cuda.synchronize()
        # the attention over the simulated cache: a list's rows in any order give the same sums
        lens = [len(sim[b][0]["pos"]) for b in range(B)]
        assert ctx.tolist() == lens and seen.tolist() == tokens
        ks, vs = np.zeros((B, kv, cap, D)), np.zeros((B, kv, cap, D))
        for b in range(B):
            for h in range(kv):
                ks[b, h, :lens[b]], vs[b, h, :lens[b]] = sim[b][h]["k"], sim[b][h]["v"]
        wo, wl, to, tl = R.tree(R.f64(q), ks, vs, R.f64(kd), R.f64(vd), lens, nodes, masks, n=n, scale=ta.scale, out=F32,
                                in_dtype=dt)
        check(o, wo, to, f"step {step} o")
        check(lse, wl, tl, f"step {step} lse")
        # accept the path to some node
        paths = [[j for j in range(n) if masks[b][rng.integers(0, nodes[b])] >> j & 1] for b in range(B)]
        paths = [p or [0] for p in paths]
        path = i32([p + [0] * (n - len(p)) for p in paths])
        count = i32([len(p) for p in paths])
        before_w = R.f64(w)
        M.cache_append(aa, kd, vd, k, v, ctx, ctx, path=path, n_path=count, seen=seen, seen_out=seen, w=w, pos=pos)
        M.cache_weights(wa, q, lse, k, ctx, w, wws, w=w, path=path, n_path=count)
        torch.cuda.synchronize()
        for b in range(B):
            for h in range(kv):
                s = sim[b][h]
                rows = [b * n + j for j in paths[b]]
                s["k"] = np.concatenate([s["k"], R.f64(kd)[h, rows]])
                s["v"] = np.concatenate([s["v"], R.f64(vd)[h, rows]])
                s["pos"] += [tokens[b] + i for i in range(len(rows))]
            tokens[b] += len(paths[b])
        lens = [len(sim[b][0]["pos"]) for b in range(B)]
        ks = np.zeros((B, kv, cap, D))
        for b in range(B):
            before_w[b, :, lens[b] - len(paths[b]):lens[b]] = 0
            for h in range(kv):
                ks[b, h, :lens[b]] = sim[b][h]["k"]
        qf, lf = R.f64(q), R.f64(lse)
        ww, tw = R.weights(lambda b, h, r: qf[h, b * n + r], lambda b, h, r: lf[h, b * n + r], ks, lens, paths, before_w,
                           heads=heads, scale=wa.scale, decay=wa.decay)
        check(w, ww, tw, f"step {step} w")
        wf = w.cpu().numpy().copy()
        M.cache_evict(ea, k, v, w, ctx, w, pos, ctx, ews, pos=pos, seen=seen)
        torch.cuda.synchronize()
        for b in range(B):
            for h in range(kv):
                s = sim[b][h]
                rows = R.evict_rows(wf[b, h, :lens[b]], np.array(s["pos"]), tokens[b], budget, recent, sinks)
                s["k"], s["v"], s["pos"] = s["k"][rows], s["v"][rows], [s["pos"][j] for j in rows]
                m = len(rows)
                assert pos[b, h, :m].tolist() == s["pos"]
                assert np.array_equal(w[b, h, :m].cpu().numpy(), wf[b, h, rows])
                assert np.array_equal(R.f64(k)[b, h, :m], s["k"]) and np.array_equal(R.f64(v)[b, h, :m], s["v"])
    assert ctx.tolist()[0] == budget and seen.tolist()[0] > budget, "nothing was evicted"


class Loop:
    """A serving step's four calls on state of its own, in place."""

    def __init__(self, seed, *, dt=F16, D=128, heads=8, kv=2, ctx=(700, 90, 1300), n=9, budget=640, cap=1400, direct=False):
        g, rng, B = gen(seed), np.random.default_rng(seed), len(ctx)
        self.first = [randn(g, (B, kv, cap, D), dt) for _ in range(2)] + [
            torch.rand((B, kv, cap), generator=g, device="cuda"),
            torch.arange(cap, dtype=torch.int32, device="cuda").expand(B, kv, cap).contiguous(), i32(list(ctx)),
            i32(list(ctx))]
        self.q = randn(g, (heads, B * n, D), dt)
        self.kd, self.vd = (randn(g, (kv, B * n, D), dt) for _ in range(2))
        masks = random_masks(rng, B, n)
        self.mask = as_i64(masks)
        paths = [[j for j in range(n) if ms[n - 1] >> j & 1] for ms in masks]
        self.path, self.count = i32([p + [0] * (n - len(p)) for p in paths]), i32([len(p) for p in paths])
        self.o = torch.zeros((B * n, heads * D), dtype=dt, device="cuda")
        self.lse = torch.zeros((heads, B * n), device="cuda")
        self.args = (M.tree_args(batch=B, n_draft=n, heads=heads, kv_heads=kv, dim=D, cap=cap, max_ctx=cap),
                     M.append_args(batch=B, n_draft=n, kv_heads=kv, dim=D, cap=cap),
                     M.weights_args(batch=B, n_q=n, heads=heads, kv_heads=kv, dim=D, cap=cap, max_ctx=cap),
                     M.evict_args(batch=B, kv_heads=kv, dim=D, cap=cap, max_ctx=cap, budget=budget, recent=40, sinks=3))
        t, _, w, e = self.args
        self.ws = [buffer(x) for x in (M.attn_tree_workspace(t), M.cache_weights_workspace(w), M.cache_evict_workspace(e))]
        self.state = [x.clone() for x in self.first]

    def reset(self):
        for x, y in zip(self.state, self.first):
            x.copy_(y)

    def step(self):
        k, v, w, pos, ctx, seen = self.state
        t, a, wa, e = self.args
        M.attn_tree(t, self.q, k, v, self.kd, self.vd, ctx, self.o, self.ws[0], mask=self.mask, lse=self.lse)
        M.cache_append(a, self.kd, self.vd, k, v, ctx, ctx, path=self.path, n_path=self.count, seen=seen, seen_out=seen,
                       w=w, pos=pos)
        M.cache_weights(wa, self.q, self.lse, k, ctx, w, self.ws[1], w=w, path=self.path, n_path=self.count)
        M.cache_evict(e, k, v, w, ctx, w, pos, ctx, self.ws[2], pos=pos, seen=seen)

    def result(self):
        return [x.clone() for x in (*self.state, self.o, self.lse)]


def same(a, b):
    return all(torch.equal(x, y) for x, y in zip(a, b))


@pytest.mark.parametrize("kw", [dict(), dict(dt=BF16, D=64, heads=4, kv=4, n=20), dict(D=256, heads=16, kv=1, n=8)],
                         ids=["few", "many", "wide"])
def test_graph_replays(kw):
    """The step captured once and replayed: every replay leaves the state that the same step made eagerly, with eager work
    and synchronizations between the replays."""
    x = Loop(21, **kw)
    want = []
    for _ in range(4):
        x.step()
        torch.cuda.synchronize()
        want.append(x.result())
    x.reset()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        x.step()
    for i in range(4):
        graph.replay()
        torch.cuda.synchronize()
        assert same(x.result(), want[i]), f"replay {i}"
        torch.randn(1 << 16, device="cuda").sum().item()


def test_two_streams_at_once():
    """Two loops with workspaces of their own on two streams: each as alone."""
    loops = [Loop(31), Loop(32, dt=BF16, D=64, heads=4, kv=4)]
    want = []
    for x in loops:
        for _ in range(5):
            x.step()
        torch.cuda.synchronize()
        want.append(x.result())
        x.reset()
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in loops]
    for _ in range(5):
        for s, x in zip(streams, loops):
            with torch.cuda.stream(s):
                x.step()
    torch.cuda.synchronize()
    for x, y in zip(loops, want):
        assert same(x.result(), y)


def test_cache_past_32_bit_offsets():
    """A cache of 10 GiB a tensor: its last lists lie past 2^32 elements and bytes. Small contexts in it, all four calls."""
    B, kv, heads, D, cap, n = 5, 8, 8, 128, 1 << 20, 3
    ctx = [0, 1, 0, 3, 300]
    k, v = (torch.zeros((B, kv, cap, D), dtype=F16, device="cuda") for _ in range(2))
    w, pos = (torch.zeros((B, kv, cap), dtype=t, device="cuda") for t in (F32, torch.int32))
    g, rng = gen(51), np.random.default_rng(51)
    for b, c in enumerate(ctx):
        for t in (k, v):
            t[b, :, :c] = randn(g, (kv, c, D), F16)
        w[b, :, :c] = torch.rand((kv, c), generator=g, device="cuda")
        pos[b, :, :c] = torch.arange(c, dtype=torch.int32, device="cuda")
    q = randn(g, (heads, B * n, D), F16)
    kd, vd = (randn(g, (kv, B * n, D), F16) for _ in range(2))
    small = [R.f64(t[:, :, :400]) for t in (k, v)]
    a = M.tree_args(batch=B, n_draft=n, heads=heads, kv_heads=kv, dim=D, cap=cap, max_ctx=cap)
    o, lse = torch.zeros((B * n, heads * D), device="cuda"), torch.zeros((heads, B * n), device="cuda")
    M.attn_tree(a, q, k, v, kd, vd, i32(ctx), o, buffer(M.attn_tree_workspace(a)), lse=lse)
    torch.cuda.synchronize()
    wo, wl, to, tl = R.tree(R.f64(q), *small, R.f64(kd), R.f64(vd), ctx, [n] * B, None, n=n, scale=a.scale, out=F32,
                            in_dtype=F16)
    check(o, wo, to, "o")
    check(lse, wl, tl, "lse")
    ctx_d, seen = i32(ctx), i32(ctx)
    M.cache_append(M.append_args(batch=B, n_draft=n, kv_heads=kv, dim=D, cap=cap), kd, vd, k, v, ctx_d, ctx_d, seen=seen,
                   seen_out=seen, w=w, pos=pos)
    wa = M.weights_args(batch=B, n_q=n, heads=heads, kv_heads=kv, dim=D, cap=cap, max_ctx=cap)
    w0 = R.f64(w[:, :, :400])
    M.cache_weights(wa, q, lse, k, ctx_d, w, buffer(M.cache_weights_workspace(wa)), w=w)
    torch.cuda.synchronize()
    after = [c + n for c in ctx]
    for b, c in enumerate(ctx):
        assert torch.equal(k[b, :, c:c + n], kd[:, b * n:(b + 1) * n]) and torch.equal(v[b, :, c:c + n], vd[:, b * n:(b + 1) * n])
        assert pos[b, 0, c:c + n].tolist() == [c, c + 1, c + 2]
    qf, lf = R.f64(q), R.f64(lse)
    ww, tw = R.weights(lambda b, h, r: qf[h, b * n + r], lambda b, h, r: lf[h, b * n + r], R.f64(k[:, :, :400]), after,
                       [list(range(n))] * B, w0, heads=heads, scale=wa.scale, decay=1.0)
    check(w[:, :, :400], ww, tw, "w")
    ea = M.evict_args(batch=B, kv_heads=kv, dim=D, cap=cap, max_ctx=cap, budget=128, recent=16, sinks=1)
    wf, before = w[:, :, :400].cpu().numpy(), [t[:, :, :400].clone() for t in (k, v)]
    M.cache_evict(ea, k, v, w, ctx_d, w, pos, ctx_d, buffer(M.cache_evict_workspace(ea)), pos=pos, seen=seen)
    torch.cuda.synchronize()
    assert ctx_d.tolist() == [min(c, 128) for c in after]
    for h in range(kv):
        rows = R.evict_rows(wf[4, h, :303], np.arange(303), 303, 128, 16, 1)
        assert torch.equal(k[4, h, :128], before[0][4, h, rows]) and torch.equal(v[4, h, :128], before[1][4, h, rows])
        assert pos[4, h, :128].tolist() == rows


def test_longest_list():
    """One list of 2^23 - 1 rows, just under 2 GiB of K: the last rows count. Keys of zero give every row the same weight."""
    n, D, ctx = 2, 128, (1 << 23) - 1
    k, v = (torch.zeros((1, 1, ctx, D), dtype=BF16, device="cuda") for _ in range(2))
    v[0, 0, ctx - 1], v[0, 0, 0] = 2.0, 1.0
    q = torch.ones((1, n, D), dtype=BF16, device="cuda")
    kd, vd = torch.zeros((1, n, D), dtype=BF16, device="cuda"), torch.zeros((1, n, D), dtype=BF16, device="cuda")
    a = M.tree_args(batch=1, n_draft=n, heads=1, kv_heads=1, dim=D, cap=ctx, max_ctx=ctx)
    o, lse = torch.zeros((n, D), device="cuda"), torch.zeros((1, n), device="cuda")
    M.attn_tree(a, q, k, v, kd, vd, i32([ctx]), o, buffer(M.attn_tree_workspace(a)), lse=lse)
    torch.cuda.synchronize()
    # powers of two all along, but for the count: 3 / (ctx + 1 + r); the sums of 16 equal terms a lane and their joins
    want = torch.tensor([3.0 / (ctx + 1), 3.0 / (ctx + 2)], device="cuda")[:, None].expand(n, D)
    torch.testing.assert_close(o, want, rtol=2.0 ** -14, atol=0)
    torch.testing.assert_close(lse, torch.log(torch.tensor([[ctx + 1.0, ctx + 2.0]], device="cuda")), rtol=0, atol=1e-4)
    wa = M.weights_args(batch=1, n_q=n, heads=1, kv_heads=1, dim=D, cap=ctx, max_ctx=ctx)
    w = torch.zeros((1, 1, ctx), device="cuda")
    M.cache_weights(wa, q, lse, k, i32([ctx]), w, buffer(M.cache_weights_workspace(wa)))
    torch.cuda.synchronize()
    # the last row is the second query's alone
    torch.testing.assert_close(w[0, 0, :-1], torch.full((ctx - 1,), 2.0 / ctx, device="cuda"), rtol=2.0 ** -12, atol=0)
    torch.testing.assert_close(w[0, 0, -1:], torch.full((1,), 1.0 / ctx, device="cuda"), rtol=2.0 ** -12, atol=0)
    w[0, 0, 5::7] = 1.0
    w[0, 0, -1] = 2.0
    ea = M.evict_args(batch=1, kv_heads=1, dim=D, cap=ctx, max_ctx=ctx, budget=1 << 20)
    pos, ctx_o = torch.zeros((1, 1, ctx), dtype=torch.int32, device="cuda"), i32([0])
    M.cache_evict(ea, k, v, w, i32([ctx]), torch.zeros_like(w), pos, ctx_o, buffer(M.cache_evict_workspace(ea)))
    torch.cuda.synchronize()
    got = pos[0, 0, :1 << 20].sort().values
    rows = torch.cat([torch.arange(5, ctx - 1, 7)[:(1 << 20) - 1], torch.tensor([ctx - 1])]).int().cuda()
    assert torch.equal(got, rows) and ctx_o.tolist() == [1 << 20]
