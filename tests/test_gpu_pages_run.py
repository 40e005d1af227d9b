"""A cache kept in pages as a serving loop uses it: pages for the new rows, their write and the attention over them in every
layer, forks, ends and compaction; eager against sequences of rows kept beside it, captured into a graph and replayed, on two
streams at once, over pools past 32-bit offsets; and through the C++ host side (tests/cpp/pages_test)."""
import math
import os
import subprocess

import pytest

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

import mako_attn as M  # noqa: E402
import pages_ref as R  # noqa: E402
from conftest import ROOT  # noqa: E402
from test_gpu_paged import DT, gen, ints, space  # noqa: E402

ALL = 1 << 30


def test_cpp_host_side():
    path = os.path.join(ROOT, "tests", "cpp", "bin", "pages_test")
    assert os.path.exists(path), f"{path} is not built (build() makes it)"
    r = subprocess.run([path], capture_output=True, text=True, timeout=120)
    print(r.stdout)
    assert r.returncode == 0 and "all passed" in r.stdout, r.stdout + r.stderr


class Server:
    """A batch's cache in pages and its calls; with `sim`, every sequence's rows beside it, [layers][kv][rows][dim] each of k
    and v."""

    def __init__(self, seed, *, batch, heads, kv, dim, page, pages, cap, layers=1, dtype="bf16", sim=True):
        self.g, self.dt = gen(seed), DT[dtype]
        self.B, self.H, self.KV, self.D, self.L, self.page, self.cap = batch, heads, kv, dim, layers, page, cap
        self.pages, self.max_pages = pages, -(-cap // page)
        self.k, self.v = (torch.full((layers, pages, kv, page, dim), math.nan, dtype=self.dt, device="cuda") for _ in range(2))
        self.table = torch.full((batch, self.max_pages), -1, dtype=torch.int32, device="cuda")
        self.refs, self.ctx, self.end = ints([0] * pages), ints([0] * batch), ints([0] * batch)
        self.base = dict(batch=batch, pages=pages, page=page, max_pages=self.max_pages)
        a = M.pages_args(rows=batch * cap, kv_heads=kv, dim=dim, layers=layers, **self.base)
        self.scratch = [space(f(a)) for f in (M.pages_reserve_workspace, M.pages_fork_workspace, M.pages_compact_workspace)]
        self.sim = [[torch.zeros((layers, kv, 0, dim), dtype=self.dt, device="cuda") for _ in range(2)]
                    for _ in range(batch)] if sim else None

    def randn(self, *shape):
        return torch.randn(shape, generator=self.g, device="cuda").to(self.dt)

    def tiles(self, rows):
        return [[self.randn(h, rows, self.D) for h in (self.H, self.KV, self.KV)] for _ in range(self.L)]

    def prepare(self, rows, max_new, max_ctx=None):
        a = M.paged_args(rows=rows, heads=self.H, kv_heads=self.KV, dim=self.D, max_new=max_new,
                         max_ctx=self.cap if max_ctx is None else max_ctx, **self.base)
        o = torch.zeros((self.L, rows, self.H * self.D), dtype=self.dt, device="cuda")
        return a, o, torch.zeros((self.L, self.H, rows), device="cuda"), space(M.attn_paged_workspace(a))

    def launch(self, plan, tiles, starts):
        """A step's calls; ctx has the new lengths afterwards."""
        a, o, lse, ws = plan
        p = M.pages_args(rows=a.rows, kv_heads=self.KV, dim=self.D, layers=self.L, **self.base)
        M.pages_reserve(p, self.k, self.v, self.table, self.refs, self.ctx, self.table, self.refs, self.end, self.scratch[0],
                        starts=starts)
        for l, (q, kd, vd) in enumerate(tiles):
            M.pages_write(p, kd, vd, self.k[l], self.v[l], self.table, self.ctx, starts=starts, end=self.end)
            M.attn_paged(a, q, self.k[l], self.v[l], self.table, self.ctx, o[l], ws, starts=starts, lse=lse[l])
        self.ctx.copy_(self.end)

    def grow(self, tiles, new):
        at = 0
        for b, n in enumerate(new):
            for x, side in enumerate(self.sim[b]):
                rows = torch.stack([t[1 + x][:, at:at + n] for t in tiles])
                self.sim[b][x] = torch.cat([side, rows], 2)
            at += n

    def check(self, plan, tiles, new, what):
        a, o, lse, _ = plan
        lens = [s[0].shape[2] for s in self.sim]
        assert self.ctx.tolist() == lens, what
        starts = [sum(new[:b]) for b in range(self.B)]
        pool = [torch.zeros((self.L, self.B, self.KV, self.cap, self.D), dtype=self.dt, device="cuda") for _ in range(2)]
        for b in range(self.B):
            for x in range(2):
                pool[x][:, b, :, :lens[b]] = self.sim[b][x]
        for l, (q, _, _) in enumerate(tiles):
            res = R.attention(q, pool[0][l], pool[1][l], [[b] for b in range(self.B)], [c - n for c, n in zip(lens, new)],
                              new, starts, scale=a.scale, max_ctx=a.max_ctx, max_new=a.max_new, out_dtype=o.dtype)
            for b, s0, n, want, want_l, tol, ltol in res:
                got = o[l, s0:s0 + n].double().view(n, self.H, self.D)
                assert ((got - want).abs() <= tol).all(), f"{what}: layer {l}, sequence {b}"
                assert ((lse[l, :, s0:s0 + n].t().double() - want_l).abs() <= ltol).all(), f"{what}: layer {l}, lse {b}"

    def step(self, new, what):
        tiles, starts = self.tiles(sum(new)), ints([sum(new[:b]) for b in range(self.B + 1)])
        plan = self.prepare(sum(new), max(new), max(s[0].shape[2] + n for s, n in zip(self.sim, new)))
        self.launch(plan, tiles, starts)
        self.grow(tiles, new)
        torch.cuda.synchronize()
        self.check(plan, tiles, new, what)
        self.check_pages(what)

    def fork(self, parent, keep, what):
        M.pages_fork(M.pages_args(**self.base), self.table, self.refs, self.ctx, self.table, self.refs, self.ctx,
                     self.scratch[1], parent=ints(parent), keep=ints(keep))
        old = self.sim
        self.sim = [[x[:, :, :keep[i] if p < self.B else 0] for x in old[min(p, self.B - 1)]] for i, p in enumerate(parent)]
        self.check_pages(what)

    def compact(self, what):
        p = M.pages_args(kv_heads=self.KV, dim=self.D, layers=self.L, **self.base)
        used = ints([0])
        M.pages_compact(p, self.k, self.v, self.table, self.refs, self.table, self.refs, used, self.scratch[2])
        refs = self.refs.tolist()
        assert used.tolist() == [sum(r > 0 for r in refs)] and all(refs[:used[0]]), what
        self.check_pages(what)

    def check_pages(self, what):
        """Every page has the holders that the table names; what the sequences' pages hold is their rows."""
        table, refs = self.table.tolist(), [0] * self.pages
        for b, row in enumerate(table):
            n = self.sim[b][0].shape[2]
            held = -(-n // self.page)
            assert all(0 <= e < self.pages for e in row[:held]) and all(e == -1 for e in row[held:]), (what, b)
            for e in row[:held]:
                refs[e] += 1
            if held:
                for x, pool in enumerate((self.k, self.v)):
                    rows = pool[:, row[:held]].transpose(1, 2).reshape(self.L, self.KV, held * self.page, self.D)[:, :, :n]
                    assert torch.equal(rows, self.sim[b][x]), (what, b)
        assert self.refs.tolist() == refs, what


@pytest.mark.parametrize("heads,kv,dim,page,dtype", [(8, 2, 128, 64, "bf16"), (16, 2, 64, 128, "f16"), (4, 1, 256, 64, "bf16")])
def test_serving_loop(heads, kv, dim, page, dtype):
    """Prompts, single tokens, chunks among them; beams that fork, sequences that end, are cut back and start again."""
    s = Server(7, batch=5, heads=heads, kv=kv, dim=dim, page=page, pages=48, cap=768, layers=2, dtype=dtype)
    h = torch.Generator().manual_seed(dim)
    pick = lambda n: int(torch.randint(0, n, (1,), generator=h))  # noqa: E731
    s.step([150, 63, 1, 0, 300], "prompts")
    for i in range(14):
        kind = i % 7
        new = [1] * 5
        if kind == 2:
            new[pick(5)] = 40 + pick(60)
        elif kind == 5:
            new = [pick(4) for _ in range(5)]
        if max(new):
            s.step(new, f"round {i}")
        lens = [x[0].shape[2] for x in s.sim]
        if kind == 1:  # the first goes on as three beams, the last ends
            s.fork([0, 0, 0, 3, 5], [ALL] * 4 + [0], f"round {i}: beams")
            s.step([1, 1, 1, 1, 90], f"round {i}: after the beams")
        elif kind == 3:
            s.fork([0, 1, 2, 3, 4], [max(0, n - pick(70)) for n in lens], f"round {i}: cut back")
        elif kind == 4:
            s.compact(f"round {i}: compaction")
        elif kind == 6:
            s.fork([1, 4, 2, 2, 0], [ALL, 130, ALL, 64, 200], f"round {i}: others'")


@pytest.mark.parametrize("heads,kv,dim", [(8, 2, 128), (8, 1, 128), (4, 2, 64), (8, 1, 256)])
def test_a_step_in_a_graph(heads, kv, dim):
    """A batch's step captured and replayed over page ends, with other tiles, eager calls and forks between; each replay against
    the rows kept beside it."""
    s = Server(3, batch=3, heads=heads, kv=kv, dim=dim, page=64, pages=40, cap=448, layers=2)
    s.step([123, 59, 1], "prompts")
    s.fork([0, 0, 2], [ALL, ALL, ALL], "fork")  # the step's first copies a page
    tiles, plan = s.tiles(3), s.prepare(3, 1)
    state = [x.clone() for x in (s.k, s.v, s.table, s.refs, s.ctx)]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        s.launch(plan, tiles, None)
    torch.cuda.synchronize()
    for x, y in zip((s.k, s.v, s.table, s.refs, s.ctx), state):
        x.copy_(y)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        s.launch(plan, tiles, None)
    torch.cuda.synchronize()
    for i in range(8):
        for t, fresh in zip(tiles, s.tiles(3)):
            for x, y in zip(t, fresh):
                x.copy_(y)
        graph.replay()
        s.grow(tiles, [1, 1, 1])
        torch.cuda.synchronize()
        s.check(plan, tiles, [1, 1, 1], f"replay {i}")
        s.check_pages(f"replay {i}")
        if i == 2:
            s.step([70, 1, 2], "eager between")
        elif i == 5:
            s.fork([1, 0, 1], [ALL, 100, ALL], "fork between")
            s.compact("compaction between")


def test_two_streams():
    """Two batches' steps at once, each with its own cache and workspaces, against the same steps one after the other."""
    def make(seed):
        s = Server(seed, batch=6, heads=8, kv=2, dim=128, page=64, pages=400, cap=3000, layers=2, sim=False)
        steps = []
        for new in ([2500, 70, 1, 900, 1, 33], [1] * 6, [1, 1, 200, 1, 1, 1], [1] * 6):
            steps.append((s.prepare(sum(new), max(new)), s.tiles(sum(new)), ints([sum(new[:b]) for b in range(7)])))
        return s, steps

    def run(s, steps, i):
        s.launch(*steps[i])

    want = []
    for seed in (1, 2):
        s, steps = make(seed)
        for i in range(4):
            run(s, steps, i)
        torch.cuda.synchronize()
        want.append([x[0][1].clone() for x in steps] + [s.table.clone(), s.ctx.clone()])
    both, streams = [make(1), make(2)], [torch.cuda.Stream(), torch.cuda.Stream()]
    torch.cuda.synchronize()
    for i in range(4):
        for (s, steps), stream in zip(both, streams):
            with torch.cuda.stream(stream):
                run(s, steps, i)
    torch.cuda.synchronize()
    for (s, steps), w in zip(both, want):
        got = [x[0][1] for x in steps] + [s.table, s.ctx]
        assert all(torch.equal(a, b) for a, b in zip(got, w))


def test_pools_past_32_bits():
    """Pools of 5 GiB a layer: rows written to, read from and moved out of pages whose offsets pass 32 bits."""
    kv, dim, page, pages = 8, 128, 64, 41000
    k, v = (torch.empty((2, pages, kv, page, dim), dtype=torch.bfloat16, device="cuda") for _ in range(2))
    g = gen(4)
    mine = [pages - 1, 3, 35000, pages - 7]
    table, refs = [mine + [-1]], [0] * pages
    for e in mine:
        refs[e] = 1
    n = 4 * page - 5
    kd, vd = (torch.randn((kv, n, dim), generator=g, device="cuda").bfloat16() for _ in range(2))
    t, st = ints(table), ints([0, n])
    a = M.pages_args(batch=1, rows=n, pages=pages, page=page, max_pages=5, kv_heads=kv, dim=dim, layers=2)
    M.pages_write(a, kd, vd, k[1], v[1], t, ints([0]), starts=st)
    for i, e in enumerate(mine):
        m = min(page, n - i * page)
        assert torch.equal(k[1, e, :, :m], kd[:, i * page:i * page + m]), e
        assert torch.equal(v[1, e, :, :m], vd[:, i * page:i * page + m]), e
    q = torch.randn((8, n, dim), generator=g, device="cuda").bfloat16()
    pa = M.paged_args(batch=1, rows=n, heads=8, kv_heads=kv, dim=dim, pages=pages, page=page, max_pages=5, max_new=n, max_ctx=n)
    o = torch.zeros((n, 8 * dim), dtype=torch.bfloat16, device="cuda")

    def attend():
        M.attn_paged(pa, q, k[1], v[1], t, ints([0]), o, space(M.attn_paged_workspace(pa)), starts=st)
        torch.cuda.synchronize()
        (_, _, _, want, _, tol, _), = R.attention(q, k[1], v[1], t.tolist(), [0], [n], [0], scale=pa.scale, max_ctx=n,
                                                  max_new=n, out_dtype=o.dtype)
        assert ((o.double().view(n, 8, dim) - want).abs() <= tol).all()
        return o.clone()
    before = attend()
    k[0][mine], v[0][mine] = 1.0, 2.0
    used, r = ints([0]), ints(refs)
    M.pages_compact(a, k, v, t, r, t, r, used, space(M.pages_compact_workspace(a)))
    assert used.tolist() == [4] and sorted(t[0, :4].tolist()) == [0, 1, 2, 3] and t[0, 1] == 3
    assert (k[0, :4] == 1).all() and (v[0, :4] == 2).all()
    assert torch.equal(attend(), before)


def test_a_compaction_of_many_holes():
    """More holes than a workgroup lists: used and free pages at random in a large pool."""
    g = torch.Generator().manual_seed(6)
    for pages, share in ((70000, 2), (200001, 3)):
        refs = (torch.randint(0, share, (pages,), generator=g) == 0).int()
        held = refs.nonzero()[:, 0]
        rows = held[torch.randperm(len(held), generator=g)][:4000].view(4, 1000).int()
        table, want = rows.tolist(), R.compact(rows.tolist(), refs.tolist())
        a = M.pages_args(batch=4, pages=pages, page=64, max_pages=1000, kv_heads=1, dim=64, layers=1)
        k, v = (torch.empty((1, pages, 1, 64, 64), dtype=torch.float16, device="cuda") for _ in range(2))
        k[0, :, 0, :, 0] = (torch.arange(pages, device="cuda") % 2048).half()[:, None]
        v[0, :, 0, :, 0] = (torch.arange(pages, device="cuda") // 2048).half()[:, None]
        t, r, used, names = ints(table), refs.cuda(), ints([0]), ints([0] * pages)
        M.pages_compact(a, k, v, t, r, t, r, used, space(M.pages_compact_workspace(a)), map_out=names)
        assert t.tolist() == want[0] and r.tolist() == want[1] and used.tolist() == [want[2]] and names.tolist() == want[3]
        to = names[held.cuda()].long()
        got = k[0, to, 0, :, 0].float() + 2048 * v[0, to, 0, :, 0].float()
        assert torch.equal(got, held.cuda().float()[:, None].expand(-1, 64))
