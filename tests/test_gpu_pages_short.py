"""A pool of pages that runs out, on the GPU: who gets room among sequences of unlike lengths in one page, and a serving loop
that makes its steps again once pages are free."""
import random

import pytest

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

import mako_attn as M  # noqa: E402
import pages_ref as R  # noqa: E402
from test_gpu_paged import gen, ints, space  # noqa: E402
from test_gpu_pages_run import ALL, Server  # noqa: E402


def room(table, refs, ctx, new, page):
    """Rows that have room: sequences and free pages in order; of those that append to one partly filled page that nobody else
    holds the last keeps it, unless another got no page for its copy and has rows where the last one's new rows would go."""
    free, appends, left, out = refs.count(0), {}, {}, []
    for b, (c, n) in enumerate(zip(ctx, new)):
        if n and c % page and c < page * len(table[b]):
            appends.setdefault(table[b][c // page], []).append(b)
    for b, (c, n) in enumerate(zip(ctx, new)):
        at, end = c, min(c + n, page * len(table[b]))
        while at < end:
            e, part = table[b][at // page], at % page
            needs = e < 0
            if e >= 0 and part and refs[e] > 1:
                needs = refs[e] > len(appends[e]) or appends[e][-1] != b
                if not needs and left.get(e, 0) > part:
                    break
                if needs and not free:
                    left[e] = max(left.get(e, 0), part)
            if needs and not free:
                break
            free -= needs
            at = min(end, (at // page + 1) * page)
        out.append(at)
    return out


@pytest.mark.parametrize("in_place", [False, True])
@pytest.mark.parametrize("batch,beams,most,spare", [(2, 2, 1, 0), (8, 4, 1, 1), (64, 4, 1, 7), (64, 8, 150, 30), (33, 33, 3, 5),
                                                    (2100, 3, 2, 900), (4096, 4096, 1, 50)])
def test_no_row_of_another_sequence_is_written(batch, beams, most, spare, in_place):
    """Sets of sequences cut back to unlike lengths inside the page that they share, a pool with too few free pages: reserve,
    then write. Every sequence's rows are as they were, its new ones behind them."""
    r, page, kv, dim = random.Random(batch + most), 64, 2, 64
    table, ctx, used = [], [], 0
    for b in range(batch):
        if b % beams == 0:
            whole, part = r.randint(0, 2), r.randint(1, page - 1)
            mine = list(range(used, used + whole + 1))
            used += whole + 1
        ctx.append(whole * page + r.randint(1, part))
        table.append(mine + [-1] * (6 - len(mine)))
    pages = used + spare
    order = list(range(pages))
    r.shuffle(order)
    table = [[order[e] if e >= 0 else -1 for e in row] for row in table]
    refs = [0] * pages
    for row in table:
        for e in row:
            if e >= 0:
                refs[e] += 1
    new = [r.randint(0 if most > 1 else 1, most) for _ in range(batch)]
    starts = [sum(new[:b]) for b in range(batch + 1)]
    g = gen(1)
    k, v = (torch.randn((1, pages, kv, page, dim), generator=g, device="cuda").half() for _ in range(2))
    kd, vd = (torch.randn((kv, max(1, starts[-1]), dim), generator=g, device="cuda").half() for _ in range(2))
    t, rf, c, st = ints(table), ints(refs), ints(ctx), ints(starts)
    to, ro = (t, rf) if in_place else (torch.empty_like(t), torch.empty_like(rf))
    old_k, old_v, old_t = k.clone(), v.clone(), t.clone()
    end = torch.empty_like(c)
    a = M.pages_args(batch=batch, rows=kd.shape[1], pages=pages, page=page, max_pages=6, kv_heads=kv, dim=dim, layers=1)
    M.pages_reserve(a, k, v, t, rf, c, to, ro, end, space(M.pages_reserve_workspace(a)), starts=st)
    M.pages_write(a, kd, vd, k[0], v[0], to, c, starts=st, end=end)
    assert end.tolist() == room(table, refs, ctx, new, page)
    holders = torch.zeros(pages + 1, dtype=torch.int32, device="cuda")
    holders.index_add_(0, torch.where(to < 0, pages, to).reshape(-1).long(), torch.ones(to.numel(), dtype=torch.int32, device="cuda"))
    assert torch.equal(holders[:pages], ro)

    def rows(pool, names):  # [batch][kv][rows][dim], rows of no page: others'
        return pool[0][names.clamp(min=0).long()].transpose(1, 2).reshape(batch, kv, 6 * page, dim)
    at = torch.arange(6 * page, device="cuda")
    before = (at < c[:, None])[:, None, :, None]
    fresh = ((at >= c[:, None]) & (at < end[:, None]))[:, None, :, None]
    nth = (st[:-1, None] + at - c[:, None]).clamp(0, kd.shape[1] - 1).long()
    for pool, old, d in ((k, old_k, kd), (v, old_v, vd)):
        got = rows(pool, to)
        assert torch.equal(torch.where(before, got, 0), torch.where(before, rows(old, old_t), 0))
        assert torch.equal(torch.where(fresh, got, 0), torch.where(fresh, d[:, nth].transpose(0, 1), 0))


class Short(Server):
    def step_in(self, new, what):
        """A step in a pool that may run out: new rows that have room, and their attention; returns the rows left."""
        lens = [x[0].shape[2] for x in self.sim]
        want = room(self.table.tolist(), self.refs.tolist(), lens, new, self.page)
        tiles, starts = self.tiles(sum(new)), [sum(new[:b]) for b in range(self.B + 1)]
        plan = self.prepare(sum(new), max(new), max(c + n for c, n in zip(lens, new)))
        self.launch(plan, tiles, ints(starts))
        torch.cuda.synchronize()
        assert self.ctx.tolist() == want, what
        got = [e - c for c, e in zip(lens, want)]
        for b, n in enumerate(got):
            for x in range(2):
                rows = torch.stack([t[1 + x][:, starts[b]:starts[b] + n] for t in tiles])
                self.sim[b][x] = torch.cat([self.sim[b][x], rows], 2)
        self.check_rows(what)
        a, o, lse, _ = plan
        pool = [torch.zeros((self.L, self.B, self.KV, self.cap, self.D), dtype=self.dt, device="cuda") for _ in range(2)]
        for b in range(self.B):
            for x in range(2):
                pool[x][:, b, :, :want[b]] = self.sim[b][x]
        for l, (q, _, _) in enumerate(tiles):
            res = R.attention(q, pool[0][l], pool[1][l], [[b] for b in range(self.B)], lens, got, starts, scale=a.scale,
                              max_ctx=a.max_ctx, max_new=a.max_new, out_dtype=o.dtype)
            for b, s0, n, out, out_l, tol, ltol in res:
                assert ((o[l, s0:s0 + n].double().view(n, self.H, self.D) - out).abs() <= tol).all(), (what, l, b)
                assert ((lse[l, :, s0:s0 + n].t().double() - out_l).abs() <= ltol).all(), (what, l, b)
        return [n - m for n, m in zip(new, got)]

    def check_rows(self, what):
        """What the pages hold of every sequence is its rows (a last chunk may hold pages behind them)."""
        table = self.table.tolist()
        for b, row in enumerate(table):
            n = self.sim[b][0].shape[2]
            held = -(-n // self.page)
            assert all(0 <= e < self.pages for e in row[:held]), (what, b)
            for x, pool in enumerate((self.k, self.v)):
                if held:
                    rows = pool[:, row[:held]].transpose(1, 2).reshape(self.L, self.KV, held * self.page, self.D)[:, :, :n]
                    assert torch.equal(rows, self.sim[b][x]), (what, b)


@pytest.mark.parametrize("heads,kv,dim,dtype", [(8, 2, 128, "bf16"), (4, 4, 64, "f16"), (8, 1, 256, "bf16")])
def test_steps_made_again(heads, kv, dim, dtype):
    """Beams of unlike lengths over one page, then steps that find too few pages; ends of other sequences free some."""
    s = Short(dim, batch=6, heads=heads, kv=kv, dim=dim, page=64, pages=9, cap=320, layers=2, dtype=dtype)
    assert s.step_in([114, 0, 0, 0, 130, 90], "prompts") == [0] * 6  # 2, 3 and 2 pages
    s.fork([0, 0, 0, 0, 4, 5], [114, 94, 107, 70, ALL, ALL], "beams")  # of one page: 50, 30, 43 and 6 rows
    # two free pages: the first two beams copy, the third gets none and the last would write over its rows
    assert s.step_in([1, 1, 1, 1, 0, 0], "two pages") == [0, 0, 1, 1, 0, 0]
    assert s.step_in([0, 0, 1, 1, 0, 0], "none") == [0, 0, 1, 1, 0, 0]
    assert s.step_in([20, 1, 40, 90, 1, 1], "none, some with room in their pages")[:4] == [7, 0, 40, 90]
    s.fork([0, 1, 2, 3, 6, 5], [ALL] * 4 + [0, ALL], "one ends")  # three pages
    assert s.step_in([7, 0, 40, 90, 0, 0], "three pages")[:4] == [0, 0, 0, 32]
    s.fork([0, 6, 2, 3, 6, 6], [ALL, 0, ALL, ALL, 0, 0], "more end")
    assert s.step_in([1, 0, 1, 32, 100, 0], "room for all") == [0] * 6
    s.check_pages("the end")
