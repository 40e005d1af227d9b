"""A pool of pages that runs out, on the GPU: who gets room among sequences of unlike lengths in one page."""
import random

import pytest

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

import mako_attn as M  # noqa: E402
from test_gpu_paged import gen, ints, space  # noqa: E402


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
