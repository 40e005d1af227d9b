"""The operators of a cache kept in pages on the GPU, against plain forms in 64 bits (tests/pages_ref.py): attention of one
token or a chunk of each sequence over its pages, the write of rows, reservation, fork and compaction."""
import math
import random

import pytest
import torch

import mako_attn as M
import pages_ref as R

pytestmark = pytest.mark.gpu
DT = {"f16": torch.float16, "bf16": torch.bfloat16}


def gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def ints(x):
    return torch.tensor(x, dtype=torch.int32, device="cuda")


def space(n):
    return torch.empty(max(16, n), dtype=torch.uint8, device="cuda")


class Pool:
    """Sequences of ctx + new rows over pages anywhere in a pool that holds NaN wherever no sequence has a row."""

    def __init__(self, g, ctx, new, kv, dim, page, dtype, spare=3, extra=2, fill=math.nan):
        total = [c + n for c, n in zip(ctx, new)]
        held = [-(-t // page) for t in total]
        self.max_pages = max(held + [1]) + extra
        self.pages, self.page = sum(held) + spare, page
        order = torch.randperm(self.pages, generator=g, device="cuda").int()
        self.table = torch.full((len(ctx), self.max_pages), -1, dtype=torch.int32, device="cuda")
        self.k, self.v = (torch.full((self.pages, kv, page, dim), fill, dtype=dtype, device="cuda") for _ in range(2))
        at = 0
        for b, h in enumerate(held):
            mine = order[at:at + h].long()
            self.table[b, :h] = mine.int()
            at += h
            for x in (self.k, self.v):
                rows = torch.randn((h * page, kv, dim), generator=g, device="cuda").to(dtype)
                rows[total[b]:] = fill
                x[mine] = rows.view(h, page, kv, dim).transpose(1, 2)


def run_attention(dtype, heads, kv, dim, page, ctx, new, *, out=None, seed=0, decode=False, max_new=None, max_ctx=None,
                  behind=0, q_pad=0, width=0, scale=None, pool=None, want_lse=True, edit=None, ws_fill=0xA5, repeat=1, q_fill=None):
    g = gen(seed)
    dt = DT[dtype]
    odt = {None: dt, "f32": torch.float32}[out]
    pool = pool or Pool(g, ctx, new, kv, dim, page, dt)
    if edit:
        edit(pool)
    B = len(ctx)
    starts = [sum(new[:b]) for b in range(B + 1)]
    rows = starts[-1] + behind
    q = torch.randn((heads, rows + q_pad, dim), generator=g, device="cuda").to(dt)
    if q_fill is not None:
        q[:, starts[-1]:] = q_fill
    w = heads * dim + width
    a = M.paged_args(batch=B, rows=rows, heads=heads, kv_heads=kv, dim=dim, pages=pool.pages, page=page,
                     max_pages=pool.max_pages, max_new=max(new) if max_new is None else max_new,
                     max_ctx=max(c + n for c, n in zip(ctx, new)) if max_ctx is None else max_ctx, q_pad=rows + q_pad,
                     width=w, scale=scale)
    o = torch.full((rows, w), 777.0, dtype=odt, device="cuda")
    lse = torch.full((heads, rows), 777.0, device="cuda")
    ws = space(M.attn_paged_workspace(a))
    for _ in range(repeat):
        ws.fill_(ws_fill)
        M.attn_paged(a, q, pool.k, pool.v, pool.table, ints(ctx), o, ws, starts=None if decode else ints(starts),
                     lse=lse if want_lse else None)
    torch.cuda.synchronize()
    res = R.attention(q, pool.k.nan_to_num(0.0), pool.v.nan_to_num(0.0), pool.table.tolist(), ctx, new, starts,
                      scale=a.scale, max_ctx=a.max_ctx, max_new=a.max_new, out_dtype=odt)
    left = torch.ones(rows, dtype=torch.bool, device="cuda")
    for b, s0, n, want, want_l, tol, ltol in res:
        got = o[s0:s0 + n, :heads * dim].double().view(n, heads, dim)
        err = (got - want).abs()
        bad = ~(err <= tol)
        assert not bad.any(), (f"sequence {b}: {int(bad.sum())} of {bad.numel()} outputs off, the worst by "
                               f"{float((err / tol).nan_to_num(math.inf).max()):.2f} of what is allowed")
        if want_lse:
            e = (lse[:, s0:s0 + n].t().double() - want_l).abs()
            assert (e <= ltol).all(), f"sequence {b}: lse off by {float(e.max()):.3g}"
        left[s0:s0 + n] = False
    assert (o[left] == 777).all() and (o[:, heads * dim:] == 777).all(), "rows or columns of no sequence were written"
    assert not want_lse or (lse[:, left] == 777).all()
    return o, lse


HEADS = [(1, 1, 128), (4, 4, 64), (4, 2, 128), (8, 2, 128), (6, 2, 128), (16, 2, 128), (8, 2, 64), (3, 1, 64), (8, 8, 128),
         (2, 1, 256), (8, 1, 256), (4, 4, 256), (3, 1, 256), (16, 2, 256)]


@pytest.mark.parametrize("heads,kv,dim", HEADS)
@pytest.mark.parametrize("dtype", ["f16", "bf16"])
def test_mixed_batch(heads, kv, dim, dtype):
    """One token, chunks of odd sizes, a prompt from nothing and a sequence without new rows in one call."""
    run_attention(dtype, heads, kv, dim, 64, [0, 391, 70, 5, 200], [130, 1, 77, 0, 65], seed=heads + dim)


@pytest.mark.parametrize("dim,heads,kv", [(64, 8, 2), (128, 8, 2), (256, 4, 2)])
@pytest.mark.parametrize("out", [None, "f32"])
@pytest.mark.parametrize("dtype", ["f16", "bf16"])
def test_types_and_layouts(dim, heads, kv, out, dtype):
    """f32 output, padded query heads, wider o rows, rows behind the last sequence, loose bounds."""
    run_attention(dtype, heads, kv, dim, 128, [300, 17], [1, 100], out=out, behind=5, q_pad=3, width=8, max_new=106,
                  max_ctx=512, seed=3)


@pytest.mark.parametrize("dim,heads,kv", [(64, 4, 4), (128, 8, 2), (128, 2, 1), (256, 16, 2)])
@pytest.mark.parametrize("ctx", [0, 1, 62, 63, 64, 65, 127, 128, 129, 255, 256, 1000])
def test_single_tokens(dim, heads, kv, ctx):
    """Decode steps (starts NULL) at every edge of a page and a tile."""
    run_attention("bf16", heads, kv, dim, 64, [ctx, max(0, ctx - 1), ctx + 3], [1, 1, 1], decode=True, seed=ctx)


@pytest.mark.parametrize("heads,kv,dim", [(8, 1, 64), (16, 2, 128), (24, 1, 128), (16, 1, 256), (32, 4, 128)])
@pytest.mark.parametrize("out", [None, "f32"])
@pytest.mark.parametrize("new", [[1, 1, 1], [3, 16, 8], [31, 1, 64], [100, 33, 1]], ids=str)
def test_groups_of_eight(heads, kv, dim, out, new):
    """Two heads a wave: steps and chunks over short and long contexts, whole items and pieces, every kind of output."""
    for ctx in ([0, 65, 300], [3000, 17, 900]):
        run_attention("bf16", heads, kv, dim, 64, ctx, new, out=out, behind=2, q_pad=5, width=8, seed=heads + new[0])


@pytest.mark.parametrize("n", [1, 2, 15, 16, 17, 31, 32, 33, 63, 64, 65, 127, 128, 129, 191, 255, 256, 257, 300])
@pytest.mark.parametrize("dim,heads,kv", [(64, 2, 2), (128, 4, 1), (256, 4, 1)])
def test_chunk_lengths(n, dim, heads, kv):
    run_attention("f16", heads, kv, dim, 64, [0, 100], [n, n], seed=n)


@pytest.mark.parametrize("page", [64, 128, 256, 1024, 4096])
@pytest.mark.parametrize("dim", [64, 128, 256])
def test_page_sizes(page, dim):
    run_attention("bf16", 4, 2, dim, page, [5000, 100, 4095], [3, 200, 2], seed=page)


@pytest.mark.parametrize("dim,heads,kv", [(64, 16, 16), (128, 32, 8), (256, 16, 2)])
def test_long_contexts(dim, heads, kv):
    """Keys split over workgroups, unlike lengths, chunks and single tokens."""
    run_attention("bf16", heads, kv, dim, 64, [20000, 33, 9000, 12345], [1, 40, 500, 1], seed=5, repeat=2)


@pytest.mark.parametrize("dim,heads,kv", [(64, 4, 1), (128, 4, 1), (128, 1, 1), (256, 4, 2)])
def test_one_long_chunk(dim, heads, kv):
    run_attention("f16", heads, kv, dim, 256, [3000], [1111], seed=6)


@pytest.mark.parametrize("batch", [64, 65, 130, 200])
def test_many_sequences(batch):
    """More sequences than one look-up of the lanes holds; some without new rows."""
    g = torch.Generator().manual_seed(batch)
    ctx = torch.randint(0, 300, (batch,), generator=g).tolist()
    new = torch.randint(0, 5, (batch,), generator=g).tolist()
    run_attention("bf16", 8, 2, 128, 64, ctx, new, seed=batch)
    run_attention("f16", 4, 4, 64, 64, ctx, [1] * batch, decode=True, seed=batch)


@pytest.mark.parametrize("dim", [64, 128, 256])
def test_missing_pages_read_as_zeros(dim):
    def edit(pool):
        pool.table[0, 2] = -1
        pool.table[0, 5] = pool.pages
        pool.table[1, 0] = 2 ** 31 - 1
    run_attention("bf16", 4, 2, dim, 64, [600, 10], [70, 20], edit=edit, seed=9)


@pytest.mark.parametrize("dim", [64, 128, 256])
def test_bounds_cut(dim):
    """Rows past max_new are left alone; cache rows past max_ctx are not seen."""
    run_attention("bf16", 4, 2, dim, 64, [100, 300, 7], [90, 5, 3], max_new=50, max_ctx=290, seed=10)


@pytest.mark.parametrize("dim", [64, 128, 256])
@pytest.mark.parametrize("growth", [0.5, 2.0])
def test_growing_scores(dim, growth):
    """Scores that pass the running maximum again and again, in whole and split segments."""
    def edit(pool):
        for b in range(2):
            for j, e in enumerate(pool.table[b].tolist()):
                if e >= 0:
                    pool.k[e] *= 1 + growth * j / 8
    run_attention("f16", 4, 2, dim, 64, [900, 5000], [70, 1], edit=edit, seed=11)


@pytest.mark.parametrize("dim", [64, 128, 256])
@pytest.mark.parametrize("n", [2, 16, 33, 100])
@pytest.mark.parametrize("value", [math.nan, math.inf, -math.inf, "low"])
def test_a_later_rows_k_is_not_seen(dim, n, value):
    """Whatever the k of a sequence's last new row holds, the rows before it are as with any other."""
    def run(x):
        g = gen(17)
        pool = Pool(g, [900, 70], [n, n], 2, dim, 64, torch.bfloat16, fill=0.0)
        at = [(900 + n - 1) // 64, (70 + n - 1) // 64]
        if x is not None:
            for b, c in ((0, 900), (1, 70)):
                pool.k[pool.table[b, at[b]].item(), :, (c + n - 1) % 64] = torch.finfo(torch.bfloat16).min if x == "low" else x
        a = M.paged_args(batch=2, rows=2 * n, heads=8, kv_heads=2, dim=dim, pages=pool.pages, page=64,
                         max_pages=pool.max_pages, max_new=n, max_ctx=900 + n)
        q = torch.randn((8, 2 * n, dim), generator=g, device="cuda").bfloat16()
        o = torch.zeros((2 * n, 8 * dim), dtype=torch.bfloat16, device="cuda")
        lse = torch.zeros((8, 2 * n), device="cuda")
        M.attn_paged(a, q, pool.k, pool.v, pool.table, ints([900, 70]), o, space(M.attn_paged_workspace(a)),
                     starts=ints([0, n, 2 * n]), lse=lse)
        torch.cuda.synchronize()
        before = [i for i in range(2 * n) if i % n != n - 1]
        return o[before], lse[:, before]
    (o, lse), (want, want_l) = run(value), run(None)
    assert torch.equal(o, want) and torch.equal(lse, want_l)


@pytest.mark.parametrize("heads,kv,dim", [(4, 2, 64), (8, 2, 128), (8, 1, 128), (4, 2, 256), (8, 1, 256)])
@pytest.mark.parametrize("n", [2, 16, 33, 100])
@pytest.mark.parametrize("value", [math.nan, math.inf])
@pytest.mark.parametrize("dtype,out", [("bf16", None), ("f16", "f32")])
def test_a_later_rows_v_is_not_seen(heads, kv, dim, n, value, dtype, out):
    """A v that is not finite in one of a sequence's new rows reaches the rows from there on, in its head dim, and none before."""
    ctx, dt, rows = [5000, 70], DT[dtype], 2 * n
    odt = torch.float32 if out else dt
    g = gen(19)
    pool = Pool(g, ctx, [n, n], kv, dim, 64, dt, fill=math.nan)
    first = n // 2  # the first row that sees it
    for b in range(2):
        j = ctx[b] + first
        pool.v[pool.table[b, j // 64].item(), kv - 1, j % 64, 5] = value
    a = M.paged_args(batch=2, rows=rows, heads=heads, kv_heads=kv, dim=dim, pages=pool.pages, page=64, max_pages=pool.max_pages,
                     max_new=n, max_ctx=5000 + n)
    q = torch.randn((heads, rows, dim), generator=g, device="cuda").to(dt)
    o, lse = torch.zeros((rows, heads * dim), dtype=odt, device="cuda"), torch.zeros((heads, rows), device="cuda")
    M.attn_paged(a, q, pool.k, pool.v, pool.table, ints(ctx), o, space(M.attn_paged_workspace(a)), starts=ints([0, n, rows]),
                 lse=lse)
    torch.cuda.synchronize()
    pool.v.nan_to_num_(nan=0.0, posinf=0.0)
    res = R.attention(q, pool.k.nan_to_num(0.0), pool.v, pool.table.tolist(), ctx, [n, n], [0, n], scale=a.scale,
                      max_ctx=a.max_ctx, max_new=n, out_dtype=odt)
    mine = torch.arange(heads, device="cuda") * kv // heads == kv - 1
    for b, s0, m, want, want_l, tol, ltol in res:
        got = o[s0:s0 + m].double().view(m, heads, dim)
        off = ~((got - want).abs() <= tol)
        assert not off[:first].any() and not off[:, :, :5].any() and not off[:, :, 6:].any() and not off[:, ~mine].any()
        hit = got[first:, mine, 5]
        assert (hit.isnan() | hit.isinf()).all()
        assert ((lse[:, s0:s0 + m].t().double() - want_l).abs() <= ltol).all()


@pytest.mark.parametrize("heads,kv,dim", [(4, 2, 64), (8, 2, 128), (8, 1, 128), (4, 2, 256), (8, 1, 256)])
@pytest.mark.parametrize("fill", [math.nan, math.inf])
def test_queries_of_no_sequence(heads, kv, dim, fill):
    """What q holds behind the last sequence's rows, and in its padding, has no part."""
    for new in ([1, 1], [3, 17], [40, 70]):
        run_attention("bf16", heads, kv, dim, 64, [700, 90], new, behind=3, q_pad=70, q_fill=fill, seed=20)


@pytest.mark.parametrize("seed", range(32))
def test_calls_of_any_kind(seed):
    """Batches, groups, lengths, pages, types, paddings and bounds drawn together."""
    r = random.Random(seed)
    dim, kv, group = r.choice([64, 128, 256]), r.choice([1, 2, 3, 8]), r.choice([1, 2, 3, 4, 5, 6, 7, 8, 12, 16, 24])
    kv = kv if kv * group <= 48 else 1
    batch = r.choice([1, 2, 3, 5, 9, 40, 70])
    high, most = (6000, 700) if batch <= 5 else (400, 40)
    ctx = [r.choice([0, 1, 63, 64, r.randint(0, 200), r.randint(0, high)]) for _ in range(batch)]
    kind = r.choice(["step", "few", "chunk", "mixed"])
    new = [1 if kind == "step" or (kind == "mixed" and r.random() < 0.7) else r.randint(0, 20 if kind == "few" else most)
           for _ in range(batch)]
    new[0] = max(new[0], 1)
    page, dtype, step = r.choice([64, 128, 512]), r.choice(["f16", "bf16"]), kind == "step"
    pool = Pool(gen(seed), ctx, new, kv, dim, page, DT[dtype], extra=r.choice([0, 512 // page]))
    run_attention(dtype, kv * group, kv, dim, page, ctx, new, out=r.choice([None, "f32"]), behind=0 if step else r.choice([0, 3]),
                  q_pad=r.choice([0, 7, 64]), width=r.choice([0, 8]), decode=step, seed=seed, pool=pool,
                  max_new=r.choice([None, sum(new)]), max_ctx=r.choice([None, pool.max_pages * page]))


def test_scale_and_no_lse():
    run_attention("bf16", 4, 2, 128, 64, [200, 0], [33, 1], scale=0.5, want_lse=False, seed=12)


def test_shared_pages():
    """Two sequences hold the same pages."""
    g = gen(13)
    pool = Pool(g, [400], [0], 2, 128, 64, torch.bfloat16)
    pool.table = torch.cat([pool.table, pool.table, pool.table]).contiguous()
    run_attention("bf16", 8, 2, 128, 64, [399, 200, 335], [1, 64, 65], pool=pool, seed=13)


@pytest.mark.parametrize("dim", [64, 128, 256])
def test_unruly_starts_stay_inside(dim):
    """Starts that fall, or lie past the rows, are cut to the rows: only rows of o are written, and calls end."""
    g = gen(14)
    pool = Pool(g, [100, 200, 300], [40, 40, 40], 2, dim, 64, torch.float16, fill=0.0)
    a = M.paged_args(batch=3, rows=120, heads=4, kv_heads=2, dim=dim, pages=pool.pages, page=64, max_pages=pool.max_pages,
                     max_new=120, max_ctx=64 * pool.max_pages)
    q = torch.randn((4, 120, dim), generator=g, device="cuda").half()
    for st in ([0, 80, 40, 120], [5, 2, 1, 0], [0, 1000, 2000, -1], [-1, -1, -1, -1]):
        o = torch.full((122, 4 * dim), 777.0, dtype=torch.float16, device="cuda")
        lse = torch.full((4 * 120 + 64,), 777.0, device="cuda")
        M.attn_paged(a, q, pool.k, pool.v, pool.table, ints([100, -5, 300]), o, space(M.attn_paged_workspace(a)),
                     starts=ints(st), lse=lse)
        torch.cuda.synchronize()
        assert (o[120:] == 777).all() and (lse[480:] == 777).all() and o.isfinite().all()


def test_nothing_to_do():
    a = M.paged_args(batch=0, rows=0, heads=4, kv_heads=2, dim=128, pages=1, page=64, max_pages=1, max_new=0, max_ctx=64)
    x = torch.zeros(64, dtype=torch.float16, device="cuda")
    i = ints([0, 0])
    M.attn_paged(a, x, x, x, i, i, x, space(M.attn_paged_workspace(a)), starts=i)
    run_attention("f16", 4, 2, 128, 64, [100, 100], [0, 0], behind=3, seed=1, max_new=1, max_ctx=128)


def test_workspace_too_short():
    a = M.paged_args(batch=2, rows=2, heads=32, kv_heads=8, dim=128, pages=2000, page=64, max_pages=1000, max_new=1,
                     max_ctx=60000)
    need = M.attn_paged_workspace(a)
    if need:
        x = torch.zeros(64, dtype=torch.float16, device="cuda")
        with pytest.raises(M.MakoError, match="workspace"):
            M.attn_paged(a, x, x, x, ints([0]), ints([0]), x, space(need)[:need - 1])


def test_another_stream_and_a_graph():
    """The call on a stream of its own, captured and replayed with other lengths, against the eager call each time."""
    g = gen(15)
    ctx, new = [700, 3000, 64], [1, 30, 70]
    pool = Pool(g, [800, 3100, 200], new, 2, 128, 64, torch.bfloat16, fill=0.0)
    a = M.paged_args(batch=3, rows=101, heads=8, kv_heads=2, dim=128, pages=pool.pages, page=64, max_pages=pool.max_pages,
                     max_new=101, max_ctx=pool.max_pages * 64)
    q = torch.randn((8, 101, 128), generator=g, device="cuda").bfloat16()
    c, st = ints(ctx), ints([0, 1, 31, 101])
    ws, o = space(M.attn_paged_workspace(a)), torch.zeros((101, 1024), dtype=torch.bfloat16, device="cuda")
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        M.attn_paged(a, q, pool.k, pool.v, pool.table, c, o, ws, starts=st)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        M.attn_paged(a, q, pool.k, pool.v, pool.table, c, o, ws, starts=st)
    for step in range(4):
        c.copy_(ints([ctx[0] + step, ctx[1] - 700 * step, ctx[2] + 3 * step]))
        q.normal_(generator=g)
        ws.random_()
        graph.replay()
        got = o.clone()
        ws.zero_()
        M.attn_paged(a, q, pool.k, pool.v, pool.table, c, o, ws, starts=st)
        torch.cuda.synchronize()
        assert torch.equal(got, o), step


# ---- the pages ------------------------------------------------------------------------------------------------------


def tables(g, batch, page, high, beams=1, spare=8, extra=3):
    ctx = torch.randint(0, high + 1, (batch,), generator=g).tolist()
    ctx = [ctx[b // beams * beams] for b in range(batch)]
    held = [-(-c // page) for c in ctx]
    pages = sum(held[::beams]) + spare
    order, at, table = torch.randperm(pages, generator=g).tolist(), 0, []
    for b in range(batch):
        if b % beams:
            table.append(list(table[-1]))
            continue
        table.append(order[at:at + held[b]] + [-1] * (max(held) + extra - held[b]))
        at += held[b]
    refs = [0] * pages
    for row in table:
        for e in row:
            if e >= 0:
                refs[e] += 1
    return table, refs, ctx, pages


@pytest.mark.parametrize("kv,dim,dtype", [(1, 64, "f16"), (8, 128, "bf16"), (2, 256, "f16"), (3, 128, "bf16")])
@pytest.mark.parametrize("batch,most,page", [(1, 1, 64), (5, 1, 64), (70, 3, 128), (3, 400, 64), (130, 20, 256)])
def test_write(kv, dim, dtype, batch, most, page):
    g, h = gen(batch), torch.Generator().manual_seed(batch + kv)
    new = torch.randint(0 if most > 1 else 1, most + 1, (batch,), generator=h).tolist()
    table, refs, ctx, pages = tables(h, batch, page, 300, extra=2)
    flat = torch.randperm(4 * pages, generator=h)[:batch * len(table[0])].tolist() if batch < 4 else None
    table = [[e if e >= 0 else (flat[b * len(row) + j] if flat else -1) for j, e in enumerate(row)]
             for b, row in enumerate(table)]  # (some past the pool)
    starts = [sum(new[:b]) for b in range(batch + 1)]
    rows = starts[-1] + 4
    kd, vd = (torch.randn((kv, rows + 2, dim), generator=g, device="cuda").to(DT[dtype]) for _ in range(2))
    k, v = (torch.randn((pages, kv, page, dim), generator=g, device="cuda").to(DT[dtype]) for _ in range(2))
    end = [c + 2 for c in ctx] if batch == 5 else None
    want_k, want_v = k.clone(), v.clone()
    R.write(want_k, want_v, kd, vd, table, ctx, new, starts, end)
    a = M.pages_args(batch=batch, rows=rows, d_pad=rows + 2, pages=pages, page=page, max_pages=len(table[0]), kv_heads=kv,
                     dim=dim)
    M.pages_write(a, kd, vd, k, v, ints(table), ints(ctx), starts=None if most == 1 else ints(starts),
                  end=None if end is None else ints(end))
    assert torch.equal(k, want_k) and torch.equal(v, want_v)


@pytest.mark.parametrize("in_place", [False, True])
@pytest.mark.parametrize("batch,most,beams,spare", [(1, 1, 1, 3), (64, 1, 4, 100), (70, 1, 3, 10), (33, 200, 1, 500),
                                                    (9, 900, 2, 20), (1200, 1, 5, 700), (16, 1, 1, 20000)])
def test_reserve(batch, most, beams, spare, in_place):
    page, kv, dim = 64, 2, 64
    h = torch.Generator().manual_seed(batch)
    new = torch.randint(0 if most > 1 else 1, most + 1, (batch,), generator=h).tolist()
    table, refs, ctx, pages = tables(h, batch, page, 300, beams, spare, extra=-(-most // page) + 1)
    starts = [sum(new[:b]) for b in range(batch + 1)]
    layers = 2 if pages < 5000 else 0
    k = v = None
    if layers:
        k, v = (torch.randn((layers, pages, kv, page, dim), generator=gen(1), device="cuda").half() for _ in range(2))
        want_k, want_v = k.clone(), v.clone()
    a = M.pages_args(batch=batch, rows=starts[-1], pages=pages, page=page, max_pages=len(table[0]), kv_heads=kv, dim=dim,
                     layers=layers)
    t, r, c = ints(table), ints(refs), ints(ctx)
    to, ro, co = (t, r, c) if in_place else (torch.empty_like(t), torch.empty_like(r), torch.empty_like(c))
    M.pages_reserve(a, k, v, t, r, c, to, ro, co, space(M.pages_reserve_workspace(a)),
                    starts=None if most == 1 else ints(starts))
    want_t, want_r, want_c, moves = R.reserve(table, refs, ctx, new, page, pages)
    assert to.tolist() == want_t and ro.tolist() == want_r and co.tolist() == want_c
    if layers:
        for src, dst, n in moves:
            want_k[:, dst, :, :n], want_v[:, dst, :, :n] = want_k[:, src, :, :n], want_v[:, src, :, :n]
        assert torch.equal(k, want_k) and torch.equal(v, want_v)


@pytest.mark.parametrize("in_place", [False, True])
@pytest.mark.parametrize("batch,beams,page", [(1, 1, 64), (64, 4, 64), (100, 1, 128), (600, 3, 64)])
@pytest.mark.parametrize("form", ["both", "parent", "keep", "neither"])
def test_fork(batch, beams, page, form, in_place):
    h = torch.Generator().manual_seed(batch)
    table, refs, ctx, pages = tables(h, batch, page, 900, beams)
    refs = [r + (i % 7 == 0) for i, r in enumerate(refs)]  # pages that the caller holds too
    parent = torch.randint(-1, batch + 1, (batch,), generator=h).tolist() if form in ("both", "parent") else None
    keep = torch.randint(0, 1000, (batch,), generator=h).tolist() if form in ("both", "keep") else None
    a = M.pages_args(batch=batch, pages=pages, page=page, max_pages=len(table[0]))
    t, r, c = ints(table), ints(refs), ints(ctx)
    to, ro, co = (t, r, c) if in_place else (torch.empty_like(t), torch.empty_like(r), torch.empty_like(c))
    M.pages_fork(a, t, r, c, to, ro, co, space(M.pages_fork_workspace(a)) if in_place else None,
                 parent=None if parent is None else ints(parent), keep=None if keep is None else ints(keep))
    want_t, want_r, want_c = R.fork(table, refs, ctx, parent, keep, page)
    assert to.tolist() == want_t and ro.tolist() == want_r and co.tolist() == want_c


@pytest.mark.parametrize("in_place", [False, True])
@pytest.mark.parametrize("batch,spare,layers", [(1, 5, 1), (20, 0, 2), (20, 77, 3), (64, 900, 1), (5, 40000, 0)])
def test_compact(batch, spare, layers, in_place):
    page, kv, dim = 64, 2, 128
    h = torch.Generator().manual_seed(spare)
    table, refs, ctx, pages = tables(h, batch, page, 700, 1, spare)
    k = v = None
    if layers:
        k, v = (torch.randn((layers, pages, kv, page, dim), generator=gen(1), device="cuda").bfloat16() for _ in range(2))
        want_k, want_v = k.clone(), v.clone()
    a = M.pages_args(batch=batch, pages=pages, page=page, max_pages=len(table[0]), kv_heads=kv, dim=dim, layers=layers)
    t, r, used, names = ints(table), ints(refs), ints([5]), ints([7] * pages)
    to, ro = (t, r) if in_place else (torch.empty_like(t), torch.empty_like(r))
    M.pages_compact(a, k, v, t, r, to, ro, used, space(M.pages_compact_workspace(a)), map_out=names if spare else None)
    want_t, want_r, n, number = R.compact(table, refs)
    assert to.tolist() == want_t and ro.tolist() == want_r and used.tolist() == [n]
    assert not spare or names.tolist() == number
    if layers:
        for src, dst in enumerate(number):
            if dst >= 0 and dst != src:
                want_k[:, dst], want_v[:, dst] = want_k[:, src], want_v[:, src]
        assert torch.equal(k, want_k) and torch.equal(v, want_v)
