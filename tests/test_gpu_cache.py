"""The cache operators on the GPU against their definitions in 64 bits (tests/cache_ref.py, with the bounds that follow
from the kernels' roundings): attention of drafted trees (mako_attn_tree), append (mako_cache_append), gathered weights
(mako_cache_weights), eviction (mako_cache_evict); at odd sizes, empty rows, ragged batches, masked places that hold NaN
and infinities, rows that must stay as they were."""
import numpy as np
import pytest

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

import cache_ref as R  # noqa: E402
import mako_attn as M  # noqa: E402

F16, BF16, F32 = torch.float16, torch.bfloat16, torch.float32
NAN = float("nan")


def gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def randn(g, shape, dt, scale=1.0):
    return (torch.randn(shape, generator=g, device="cuda") * scale).to(dt)


def i32(x):
    return torch.tensor(x, dtype=torch.int32, device="cuda")


def buffer(n):
    return torch.full((max(n, 16),), 0xA5, dtype=torch.uint8, device="cuda")


def random_masks(rng, B, n, empty=0.0):
    """Trees: node r sees its ancestors and itself; a share of the rows sees no draft."""
    masks = []
    for _ in range(B):
        m = []
        for r in range(n):
            up = rng.integers(-1, r) if r else -1
            m.append((m[up] if up >= 0 else 0) | 1 << r)
        masks.append([0 if rng.random() < empty else x for x in m])
    return masks


def as_i64(masks):
    return torch.from_numpy(np.array(masks, dtype=np.uint64).view(np.int64)).cuda()


def check(got, want, tol, what):
    got = got.cpu().double().numpy()
    nan = np.isnan(want)
    assert np.array_equal(np.isnan(got) & ~nan, np.zeros_like(nan)), f"{what}: NaN in a row that has a value"
    inf = np.isinf(want)
    assert np.array_equal(got[inf], want[inf]), f"{what}: infinities differ"
    ok = ~nan & ~inf
    err = np.abs(got[ok] - want[ok])
    bad = err > tol[ok]
    assert not bad.any(), f"{what}: {bad.sum()} of {bad.size} over the bound, worst {np.max(err / np.maximum(tol[ok], 1e-300)):.2f} times"


def run_tree(*, dt, out, dim, heads, kv, ctx, n, nodes=None, masks="tree", cap=None, max_ctx=None, pad=0, wide=0,
             seed=0, scale=1.0, empty=0.0, dirty=True):
    """Everything that a row does not see, and every padding row, holds NaN (dirty); rows and columns that the call leaves
    alone are checked to be as they were."""
    B, g, rng = len(ctx), gen(seed), np.random.default_rng(seed)
    cap = max(max(ctx), 1) + 5 if cap is None else cap
    rows = B * n
    q = randn(g, (heads, rows + pad, dim), dt, scale)
    k, v = (randn(g, (B, kv, cap, dim), dt) for _ in range(2))
    kd, vd = (randn(g, (kv, rows + pad, dim), dt) for _ in range(2))
    live = [n] * B if nodes is None else nodes
    m = random_masks(rng, B, n, empty) if masks == "tree" else None
    clean = [R.f64(t) for t in (q, k, v, kd, vd)]
    if dirty:
        for b in range(B):
            k[b, :, ctx[b]:], v[b, :, ctx[b]:] = NAN, NAN
            for t in (kd, vd):
                t[:, b * n + live[b]:(b + 1) * n] = NAN
        for t in (q, kd, vd):
            t[:, rows:] = NAN
    o = torch.full((rows + 1, heads * dim + wide), 7.0, dtype=out, device="cuda")
    lse = torch.full((heads, rows), 7.0, device="cuda")
    a = M.tree_args(batch=B, n_draft=n, heads=heads, kv_heads=kv, dim=dim, cap=cap,
                    max_ctx=cap if max_ctx is None else max_ctx, q_pad=rows + pad, d_pad=rows + pad,
                    width=heads * dim + wide)
    ws = buffer(M.attn_tree_workspace(a))
    print(f"tree {dt} {out} dim {dim} heads {heads}/{kv} ctx {ctx} n {n} nodes {nodes}", flush=True)
    M.attn_tree(a, q, k, v, kd, vd, i32(ctx), o, ws, n_nodes=None if nodes is None else i32(nodes),
                mask=None if m is None else as_i64(m), lse=lse)
    torch.cuda.synchronize()
    seen = [min(c, a.max_ctx) for c in ctx]
    wo, wl, to, tl = R.tree(*clean, seen, live, m, n=n, scale=a.scale, out=out, in_dtype=dt)
    gone = np.isnan(wl[0])  # rows past their tree's nodes
    got = o[:rows, :heads * dim]
    check(got, wo, to, "o")
    check(lse, wl, tl, "lse")
    assert torch.all(got[torch.from_numpy(gone)] == 7.0) and torch.all(lse[:, torch.from_numpy(gone).cuda()] == 7.0)
    assert torch.all(o[rows:] == 7.0) and torch.all(o[:, heads * dim:] == 7.0)
    return o, lse


TREES = [
    # dtype, out, dim, heads, kv, contexts, n, nodes
    (F16, F16, 128, 8, 2, [391], 6, None),
    (BF16, BF16, 128, 4, 4, [1], 1, None),
    (BF16, F32, 128, 8, 2, [0, 31, 32, 33, 64, 65], 3, [3, 1, 2, 3, 0, 3]),
    (F16, F32, 128, 4, 2, [129, 0, 700], 17, [17, 5, 9]),
    (BF16, BF16, 128, 8, 2, [513, 95], 64, [64, 33]),
    (F16, F16, 64, 4, 4, [300, 2, 77], 11, [11, 11, 4]),
    (BF16, F32, 64, 6, 2, [257], 23, None),
    (BF16, BF16, 256, 4, 1, [130, 34], 19, [19, 18]),
    (F16, F32, 256, 4, 2, [65], 5, None),
    (F16, F16, 256, 16, 2, [40, 200], 64, [3, 64]),
    (BF16, BF16, 128, 24, 1, [77], 64, None),  # 1536 columns a kv head
    (F16, F16, 128, 3, 1, [1500], 33, None),
    (BF16, BF16, 64, 16, 16, [2000, 1], 1, None),
]


@pytest.mark.parametrize("case", TREES, ids=lambda c: f"d{c[2]}h{c[3]}kv{c[4]}b{len(c[5])}n{c[6]}")
def test_tree(case):
    dt, out, dim, heads, kv, ctx, n, nodes = case
    run_tree(dt=dt, out=out, dim=dim, heads=heads, kv=kv, ctx=ctx, n=n, nodes=nodes, seed=len(ctx) + n)


@pytest.mark.parametrize("dt,out,dim,heads,n,ctx", [
    (F16, F16, 64, 2, 4, 300001), (BF16, F32, 64, 2, 32, 150000), (F16, F32, 64, 4, 64, 45001),
    (BF16, BF16, 128, 2, 4, 150000), (F16, F16, 128, 2, 32, 70001), (BF16, F32, 128, 4, 64, 45000),
    (F16, F16, 256, 2, 4, 70001), (BF16, BF16, 256, 2, 32, 70000), (F16, F16, 256, 2, 64, 45000), (BF16, F32, 256, 4, 64, 25001)])
def test_tree_long_ranges(dt, out, dim, heads, n, ctx):
    """One list so long that each of 256 workgroups goes round its ring several times."""
    run_tree(dt=dt, out=out, dim=dim, heads=heads, kv=1, ctx=[ctx], n=n, seed=9)


def test_tree_chain_padding_and_wide_rows():
    """No mask: node r sees the drafts up to it. Padded heads of q and the draft tiles, o rows wider than the heads, a
    context over max_ctx (cut to it)."""
    run_tree(dt=BF16, out=F32, dim=128, heads=4, kv=2, ctx=[50, 333], n=9, nodes=[9, 4], masks=None, pad=3, wide=12,
             cap=400, max_ctx=300, seed=3)
    run_tree(dt=F16, out=F16, dim=64, heads=2, kv=1, ctx=[33], n=64, masks=None, seed=4)


def test_tree_rows_that_see_nothing():
    run_tree(dt=F16, out=F16, dim=128, heads=4, kv=2, ctx=[0, 0, 40], n=8, empty=0.6, seed=5)
    run_tree(dt=BF16, out=F32, dim=256, heads=2, kv=2, ctx=[0], n=5, empty=1.0, seed=6)


def test_tree_large_scores():
    """Scores to about +-500: the running maximum moves often, most probabilities vanish."""
    run_tree(dt=BF16, out=F32, dim=128, heads=4, kv=2, ctx=[700, 45], n=12, scale=120.0, seed=7)
    run_tree(dt=F16, out=F16, dim=64, heads=4, kv=2, ctx=[300], n=40, scale=60.0, seed=8)


@pytest.mark.parametrize("bad", [NAN, float("inf"), -float("inf")])
@pytest.mark.parametrize("dt", [F16, BF16])
def test_tree_masked_drafts_hold_anything(dt, bad):
    """A draft that some nodes see and others do not: its K and V change only the rows that see it."""
    B, n, heads, kv, dim, ctx = 2, 10, 4, 2, 128, [70, 5]
    g, rng = gen(11), np.random.default_rng(11)
    q = randn(g, (heads, B * n, dim), dt)
    k, v = (randn(g, (B, kv, 80, dim), dt) for _ in range(2))
    kd, vd = (randn(g, (kv, B * n, dim), dt) for _ in range(2))
    m = random_masks(rng, B, n)
    a = M.tree_args(batch=B, n_draft=n, heads=heads, kv_heads=kv, dim=dim, cap=80, max_ctx=80)
    ws, ctx_d = buffer(M.attn_tree_workspace(a)), i32(ctx)

    def call(x, y):
        o = torch.zeros((B * n, heads * dim), device="cuda")
        lse = torch.zeros((heads, B * n), device="cuda")
        M.attn_tree(a, q, k, v, x, y, ctx_d, o, ws, mask=as_i64(m), lse=lse)
        torch.cuda.synchronize()
        return o, lse

    o0, l0 = call(kd, vd)
    for j in (0, 3, n - 1):
        for which in "kv":
            x, y = kd.clone(), vd.clone()
            (x if which == "k" else y)[:, [j, n + j], ::7] = bad
            o1, l1 = call(x, y)
            sees = torch.tensor([[mm >> j & 1 for mm in s] for s in m], dtype=torch.bool).reshape(-1).cuda()
            # (a row that does not see it may sum in another order, not lose it: the bounds are test_tree's)
            torch.testing.assert_close(o1[~sees], o0[~sees], rtol=2.0 ** -9 if dt == BF16 else 2.0 ** -12, atol=1e-4)
            torch.testing.assert_close(l1[:, ~sees], l0[:, ~sees], rtol=1e-6, atol=1e-5)
            if which == "v":
                assert not torch.isfinite(o1.view(B * n, heads, dim)[sees][..., ::7]).any()
            elif bad != bad:
                assert torch.isnan(o1[sees]).all() and torch.isnan(l1[:, sees]).all()


def test_tree_value_range():
    """bf16 values over bf16's whole range meet P in bf16: 1e30 beside 1e-30."""
    dt, n, dim = BF16, 4, 128
    g = gen(12)
    q, kd = randn(g, (2, n, dim), dt), randn(g, (1, n, dim), dt)
    k = randn(g, (1, 1, 100, dim), dt)
    v, vd = randn(g, (1, 1, 100, dim), dt), randn(g, (1, n, dim), dt)
    for t in (v, vd):
        t[..., :32] *= 1e30
        t[..., 32:64] *= 1e-30
    a = M.tree_args(batch=1, n_draft=n, heads=2, kv_heads=1, dim=dim, cap=100, max_ctx=100)
    o, ws = torch.zeros((n, 2 * dim), device="cuda"), buffer(M.attn_tree_workspace(a))
    M.attn_tree(a, q, k, v, kd, vd, i32([100]), o, ws)
    torch.cuda.synchronize()
    wo, _, to, _ = R.tree(*[R.f64(t) for t in (q, k, v, kd, vd)], [100], [n], None, n=n, scale=a.scale, out=F32,
                          in_dtype=dt)
    check(o, wo, to, "o")


def test_tree_one_node_is_decode():
    """A node a sequence whose draft is the cache's last row: mako_attn_decode's result over the cache."""
    B, heads, kv, cap, ctx = 5, 16, 4, 900, [1, 2, 33, 640, 900]
    g = gen(13)
    k, v = (randn(g, (B, kv, cap, 128), F16) for _ in range(2))
    q = randn(g, (heads, B, 128), F16)
    last = torch.tensor(ctx) - 1
    kd, vd = (torch.stack([t[b, :, last[b]] for b in range(B)], 1).contiguous() for t in (k, v))
    a = M.tree_args(batch=B, n_draft=1, heads=heads, kv_heads=kv, dim=128, cap=cap, max_ctx=cap)
    o, lse = torch.zeros((B, heads * 128), device="cuda"), torch.zeros((heads, B), device="cuda")
    M.attn_tree(a, q, k, v, kd, vd, i32([c - 1 for c in ctx]), o, buffer(M.attn_tree_workspace(a)), lse=lse)
    d = M.decode_args(batch=B, heads=heads, kv_heads=kv, dim=128, cap=cap, max_ctx=cap)
    o2, lse2 = torch.zeros_like(o), torch.zeros((B, heads), device="cuda")
    M.attn_decode(d, q.transpose(0, 1).contiguous(), k, v, i32(ctx), o2, buffer(M.decode_workspace(d)), lse=lse2)
    torch.cuda.synchronize()
    # decode's P has 11 bits: 2^-11 of sum p |v| (below 4)
    torch.testing.assert_close(o, o2, rtol=0, atol=4 * 2.0 ** -11)
    torch.testing.assert_close(lse, lse2.t(), rtol=0, atol=2e-5)


def test_tree_same_bits_every_time():
    """No order that changes between calls: the same call again gives the same bits, beside another call's work."""
    first = run_tree(dt=BF16, out=BF16, dim=128, heads=8, kv=2, ctx=[1200, 900], n=9, seed=20)
    again = run_tree(dt=BF16, out=BF16, dim=128, heads=8, kv=2, ctx=[1200, 900], n=9, seed=20)
    assert torch.equal(first[0], again[0]) and torch.equal(first[1], again[1])


# ---- append --------------------------------------------------------------------------------------------------------


APPENDS = [
    # dtype, dim, kv, n, contexts, n_path, cap
    (F16, 128, 8, 8, [333], [5], 4096),
    (BF16, 64, 3, 5, [0, 10, 40, 37], [5, 0, 5, 9], 40),  # at the cap, over it, more than n_draft
    (BF16, 256, 2, 64, [7, 0], [64, 63], 100),
    (F16, 128, 1, 1, [0], [1], 1),
]


@pytest.mark.parametrize("case", APPENDS, ids=lambda c: f"d{c[1]}kv{c[2]}n{c[3]}b{len(c[4])}")
@pytest.mark.parametrize("in_place", [False, True])
def test_append(case, in_place):
    dt, dim, kv, n, ctx, count, cap = case
    B, g, rng = len(ctx), gen(30), np.random.default_rng(30)
    kd, vd = (randn(g, (kv, B * n + 2, dim), dt) for _ in range(2))
    k, v = (randn(g, (B, kv, cap, dim), dt) for _ in range(2))
    w = torch.rand((B, kv, cap), generator=g, device="cuda") + 1
    pos = torch.randint(0, 1 << 30, (B, kv, cap), generator=g, device="cuda", dtype=torch.int32)
    path = rng.integers(0, n + 2, (B, n))  # some past the drafts, some twice
    seen = [c + 1000 * b for b, c in enumerate(ctx)]
    want = [t.clone() for t in (k, v, w, pos)]
    ends = []
    for b in range(B):
        m = min(count[b], n, cap - ctx[b])
        for i in range(m):
            src, at = int(path[b, i]), ctx[b] + i
            for t, d in ((want[0], kd), (want[1], vd)):
                t[b, :, at] = d[:, b * n + src] if src < n else 0
            want[2][b, :, at], want[3][b, :, at] = 0, seen[b] + i
        ends.append(m)
    ctx_d, seen_d = i32(ctx), i32(seen)
    ctx_o, seen_o = (ctx_d, seen_d) if in_place else (torch.zeros_like(ctx_d), torch.zeros_like(seen_d))
    a = M.append_args(batch=B, n_draft=n, kv_heads=kv, dim=dim, cap=cap, d_pad=B * n + 2)
    print(f"append {case} {in_place}", flush=True)
    M.cache_append(a, kd, vd, k, v, ctx_d, ctx_o, path=i32(path.tolist()), n_path=i32(count), seen=seen_d,
                   seen_out=seen_o, w=w, pos=pos)
    torch.cuda.synchronize()
    for got, exp in zip((k, v, w, pos), want):
        assert torch.equal(got, exp)
    assert ctx_o.tolist() == [c + m for c, m in zip(ctx, ends)]
    assert seen_o.tolist() == [c + m for c, m in zip(seen, ends)]


def test_append_all_rows_without_weights():
    """No path, counts, weights or positions: every draft in order."""
    B, n, kv, dim, cap = 3, 7, 2, 128, 50
    g = gen(31)
    kd, vd = (randn(g, (kv, B * n, dim), BF16) for _ in range(2))
    k, v = (randn(g, (B, kv, cap, dim), BF16) for _ in range(2))
    wk, wv, ctx = k.clone(), v.clone(), [0, 20, 43]
    for b, c in enumerate(ctx):
        wk[b, :, c:c + n], wv[b, :, c:c + n] = kd[:, b * n:(b + 1) * n], vd[:, b * n:(b + 1) * n]
    ctx_o = i32([0] * B)
    M.cache_append(M.append_args(batch=B, n_draft=n, kv_heads=kv, dim=dim, cap=cap), kd, vd, k, v, i32(ctx), ctx_o)
    torch.cuda.synchronize()
    assert torch.equal(k, wk) and torch.equal(v, wv) and ctx_o.tolist() == [c + n for c in ctx]


# ---- weights -------------------------------------------------------------------------------------------------------


def run_weights(*, dt, dim, heads, kv, ctx, n, form, count=None, decay=1.0, with_w=True, pad=0, seed=0, in_place=False,
                path=None, lse_set=None, max_ctx=None):
    """form: decode (q by sequence), rows (tiles). lse: the attention's over the keys that a query sees; lse_set changes
    some. Keys that no query sees, and rows past the context, hold NaN."""
    B, g = len(ctx), gen(seed)
    cap = max(ctx) + 3
    k = randn(g, (B, kv, cap, dim), dt)
    q = randn(g, (B, heads, n, dim) if form == "decode" else (heads, B * n + pad, dim), dt)
    at = (lambda t, b, h, r: t[b, h, r]) if form == "decode" else (lambda t, b, h, r: t[h, b * n + r])
    live = [min(c, n) for c in (count or [n] * B)]
    ids = [[r if r < n else None for r in (path[b][:live[b]] if path else range(live[b]))] for b in range(B)]
    seen = [min(c, max_ctx or cap) for c in ctx]
    kf, qf = R.f64(k), R.f64(q)
    lse = np.full((B, heads, n) if form == "decode" else (heads, B * n), 0.25)
    for b in range(B):
        for i, r in enumerate(ids[b]):
            for h in range(heads):
                m = seen[b] - len(ids[b]) + i + 1
                if r is not None and m > 0:
                    s = kf[b, h // (heads // kv), :m] @ at(qf, b, h, r) / dim ** 0.5
                    val = np.float32(s.max() + np.log(np.exp(s - s.max()).sum()))
                    if form == "decode":
                        lse[b, h, r] = val
                    else:
                        lse[h, b * n + r] = val
    if lse_set:
        lse_set(lse)
    for b in range(B):
        k[b, :, ctx[b]:] = NAN
    if pad:
        q[:, B * n:] = NAN
    w = torch.rand((B, kv, cap), generator=g, device="cuda") * 3 if with_w else None
    w_out = w if in_place else torch.full((B, kv, cap), 7.0, device="cuda")
    old = None if w is None else R.f64(w)
    a = M.weights_args(batch=B, n_q=n, heads=heads, kv_heads=kv, dim=dim, cap=cap, max_ctx=max_ctx or cap,
                       q_pad=B * n + pad, decode=form == "decode", decay=decay)
    ws = buffer(M.cache_weights_workspace(a))
    print(f"weights {dt} dim {dim} heads {heads}/{kv} ctx {ctx} n {n} {form} count {count}", flush=True)
    M.cache_weights(a, q, torch.from_numpy(lse).float().cuda(), k, i32(ctx), w_out, ws, w=w,
                    path=None if path is None else i32(path), n_path=None if count is None else i32(count))
    torch.cuda.synchronize()
    want, tol = R.weights(lambda b, h, r: at(qf, b, h, r), lambda b, h, r: float(np.float32(at(lse, b, h, r))), kf, seen, ids,
                          old, heads=heads, scale=a.scale, decay=decay)
    check(w_out, want, tol, "w")
    for b in range(B):
        rest = w_out[b, :, seen[b]:].cpu().double().numpy()
        assert np.array_equal(rest, old[b, :, seen[b]:] if in_place else np.full_like(rest, 7.0)), "rows behind the context"
    return w_out


WEIGHTS = [
    dict(dt=F16, dim=128, heads=8, kv=2, ctx=[300, 1, 77], n=1, form="decode"),
    dict(dt=BF16, dim=64, heads=4, kv=4, ctx=[65, 500], n=1, form="decode", decay=0.5),
    dict(dt=BF16, dim=256, heads=8, kv=1, ctx=[129], n=1, form="decode", with_w=False),
    dict(dt=F16, dim=128, heads=4, kv=2, ctx=[40, 64, 700], n=5, form="decode", in_place=True),
    dict(dt=BF16, dim=128, heads=4, kv=2, ctx=[257], n=257, form="rows"),
    dict(dt=F16, dim=128, heads=4, kv=1, ctx=[500], n=130, form="rows", pad=5),
    dict(dt=BF16, dim=64, heads=3, kv=3, ctx=[333, 200], n=200, form="rows", decay=0.0),
    dict(dt=F16, dim=256, heads=2, kv=1, ctx=[96, 61], n=61, form="rows"),
    dict(dt=BF16, dim=128, heads=32, kv=1, ctx=[70], n=3, form="rows"),
    dict(dt=F16, dim=64, heads=4, kv=2, ctx=[90, 3, 0], n=7, form="rows", count=[4, 3, 0], in_place=True),
    dict(dt=BF16, dim=128, heads=2, kv=1, ctx=[2, 0], n=6, form="rows"),  # more queries than rows
    dict(dt=BF16, dim=128, heads=4, kv=2, ctx=[1100, 1023], n=40, form="rows", count=[40, 9], max_ctx=1024),
]


@pytest.mark.parametrize("case", WEIGHTS, ids=lambda c: f"d{c['dim']}h{c['heads']}kv{c['kv']}n{c['n']}{c['form']}")
def test_weights(case):
    run_weights(seed=len(case["ctx"]) + case["n"], **case)


def test_weights_path():
    """The queries of an accepted path: some of the tree's rows, one twice, one past the drafts (no query)."""
    run_weights(dt=BF16, dim=128, heads=4, kv=2, ctx=[100, 64], n=8, form="rows", count=[5, 8],
                path=[[0, 2, 2, 7, 5, 1, 1, 1], [3, 1, 8, 0, 200, 6, 7, 4]], seed=40)


def test_weights_queries_that_saw_nothing():
    def some(lse):
        lse[1, ::2] = -np.inf
        lse[0, 3] = np.inf

    run_weights(dt=F16, dim=128, heads=2, kv=1, ctx=[150], n=30, form="rows", lse_set=some, seed=41)


@pytest.mark.parametrize("n", [4, 200])
def test_weights_of_keys_that_hold_anything(n):
    """A key that is not finite: its weight is NaN where a query sees it, its old weight where none does, and no other
    key's changes."""
    heads, kv, dim, ctx = 2, 1, 64, 300
    g = gen(43)
    k, q = randn(g, (1, kv, ctx, dim), F16), randn(g, (heads, n, dim), F16)
    lse = torch.full((heads, n), 4.0, device="cuda")
    lse[:, n - 2:] = -float("inf")  # the last two queries, and so the last two keys, are out
    w = torch.rand((1, kv, ctx), generator=g, device="cuda")
    a = M.weights_args(batch=1, n_q=n, heads=heads, kv_heads=kv, dim=dim, cap=ctx, max_ctx=ctx)
    ws, outs = buffer(M.cache_weights_workspace(a)), []
    for bad in (None, NAN, float("inf")):
        if bad is not None:
            k[:, :, [5, ctx - 40, ctx - 1], ::9] = bad
        out = torch.zeros_like(w)
        M.cache_weights(a, q, lse, k, i32([ctx]), out, ws, w=w)
        torch.cuda.synchronize()
        outs.append(out)
    for out in outs[1:]:
        assert torch.isnan(out[..., 5]).all() or torch.isinf(out[..., 5]).all()
        assert torch.equal(out[..., ctx - 1], w[..., ctx - 1])
        fine = torch.ones(ctx, dtype=torch.bool, device="cuda")
        fine[[5, ctx - 40, ctx - 1]] = False
        assert torch.equal(out[..., fine], outs[0][..., fine])


def test_weights_sum_to_the_queries():
    """A whole prompt's weights sum to its queries times the heads of a group, over mako_attn_fwd's lse."""
    n, heads, kv = 1000, 8, 2
    g = gen(42)
    q, k, v = (randn(g, (h, n, 128), BF16) for h in (heads, kv, kv))
    o, lse = torch.zeros((n, heads * 128), device="cuda"), torch.zeros((heads, n), device="cuda")
    M.attn_fwd(q, k, v, o, n_q=n, q_pad=n, n_k=n, k_pad=n, heads=heads, kv_heads=kv, q_pos0=0, block=M.U32_MAX, dim=128,
               lse=lse)
    a = M.weights_args(batch=1, n_q=n, heads=heads, kv_heads=kv, dim=128, cap=n, max_ctx=n)
    w = torch.zeros((1, kv, n), device="cuda")
    M.cache_weights(a, q, lse, k, i32([n]), w, buffer(M.cache_weights_workspace(a)))
    torch.cuda.synchronize()
    # each query's weights sum to exp of its lse's error: below 1e-3 (the attention path's LSE bound)
    torch.testing.assert_close(w.double().sum(-1).cpu(), torch.full((1, kv), float(n * heads // kv), dtype=torch.float64),
                               rtol=1e-3, atol=0)


# ---- eviction ------------------------------------------------------------------------------------------------------


def run_evict(*, dt, dim, kv, ctx, budget, recent=0, sinks=0, moved=False, in_place=False, seed=0, weigh=None,
              max_ctx=None):
    B, g, rng = len(ctx), gen(seed), np.random.default_rng(seed)
    cap = max(ctx) + 2
    k, v = (randn(g, (B, kv, cap, dim), dt) for _ in range(2))
    w = (np.exp(2 * rng.standard_normal((B, kv, cap))) * (rng.random((B, kv, cap)) > 0.2)).astype(np.float32)
    if weigh:
        weigh(w, rng)
    pos = np.stack([[rng.permutation(cap + 50)[:cap] for _ in range(kv)] for _ in range(B)]) if moved else None
    seen = [c + 40 for c in ctx]
    w_d = torch.from_numpy(w).cuda()
    pos_d = None if pos is None else i32(pos.tolist())
    ctx_d = i32(ctx)
    w_o = w_d if in_place else torch.full_like(w_d, 7.0)
    pos_o = pos_d if in_place and moved else torch.full((B, kv, cap), 7, dtype=torch.int32, device="cuda")
    ctx_o = ctx_d if in_place else torch.zeros_like(ctx_d)
    wk, wv, ww, wp = k.clone(), v.clone(), w_o.clone(), pos_o.clone()
    lens = [min(c, max_ctx or cap) for c in ctx]
    for b in range(B):
        n = lens[b]
        for h in range(kv):
            p = np.arange(n) if pos is None else pos[b, h, :n]
            rows = R.evict_rows(w[b, h, :n], p, seen[b] if moved else n, budget, recent, sinks)
            for to, src in ((wk, k), (wv, v)):
                to[b, h, :len(rows)] = src[b, h, rows]
            ww[b, h, :len(rows)] = torch.from_numpy(w[b, h, :n][rows]).cuda()
            wp[b, h, :len(rows)] = i32(p[rows].tolist())
    a = M.evict_args(batch=B, kv_heads=kv, dim=dim, cap=cap, max_ctx=max_ctx or cap, budget=budget, recent=recent,
                     sinks=sinks)
    ws = buffer(M.cache_evict_workspace(a))
    print(f"evict dim {dim} kv {kv} ctx {ctx} budget {budget} recent {recent} sinks {sinks} moved {moved}", flush=True)
    for _ in range(1 if in_place else 2):  # with outputs of its own, the call can be made again
        M.cache_evict(a, k, v, w_d, ctx_d, w_o, pos_o, ctx_o, ws, pos=pos_d, seen=i32(seen) if moved else None)
    torch.cuda.synchronize()
    assert ctx_o.tolist() == [min(n, budget) for n in lens]
    assert torch.equal(pos_o, wp)
    assert torch.equal(w_o.view(torch.int32), ww.view(torch.int32))
    assert torch.equal(k, wk) and torch.equal(v, wv)


def ties(w, rng):
    w[:] = rng.integers(0, 3, w.shape)
    w[:, :, ::5] = -0.0


def odd_values(w, rng):
    w[:] = rng.standard_normal(w.shape)
    for i, x in enumerate((np.nan, np.inf, -np.inf, 1e-42, -1e-42, -np.nan, 3e38)):
        w[:, :, i::23] = x


EVICTS = [
    dict(dt=F16, dim=128, kv=2, ctx=[300], budget=100, recent=20, sinks=4),
    dict(dt=BF16, dim=64, kv=3, ctx=[64, 65, 200, 0, 1], budget=64, recent=16, sinks=2, moved=True),
    dict(dt=BF16, dim=256, kv=1, ctx=[1025, 2500], budget=1024, recent=1024),
    dict(dt=F16, dim=128, kv=2, ctx=[5000], budget=4900, recent=7, moved=True),
    dict(dt=F16, dim=128, kv=2, ctx=[3000, 200], budget=250, weigh=ties),
    dict(dt=BF16, dim=128, kv=2, ctx=[2000, 1999], budget=777, recent=5, sinks=3, weigh=ties, moved=True),
    dict(dt=F16, dim=64, kv=2, ctx=[1500], budget=300, weigh=odd_values),
    dict(dt=F16, dim=64, kv=2, ctx=[1500], budget=1400, weigh=odd_values, recent=31),
    dict(dt=F16, dim=64, kv=1, ctx=[10, 0], budget=0),
    dict(dt=F16, dim=64, kv=1, ctx=[70, 3], budget=1),
    dict(dt=BF16, dim=128, kv=1, ctx=[900, 1000], budget=100, max_ctx=500, recent=9),
    dict(dt=BF16, dim=128, kv=1, ctx=[40000], budget=1000, recent=100, sinks=1),
    dict(dt=BF16, dim=64, kv=1, ctx=[70001, 20], budget=33333, weigh=ties),
]


@pytest.mark.parametrize("case", EVICTS, ids=lambda c: f"d{c['dim']}n{max(c['ctx'])}to{c['budget']}")
@pytest.mark.parametrize("in_place", [False, True])
def test_evict(case, in_place):
    run_evict(in_place=in_place, seed=50 + len(case["ctx"]), **case)


def test_evict_positions_twice_over():
    """Positions that protect more rows than the budget (they do not come from this library): the lower rows stay."""
    n, budget = 200, 50
    g = gen(60)
    k, v = (randn(g, (1, 1, n, 64), F16) for _ in range(2))
    k0, v0 = k.clone(), v.clone()
    w = torch.rand((1, 1, n), generator=g, device="cuda")
    pos = torch.full((1, 1, n), 999, dtype=torch.int32, device="cuda")
    w_o, pos_o, ctx_o = torch.zeros_like(w), torch.zeros_like(pos), i32([0])
    a = M.evict_args(batch=1, kv_heads=1, dim=64, cap=n, max_ctx=n, budget=budget, recent=10)
    M.cache_evict(a, k, v, w, i32([n]), w_o, pos_o, ctx_o, buffer(M.cache_evict_workspace(a)), pos=pos, seen=i32([1000]))
    torch.cuda.synchronize()
    assert torch.equal(k, k0) and torch.equal(v, v0) and torch.equal(w_o[..., :budget], w[..., :budget])
    assert ctx_o.tolist() == [budget]
