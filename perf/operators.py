"""The key / value cache's operators, with the sizes they are timed at: attention of drafted tokens over a cache, the
append of the accepted ones, the attention weight that each cached row has gathered, and the eviction by it.

Each case is one call on resident tensors. With `own` false the operator is computed from elementary torch operations in
32 bits; with `own` true by the library's kernels through the public binding (mako-common_amd/mako_attn.py).
"""
import math
import os
import sys

import torch

own = False
TORCH = {"f16": torch.float16, "bf16": torch.bfloat16}


def _library():
    path = os.path.abspath("mako-common_amd")
    if path not in sys.path:
        sys.path.insert(0, path)
    import mako_attn

    return mako_attn


def listed():
    return [
        # a few drafted tokens early in a chat with a small model: latency
        dict(name="tree_small", kind="tree", batch=1, n=6, heads=16, kv=8, dim=128, low=391, cap=391, dtype="f16"),
        # one sequence with a long context and a tree of 16 drafts
        dict(name="tree_one", kind="tree", batch=1, n=16, heads=32, kv=8, dim=128, low=32768, cap=32768, dtype="bf16"),
        # a serving batch with mixed contexts, odd tree sizes
        dict(name="tree_batch", kind="tree", batch=16, n=13, heads=32, kv=8, dim=128, low=1024, cap=32768,
             dtype="f16"),
        # full trees on the gated-attention layers' heads of 256
        dict(name="tree_d256", kind="tree", batch=4, n=64, heads=16, kv=2, dim=256, low=8000, cap=16384, dtype="bf16"),
        # the accepted path of one sequence's tree
        dict(name="append_one", kind="append", batch=1, n=8, kv=8, dim=128, low=333, cap=4096, dtype="bf16"),
        # the accepted paths of a large serving batch
        dict(name="append_batch", kind="append", batch=64, n=64, kv=8, dim=128, low=100, cap=2048, dtype="f16"),
        # a decode step's weights in a serving batch
        dict(name="weights_step", kind="weights", batch=16, n=1, heads=32, kv=8, dim=128, low=1024, cap=32768,
             dtype="f16", form="step"),
        # the weights of an accepted path after its append, heads of 64
        dict(name="weights_path", kind="weights", batch=7, n=11, heads=16, kv=16, dim=64, low=500, cap=2011,
             dtype="bf16", form="path"),
        # a long prompt's weights on an 8B-class model
        dict(name="weights_prompt", kind="weights", batch=1, n=4096, heads=32, kv=8, dim=128, low=4096, cap=4096,
             dtype="bf16", form="rows"),
        # a serving batch a little over its budget, rows in the order that earlier evictions left
        dict(name="evict_step", kind="evict", batch=16, kv=8, dim=128, low=2049, cap=2176, budget=2048, recent=256,
             sinks=4, dtype="bf16", moved=True),
        # one long prompt cut to its budget
        dict(name="evict_prompt", kind="evict", batch=1, kv=8, dim=128, low=32768, cap=32768, budget=4096, recent=512,
             sinks=4, dtype="bf16", moved=False),
        # a serving batch of long prompts cut to their budget
        dict(name="evict_batch", kind="evict", batch=16, kv=8, dim=128, low=1024, cap=32768, budget=4096, recent=333,
             sinks=0, dtype="f16", moved=False),
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    kind = rng.choice(["tree", "tree", "append", "weights", "weights", "evict"])
    dtype = rng.choice(["f16", "bf16"])
    heads, kv, dim = rng.choice([(32, 8, 128), (16, 8, 128), (8, 2, 128), (16, 16, 64), (16, 2, 256)])
    batch = _log(rng, 1, 32)
    cap = _log(rng, 64, min(32768, (16 * 8 * 128 * 32768) // (batch * kv * dim)))
    low = rng.choice([cap, max(1, cap // 2), max(1, cap // 32)])
    if kind == "tree":
        most = 64 if batch * cap <= 65536 else 16
        return dict(kind=kind, batch=batch, n=_log(rng, 1, most), heads=heads, kv=kv, dim=dim, low=low, cap=cap,
                    dtype=dtype)
    if kind == "append":
        n = _log(rng, 1, 64)
        return dict(kind=kind, batch=batch, n=n, kv=kv, dim=dim, low=min(low, max(1, cap - n)), cap=max(cap, n + 1),
                    dtype=dtype)
    if kind == "weights":
        form = rng.choice(["step", "path", "rows"])
        if form == "rows":
            batch, cap = _log(rng, 1, 4), _log(rng, 64, 4096)
            n = _log(rng, 2, max(2, min(cap, 8192 // batch // 2)))
            return dict(kind=kind, batch=batch, n=n, heads=heads, kv=kv, dim=dim, low=max(n, cap // 2), cap=cap,
                        dtype=dtype, form=form)
        n = 1 if form == "step" else _log(rng, 2, min(16, cap))
        return dict(kind=kind, batch=batch, n=n, heads=heads, kv=kv, dim=dim, low=max(low, n), cap=cap, dtype=dtype,
                    form=form)
    budget = _log(rng, 16, cap)
    recent = rng.randint(0, budget // 2)
    return dict(kind=kind, batch=batch, kv=kv, dim=dim, low=low, cap=cap, budget=budget, recent=recent,
                sinks=rng.randint(0, min(8, budget - recent)), dtype=dtype, moved=rng.random() < 0.5)


# ---- inputs ------------------------------------------------------------------------------------------------------


def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _randn(g, shape, dtype):
    """Unit-normal values, as the per-head RMS norms of q and k give them."""
    return torch.randn(shape, generator=g, device="cuda", dtype=torch.float32).to(dtype)


def _counts(g, low, high, n):
    return torch.randint(low, high + 1, (n,), generator=g, device="cuda", dtype=torch.int32)


def _trees(g, batch, n):
    """Random trees: the parent of node r is a node before it (node 0 follows the context). seen [batch][n][n]: r sees its ancestors
    and itself; nodes: the size of each sequence's tree, the largest n."""
    up = (torch.rand((batch, n), generator=g, device="cuda") * torch.arange(n, device="cuda")).long()
    a = torch.eye(n, device="cuda").expand(batch, n, n).clone()
    if n > 1:
        link = torch.zeros((batch, n, n), device="cuda").scatter_(2, up[..., None], 1.0)
        link[:, 0] = 0
        a = a + link
        for _ in range(6):  # ancestors up to 64 steps away
            a = (a @ a).clamp(max=1.0)
    nodes = _counts(g, max(1, n // 2), n, batch)
    nodes[0] = n
    return a > 0, nodes


def _paths(seen, nodes):
    """The last node's path from the context of each tree, as the acceptance of drafts gives it: its ancestors in
    order, then zeros."""
    batch, n, _ = seen.shape
    on = seen[torch.arange(batch, device="cuda"), nodes.long() - 1]
    order = torch.argsort((~on).int(), dim=1, stable=True)
    count = on.sum(1)
    return torch.where(torch.arange(n, device="cuda") < count[:, None], order, 0).int(), count.int()


def _bits(seen):
    n = seen.shape[2]
    one = torch.ones(n, dtype=torch.int64, device="cuda") << torch.arange(n, device="cuda")
    return (seen.long() * one).sum(2)


def _tree_inputs(c, g):
    dt, rows, D = TORCH[c["dtype"]], c["batch"] * c["n"], c["dim"]
    q = _randn(g, (c["heads"], rows, D), dt)
    kd, vd = (_randn(g, (c["kv"], rows, D), dt) for _ in range(2))
    k, v = (_randn(g, (c["batch"], c["kv"], c["cap"], D), dt) for _ in range(2))
    seen, nodes = _trees(g, c["batch"], c["n"])
    return dict(q=q, k=k, v=v, kd=kd, vd=vd, ctx=_counts(g, c["low"], c["cap"], c["batch"]), seen=seen, nodes=nodes)


def _append_inputs(c, g):
    dt, B, KV, D, n = TORCH[c["dtype"]], c["batch"], c["kv"], c["dim"], c["n"]
    kd, vd = (_randn(g, (KV, B * n, D), dt) for _ in range(2))
    k, v = (_randn(g, (B, KV, c["cap"], D), dt) for _ in range(2))
    seen, nodes = _trees(g, B, n)
    path, count = _paths(seen, nodes)
    ctx = _counts(g, c["low"], c["cap"] - n, B)
    return dict(kd=kd, vd=vd, k=k, v=v, path=path, count=count, ctx=ctx, tokens=ctx + _counts(g, 0, 1000, B),
                w=torch.rand((B, KV, c["cap"]), generator=g, device="cuda"),
                pos=torch.arange(c["cap"], device="cuda", dtype=torch.int32).expand(B, KV, -1).contiguous())


def _weights_inputs(c, g):
    """Query rows r of a sequence with ctx rows: the last of them, or in order along a path through n drafts. lse is the
    attention's over the rows that each query sees."""
    dt, B, H, KV, D, n = TORCH[c["dtype"]], c["batch"], c["heads"], c["kv"], c["dim"], c["n"]
    k = _randn(g, (B, KV, c["cap"], D), dt)
    ctx = _counts(g, c["low"], c["cap"], B)
    q = _randn(g, (B, H, 1, D) if c["form"] == "step" else (H, B * n, D), dt)
    path = count = None
    if c["form"] == "path":
        path, count = _paths(*_trees(g, B, n))
        count = torch.minimum(count, ctx)
    qs = q if c["form"] == "step" else q.view(H, B, n, D).transpose(0, 1)  # [B][H][n][D]
    lse = torch.empty((B, H, n), device="cuda")
    key = torch.arange(c["cap"], device="cuda")
    place = torch.zeros((B, n), dtype=torch.int64, device="cuda")
    if path is None:
        place += torch.arange(n, device="cuda") + ctx[:, None] - n
    else:
        step = torch.arange(n, device="cuda").expand(B, n)
        at = torch.where(step < count[:, None], path.long(), n)
        place = torch.zeros((B, n + 1), dtype=torch.int64, device="cuda").scatter_(1, at, step)[:, :n]
        place += (ctx - count)[:, None]
    for b in range(B):
        for h in range(KV):
            G = H // KV
            s = qs[b, h * G:(h + 1) * G].float().reshape(G * n, D) @ k[b, h].float().t() / math.sqrt(D)
            s = s.view(G, n, -1).masked_fill(key > place[b][None, :, None], -math.inf)
            lse[b, h * G:(h + 1) * G] = torch.logsumexp(s, -1)
    lse = lse if c["form"] == "step" else lse.transpose(0, 1).reshape(H, B * n).contiguous()
    return dict(q=q, k=k, lse=lse, ctx=ctx, path=path, count=count,
                w=torch.rand((B, KV, c["cap"]), generator=g, device="cuda") * 4)


def _evict_inputs(c, g):
    """w: weights over several orders of magnitude, a tenth of them 0 (rows just appended, or never looked at). moved: the
    rows' positions are those that earlier evictions leave, in no order but for the newest."""
    dt, B, KV, cap = TORCH[c["dtype"]], c["batch"], c["kv"], c["cap"]
    k, v = (_randn(g, (B, KV, cap, c["dim"]), dt) for _ in range(2))
    ctx = _counts(g, c["low"], cap, B)
    w = torch.exp(2 * torch.randn((B, KV, cap), generator=g, device="cuda"))
    w = w * (torch.rand((B, KV, cap), generator=g, device="cuda") > 0.1)
    pos = tokens = None
    if c["moved"]:
        lost = 1000  # tokens whose rows are gone
        late = torch.minimum(ctx, torch.full_like(ctx, c["recent"] + 16))
        pool = ctx - late + lost
        keys = torch.rand((B, KV, cap + lost), generator=g, device="cuda")
        keys[(torch.arange(cap + lost, device="cuda") >= pool[:, None])[:, None].expand(B, KV, -1)] = 2.0
        row = torch.arange(cap, device="cuda", dtype=torch.int32)
        pos = torch.where((row < (ctx - late)[:, None])[:, None], torch.argsort(keys, -1)[..., :cap].int(),
                          (row + lost)[None, None])
        tokens = ctx + lost
    return dict(k=k, v=v, w=w, ctx=ctx, pos=pos, tokens=tokens)


def prepare(case, seed):
    c, kind = dict(case), case["kind"]
    s = dict(c=c, **{"tree": _tree_inputs, "append": _append_inputs, "weights": _weights_inputs,
                     "evict": _evict_inputs}[kind](c, _gen(seed)))
    dev = dict(device="cuda")
    if kind == "tree":
        s["mask"] = _bits(s["seen"])
        s["o"] = torch.zeros((c["batch"] * c["n"], c["heads"] * c["dim"]), dtype=TORCH[c["dtype"]], **dev)
        s["lse"] = torch.zeros((c["heads"], c["batch"] * c["n"]), **dev)
    elif kind == "append":
        s["ctx_out"], s["tokens_out"] = torch.empty_like(s["ctx"]), torch.empty_like(s["ctx"])
    elif kind == "weights":
        s["w_out"] = torch.zeros_like(s["w"])
    else:
        s["w_out"], s["ctx_out"] = torch.zeros_like(s["w"]), torch.empty_like(s["ctx"])
        s["pos_out"] = torch.zeros(s["w"].shape, dtype=torch.int32, **dev)
    s["plan"] = {}  # the library's argument struct and workspace, made by the first call and kept by the program
    return s


# ---- the plain forms ---------------------------------------------------------------------------------------------


def _groups(q, B, n, KV):
    """[H][B n][D] -> [B][KV][H / KV * n][D] in 32 bits."""
    H, _, D = q.shape
    return q.float().view(KV, H // KV, B, n, D).permute(2, 0, 1, 3, 4).reshape(B, KV, -1, D)


def _tree(s):
    c = s["c"]
    B, n, H, KV, D, cap = (c[x] for x in ("batch", "n", "heads", "kv", "dim", "cap"))
    G = H // KV
    keys, values = (torch.cat([x.float(), d.float().view(KV, B, n, D).transpose(0, 1)], 2)
                    for x, d in ((s["k"], s["kd"]), (s["v"], s["vd"])))
    sc = _groups(s["q"], B, n, KV) @ keys.transpose(2, 3) / math.sqrt(D)
    at, node = torch.arange(cap, device="cuda"), torch.arange(n, device="cuda")
    cached = (at < s["ctx"][:, None])[:, None].expand(B, n, cap)
    drafts = (s["mask"][..., None] >> node & 1).bool() & (node < s["nodes"][:, None])[:, None]
    sees = torch.cat([cached, drafts], 2)[:, None, None]
    sc = sc.view(B, KV, G, n, cap + n).masked_fill(~sees, -math.inf)
    top = sc.amax(-1, keepdim=True)
    top = torch.where(top == -math.inf, 0.0, top)
    p = torch.exp(sc - top)
    total = p.sum(-1, keepdim=True)
    o = (p.view(B, KV, G * n, cap + n) @ values).view(B, KV, G, n, D) / torch.where(total > 0, total, 1.0)
    lse = (top + torch.log(total))[..., 0]
    live = node < s["nodes"][:, None]
    o = torch.where(live[:, :, None], o.permute(0, 3, 1, 2, 4).reshape(B, n, H * D).to(s["o"].dtype),
                    s["o"].view(B, n, H * D))
    lse = torch.where(live[None], lse.permute(1, 2, 0, 3).reshape(H, B, n), s["lse"].view(H, B, n))
    return o.view(B * n, H * D), lse.reshape(H, B * n)


def _append(s):
    c = s["c"]
    B, n, KV, D, cap = (c[x] for x in ("batch", "n", "kv", "dim", "cap"))
    step = torch.arange(n, device="cuda")
    added = torch.minimum(s["count"], cap - s["ctx"])
    live = (step < added[:, None])[:, None]  # [B][1][n]
    at = ((s["ctx"][:, None] + step) % cap).long()[:, None].expand(B, KV, n)
    src = s["path"].long()[:, None, :, None].expand(B, KV, n, D)
    for x, d in ((s["k"], s["kd"]), (s["v"], s["vd"])):
        rows = d.view(KV, B, n, D).transpose(0, 1).gather(2, src)
        to = at[..., None].expand(B, KV, n, D)
        x.scatter_(2, to, torch.where(live[..., None], rows, x.gather(2, to)))
    s["w"].scatter_(2, at, torch.where(live, 0.0, s["w"].gather(2, at)))
    new = (s["tokens"][:, None] + step).int()[:, None].expand(B, KV, n)
    s["pos"].scatter_(2, at, torch.where(live, new, s["pos"].gather(2, at)))
    return s["k"], s["v"], s["w"], s["pos"], s["ctx"] + added, s["tokens"] + added


def _weights(s):
    c = s["c"]
    B, n, H, KV, D, cap = (c[x] for x in ("batch", "n", "heads", "kv", "dim", "cap"))
    G, step = H // KV, torch.arange(c["n"], device="cuda")
    if c["form"] == "step":
        q, lse = s["q"].float().view(B, KV, G, D), s["lse"].view(B, KV, G, 1)
    else:
        q = _groups(s["q"], B, n, KV).view(B, KV, G, n, D)
        lse = s["lse"].view(KV, G, B, n).permute(2, 0, 1, 3)
        if s["path"] is not None:
            at = s["path"].long()[:, None, None].expand(B, KV, G, n)
            q, lse = q.gather(3, at[..., None].expand(B, KV, G, n, D)), lse.gather(3, at)
        q = q.reshape(B, KV, G * n, D)
    count = s["count"] if s["count"] is not None else torch.full_like(s["ctx"], n)
    place = (s["ctx"] - count)[:, None] + step
    key = torch.arange(cap, device="cuda")
    sees = (key <= place[..., None]) & (step < count[:, None])[..., None]  # [B][n][cap]
    sc = (q @ s["k"].float().transpose(2, 3) / math.sqrt(D)).view(B, KV, G, n, cap)
    p = torch.where(sees[:, None, None], torch.exp(sc - lse[..., None]), 0.0)
    got = s["w"] + p.view(B, KV, G * n, cap).sum(2)
    return torch.where((key < s["ctx"][:, None])[:, None], got, s["w_out"])


def _evict(s):
    c = s["c"]
    B, KV, D, cap, budget = (c[x] for x in ("batch", "kv", "dim", "cap", "budget"))
    row = torch.arange(cap, device="cuda", dtype=torch.int32)
    ctx = s["ctx"][:, None, None]
    pos = s["pos"] if s["pos"] is not None else row.expand(B, KV, cap)
    tokens = (s["tokens"] if s["tokens"] is not None else s["ctx"])[:, None, None]
    safe = (pos < c["sinks"]) | (pos >= tokens - c["recent"])
    value = torch.where(safe, math.inf, s["w"]).masked_fill(row >= ctx, -math.inf)
    rank = torch.argsort(torch.argsort(value, dim=-1, descending=True, stable=True), dim=-1)
    kept = (rank < budget) & (row < ctx)
    low = row < torch.clamp(ctx, max=budget)  # rows of the cache afterwards
    hole, source = low & ~kept, kept & (row >= budget)
    # the i-th source goes into the i-th hole
    nth = torch.where(source, source.cumsum(-1) - 1, cap)
    sources = torch.zeros((B, KV, cap + 1), dtype=torch.int64, device="cuda")
    sources.scatter_(2, nth, row.long().expand(B, KV, cap))
    take = torch.where(hole, sources.gather(2, (hole.cumsum(-1) - 1).clamp(min=0)), row.long())[..., :budget]
    for x in (s["k"], s["v"]):
        x[:, :, :budget] = x.gather(2, take[..., None].expand(B, KV, take.shape[2], D))
    for x, y in ((s["w"], s["w_out"]), (pos, s["pos_out"])):
        y[..., :budget] = torch.where(low[..., :budget], x.gather(2, take), y[..., :budget])
    return s["k"], s["v"], s["w_out"], s["pos_out"], torch.clamp(s["ctx"], max=budget)


# ---- the library's calls -----------------------------------------------------------------------------------------


def _own(s):
    M, c, p = _library(), s["c"], s["plan"]
    kind, ws = c["kind"], lambda n: torch.empty(max(n, 16), dtype=torch.uint8, device="cuda")
    if kind == "tree":
        if not p:
            a = M.tree_args(batch=c["batch"], n_draft=c["n"], heads=c["heads"], kv_heads=c["kv"], dim=c["dim"],
                            cap=c["cap"], max_ctx=c["cap"])
            p.update(a=a, ws=ws(M.attn_tree_workspace(a)))
        M.attn_tree(p["a"], s["q"], s["k"], s["v"], s["kd"], s["vd"], s["ctx"], s["o"], p["ws"], n_nodes=s["nodes"],
                    mask=s["mask"], lse=s["lse"])
        return s["o"], s["lse"]
    if kind == "append":
        if not p:
            p["a"] = M.append_args(batch=c["batch"], n_draft=c["n"], kv_heads=c["kv"], dim=c["dim"], cap=c["cap"])
        M.cache_append(p["a"], s["kd"], s["vd"], s["k"], s["v"], s["ctx"], s["ctx_out"], path=s["path"],
                       n_path=s["count"], seen=s["tokens"], seen_out=s["tokens_out"], w=s["w"], pos=s["pos"])
        return s["k"], s["v"], s["w"], s["pos"], s["ctx_out"], s["tokens_out"]
    if kind == "weights":
        if not p:
            a = M.weights_args(batch=c["batch"], n_q=c["n"], heads=c["heads"], kv_heads=c["kv"], dim=c["dim"],
                               cap=c["cap"], max_ctx=c["cap"], decode=c["form"] == "step")
            p.update(a=a, ws=ws(M.cache_weights_workspace(a)))
        M.cache_weights(p["a"], s["q"], s["lse"], s["k"], s["ctx"], s["w_out"], p["ws"], w=s["w"], path=s["path"],
                        n_path=s["count"])
        return s["w_out"]
    if not p:
        a = M.evict_args(batch=c["batch"], kv_heads=c["kv"], dim=c["dim"], cap=c["cap"], max_ctx=c["cap"],
                         budget=c["budget"], recent=c["recent"], sinks=c["sinks"])
        p.update(a=a, ws=ws(M.cache_evict_workspace(a)))
    M.cache_evict(p["a"], s["k"], s["v"], s["w"], s["ctx"], s["w_out"], s["pos_out"], s["ctx_out"], p["ws"],
                  pos=s["pos"], seen=s["tokens"])
    return s["k"], s["v"], s["w_out"], s["pos_out"], s["ctx_out"]


def run(state):
    if own:
        return _own(state)
    return {"tree": _tree, "append": _append, "weights": _weights, "evict": _evict}[state["c"]["kind"]](state)


# ---- what a call cannot do without -------------------------------------------------------------------------------


def work(case):
    c, kind = case, case["kind"]
    B, KV, D = c["batch"], c["kv"], c["dim"]
    if kind == "append":  # a random tree's path is about 1 + ln n long; each row is read and written
        rows = B * (1 + math.log(c["n"]))
        return {"bytes": KV * rows * (8.0 * D + 8) + 20.0 * B, "flops": 0.0}
    keys = B * (c["low"] + c["cap"]) / 2  # contexts uniform over [low, cap]
    if kind == "tree":
        rows = B * c["n"]
        return {"bytes": 4.0 * D * KV * (keys + rows) + rows * (c["heads"] * (4.0 * D + 4) + 8),
                "flops": 4.0 * D * c["heads"] * c["n"] * (keys + B * (1 + math.log(c["n"])))}
    if kind == "weights":
        rows = c["n"] if c["form"] != "path" else 1 + math.log(c["n"])
        pairs = rows * keys - B * rows * (rows - 1) / 2
        return {"bytes": KV * keys * (2.0 * D + 8) + B * rows * c["heads"] * (2.0 * D + 4),
                "flops": 2.0 * D * c["heads"] * pairs}
    low, cap, budget = c["low"], c["cap"], c["budget"]
    n, steps, moved, left = 64, 64, 0.0, 0.0
    for i in range(steps):  # the mean over contexts of the rows that move: the kept ones behind the budget
        n = low + (cap - low) * (i + 0.5) / steps
        late = min(c["recent"], max(0.0, n - budget)) if n > budget else 0.0
        moved += (late + max(0.0, n - budget - late) * max(0.0, budget - c["recent"]) / max(1.0, n - c["recent"])
                  if n > budget else 0.0) / steps
        left += min(n, budget) / steps
    return {"bytes": KV * (keys * (8.0 if c["moved"] else 4.0) + B * (left * 8.0 + moved * 8.0 * D)), "flops": 0.0}


# ---- in 64 bits, from the definitions ----------------------------------------------------------------------------


def _exact_tree(c, x):
    B, n, H, KV, D = (c[k] for k in ("batch", "n", "heads", "kv", "dim"))
    o = torch.zeros((B, n, H, D), dtype=torch.float64, device="cuda")
    lse = torch.zeros((H, B, n), dtype=torch.float64, device="cuda")
    for b in range(B):
        ctx, live = int(x["ctx"][b]), int(x["nodes"][b])
        for h in range(H):
            q = x["q"][h, b * n:b * n + live].double()
            kk, vv = (torch.cat([a[b, h * KV // H, :ctx], d[h * KV // H, b * n:b * n + live]]).double()
                      for a, d in ((x["k"], x["kd"]), (x["v"], x["vd"])))
            sc = torch.matmul(q, kk.t()) * D ** -0.5
            sc[:, ctx:][~x["seen"][b, :live, :live]] = -math.inf
            lse[h, b, :live] = sc.logsumexp(1)
            o[b, :live, h] = torch.softmax(sc, 1) @ vv
    return o.view(B * n, H * D), lse.view(H, B * n)


def _exact_append(c, x):
    n, cap = c["n"], c["cap"]
    ctx, tokens, counts, paths = (x[k].tolist() for k in ("ctx", "tokens", "count", "path"))
    for b in range(c["batch"]):
        for i in range(min(counts[b], cap - ctx[b])):
            for to, of in ((x["k"], x["kd"]), (x["v"], x["vd"])):
                to[b, :, ctx[b] + i] = of[:, b * n + paths[b][i]]
            x["w"][b, :, ctx[b] + i] = 0
            x["pos"][b, :, ctx[b] + i] = tokens[b] + i
    more = [min(counts[b], cap - ctx[b]) for b in range(c["batch"])]
    return (x["k"], x["v"], x["w"].double(), x["pos"], torch.tensor([a + m for a, m in zip(ctx, more)], dtype=torch.int32),
            torch.tensor([a + m for a, m in zip(tokens, more)], dtype=torch.int32))


def _exact_weights(c, x):
    B, n, H, KV, D = (c[k] for k in ("batch", "n", "heads", "kv", "dim"))
    out = torch.zeros((B, KV, c["cap"]), dtype=torch.float64, device="cuda")
    for b in range(B):
        ctx = int(x["ctx"][b])
        rows = torch.arange(n, device="cuda") if x["path"] is None else x["path"][b, :int(x["count"][b])].long()
        m = len(rows)
        hidden = torch.ones((m, ctx), dtype=torch.bool, device="cuda").triu(ctx - m + 1)
        out[b, :, :ctx] = x["w"][b, :, :ctx].double()
        for h in range(H):
            q, l = (x["q"][b, h], x["lse"][b, h]) if c["form"] == "step" else \
                (x["q"][h, b * n + rows], x["lse"][h, b * n + rows])
            sc = torch.matmul(q.double(), x["k"][b, h * KV // H, :ctx].double().t()) * D ** -0.5
            out[b, h * KV // H, :ctx] += torch.exp(sc - l.double()[:, None]).masked_fill(hidden, 0.0).sum(0)
    return out


def _exact_evict(c, x):
    import numpy as np

    KV, budget = c["kv"], c["budget"]
    w_out = np.zeros(x["w"].shape)
    pos_out = np.zeros(x["w"].shape, np.int32)
    w, ctx = x["w"].cpu().numpy().astype(np.float64), x["ctx"].tolist()
    pos = None if x["pos"] is None else x["pos"].cpu().numpy()
    for b in range(c["batch"]):
        n = ctx[b]
        tokens = n if pos is None else int(x["tokens"][b])
        for h in range(KV):
            p = np.arange(n, dtype=np.int32) if pos is None else pos[b, h, :n]
            keep = np.arange(n)
            if n > budget:
                safe = (p < c["sinks"]) | (p >= tokens - c["recent"])
                keep = np.sort(np.lexsort((np.arange(n), -w[b, h, :n], ~safe))[:budget])
            left = np.arange(min(n, budget))
            empty = np.setdiff1d(left, keep)
            left[empty] = keep[keep >= budget]
            at = torch.from_numpy(left).cuda()
            for y in (x["k"], x["v"]):
                y[b, h, :len(left)] = y[b, h, at]
            w_out[b, h, :len(left)], pos_out[b, h, :len(left)] = w[b, h, left], p[left]
    return (x["k"], x["v"], torch.from_numpy(w_out), torch.from_numpy(pos_out),
            torch.tensor([min(n, budget) for n in ctx], dtype=torch.int32))


def exact(case, seed):
    c, g = case, _gen(seed)
    if c["kind"] == "tree":
        return _exact_tree(c, _tree_inputs(c, g))
    if c["kind"] == "append":
        return _exact_append(c, _append_inputs(c, g))
    if c["kind"] == "weights":
        return _exact_weights(c, _weights_inputs(c, g))
    return _exact_evict(c, _evict_inputs(c, g))
