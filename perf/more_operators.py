"""The operators of a cache kept in pages, with the sizes they are timed at: attention of each sequence's new tokens (one,
or a chunk) over its pages, the write of their rows, the reservation of pages for them (with the copy of a last page that
others hold too), the fork of sequences with the release of what nobody holds any more, and the compaction of the pool.

Each case is one call on resident tensors. With `own` false the operator is computed from elementary torch operations, its
arithmetic in 32 bits; with `own` true by the library's kernels through the public binding (mako-common_amd/mako_attn.py).
Pages hold `page` rows of every kv head: k and v [layers][pages][kv][page][dim] (attention and write: one layer). A
sequence's pages are a row of a table; -1 is no page. refs counts the holders of each page, 0 for a free one.
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
        # one token early in a chat with a small model: latency
        dict(name="paged_small", kind="attn", steps=1, chunks=0, new=1, heads=16, kv=8, dim=128, low=391, high=391,
             page=64, dtype="f16"),
        # a decode step of a serving batch with mixed contexts
        dict(name="paged_step", kind="attn", steps=16, chunks=0, new=1, heads=32, kv=8, dim=128, low=1024, high=32767,
             page=64, dtype="f16"),
        # a step that carries decoding sequences and two chunks of prompts, odd sizes
        dict(name="paged_mixed", kind="attn", steps=11, chunks=2, new=1333, heads=32, kv=8, dim=128, low=500,
             high=12001, page=128, dtype="bf16"),
        # chunks on the gated-attention layers' heads of 256
        dict(name="paged_d256", kind="attn", steps=0, chunks=4, new=300, heads=16, kv=2, dim=256, low=8000,
             high=16000, page=64, dtype="bf16"),
        # the rows of a decode step in a serving batch
        dict(name="write_step", kind="write", steps=64, chunks=0, new=1, kv=8, dim=128, low=100, high=1000, page=64,
             dtype="bf16"),
        # the rows of a long prompt beside some decoding sequences
        dict(name="write_prompt", kind="write", steps=7, chunks=1, new=4096, kv=8, dim=128, low=100, high=1000,
             page=64, dtype="f16"),
        # a decode step's pages in a serving batch: most last pages have room
        dict(name="reserve_step", kind="reserve", steps=64, chunks=0, new=1, kv=8, dim=128, low=100, high=2000, page=64,
             pages=4096, layers=0, beams=1, dtype="bf16"),
        # the step after a fork: the beams of a prompt share their last page, which is copied in each layer
        dict(name="reserve_beams", kind="reserve", steps=64, chunks=0, new=1, kv=8, dim=128, low=100, high=2000,
             page=64, pages=1024, layers=2, beams=4, dtype="bf16"),
        # a step of beam search: each sequence goes on from one of its prompt's beams
        dict(name="fork_beams", kind="fork", batch=64, low=100, high=2000, page=64, pages=4096, beams=4),
        # a large batch of long sequences: some end, some go on from others, some are cut back
        dict(name="fork_batch", kind="fork", batch=1024, low=100, high=8192, page=64, pages=65536, beams=1),
        # a small pool with holes between its pages
        dict(name="compact_small", kind="compact", batch=16, kv=8, dim=128, low=100, high=1000, page=64, pages=512,
             layers=1, dtype="bf16"),
        # a pool of several layers, half of it in use
        dict(name="compact_pool", kind="compact", batch=128, kv=8, dim=128, low=100, high=2000, page=64, pages=4096,
             layers=2, dtype="f16"),
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    kind = rng.choice(["attn", "attn", "attn", "attn", "write", "reserve", "fork", "compact"])
    dtype = rng.choice(["f16", "bf16"])
    heads, kv, dim = rng.choice([(32, 8, 128), (16, 8, 128), (8, 2, 128), (16, 16, 64), (16, 2, 256)])
    page = rng.choice([64, 64, 128, 256])
    if kind == "attn":
        form = rng.choice(["step", "chunk", "mixed"])
        steps = 0 if form == "chunk" else _log(rng, 1, 32)
        chunks = 0 if form == "step" else _log(rng, 1, 6)
        new = 1 if form == "step" else _log(rng, 2, 2048)
        high = _log(rng, 16, 32767)
        high = max(16, min(high, 16 * 8 * 128 * 32768 // ((steps + chunks) * kv * dim)))
        if chunks:  # at most about the operations of the largest listed case
            new = max(2, min(new, int(2.2e11 / (chunks * heads * dim * 4 * (high + 64)))))
        return dict(kind=kind, steps=steps, chunks=chunks, new=new, heads=heads, kv=kv, dim=dim,
                    low=rng.choice([high, max(1, high // 2), max(1, high // 32)]), high=high, page=page, dtype=dtype)
    high = _log(rng, 16, 4096)
    low = rng.choice([high, max(1, high // 2), max(1, high // 32)])
    if kind in ("write", "reserve"):
        steps, chunks = rng.choice([(_log(rng, 1, 128), 0), (0, 1), (_log(rng, 1, 32), _log(rng, 1, 4))])
        new = _log(rng, 2, 2048) if chunks else 1
        c = dict(kind=kind, steps=steps, chunks=chunks, new=new, kv=kv, dim=dim, low=low, high=high, page=page,
                 dtype=dtype)
        if kind == "write":
            c["high"] = max(16, min(high, 100000 // (steps + chunks)))
            c["low"] = min(low, c["high"])
            return c
        c["beams"] = rng.choice([1, 1, 2, 4])
        need = (steps + chunks) * (high + new + 2 * page) // page + 64
        c["layers"] = 0 if need * page * kv * dim > 1 << 27 else rng.choice([0, 1, 2])
        c["pages"] = need + _log(rng, 1, 4096 if c["layers"] == 0 else need)
        return c
    batch = _log(rng, 1, 512)
    if kind == "fork":
        need = batch * (high // page + 2)
        return dict(kind=kind, batch=batch, low=low, high=high, page=page, pages=need + _log(rng, 1, 4096),
                    beams=rng.choice([1, 2, 4]))
    high = max(16, min(high, 128 * 2000 * 8 * 128 // (batch * kv * dim)))
    need = batch * (high // page + 2)
    return dict(kind=kind, batch=batch, kv=kv, dim=dim, low=min(low, high), high=high, page=page,
                pages=need + _log(rng, 1, max(2, need)), layers=1, dtype=dtype)


# ---- inputs ------------------------------------------------------------------------------------------------------


def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _randn(g, shape, dtype):
    """Unit-normal values, as the per-head RMS norms of q and k give them."""
    return torch.randn(shape, generator=g, device="cuda", dtype=torch.float32).to(dtype)


def _ints(g, low, high, n):
    return torch.randint(low, high + 1, (n,), generator=g, device="cuda", dtype=torch.int32)


def _up(x, page):
    return (x + page - 1) // page


def _lengths(c, g):
    """new rows and rows before them of each sequence, the decoding ones first, as a program knows them on both sides."""
    steps, chunks = c["steps"], c["chunks"]
    new = torch.cat([torch.ones(steps, dtype=torch.int32, device="cuda"),
                     _ints(g, max(1, c["new"] // 2), c["new"], chunks)])
    ctx = _ints(g, c["low"], c["high"], steps + chunks)
    starts = torch.zeros(steps + chunks + 1, dtype=torch.int32, device="cuda")
    starts[1:] = torch.cumsum(new, 0)
    return ctx, None if chunks == 0 else starts, new


def _max_pages(c):
    return _up(c["high"] + c.get("new", 0), c["page"])


def _tables(g, held, max_pages, pages):
    """Tables of `held` pages a sequence, anywhere in the pool, as earlier sequences have left it."""
    b = held.shape[0]
    order = torch.randperm(pages, generator=g, device="cuda").int()
    at = torch.arange(max_pages, device="cuda")[None] < held[:, None]
    nth = torch.cumsum(at.reshape(-1).int(), 0).view(b, max_pages) - 1
    return torch.where(at, order[nth.clamp(0, pages - 1)], -1)


def _refs(table, pages):
    bins = torch.zeros(pages + 1, dtype=torch.int32, device="cuda")
    return bins.index_add_(0, torch.where(table < 0, pages, table).reshape(-1).long(),
                           torch.ones(table.numel(), dtype=torch.int32, device="cuda"))[:pages].contiguous()


def _attn_inputs(c, g):
    dt, D, page = TORCH[c["dtype"]], c["dim"], c["page"]
    B, rows = c["steps"] + c["chunks"], c["steps"] + c["chunks"] * c["new"]
    ctx, starts, new = _lengths(c, g)
    pages = B * _max_pages(c) + 3
    return dict(q=_randn(g, (c["heads"], rows, D), dt), k=_randn(g, (pages, c["kv"], page, D), dt),
                v=_randn(g, (pages, c["kv"], page, D), dt), ctx=ctx, starts=starts, new=new,
                table=_tables(g, _up(ctx + new, page), _max_pages(c), pages))


def _write_inputs(c, g):
    dt, D, page = TORCH[c["dtype"]], c["dim"], c["page"]
    B, rows = c["steps"] + c["chunks"], c["steps"] + c["chunks"] * c["new"]
    ctx, starts, new = _lengths(c, g)
    pages = B * _max_pages(c) + 3
    kd, vd = (_randn(g, (c["kv"], rows, D), dt) for _ in range(2))
    k, v = (_randn(g, (pages, c["kv"], page, D), dt) for _ in range(2))
    return dict(kd=kd, vd=vd, k=k, v=v, ctx=ctx, starts=starts, new=new,
                table=_tables(g, _up(ctx + new, page), _max_pages(c), pages))


def _shared(c, g, batch, max_pages):
    """Tables whose sequences come in sets of `beams` that hold the same pages, the rows of each set alike."""
    ctx = _ints(g, c["low"], c["high"], batch)
    lead = torch.arange(batch, device="cuda") // c["beams"] * c["beams"]
    ctx = ctx[lead].contiguous()
    held = torch.where(lead == torch.arange(batch, device="cuda"), _up(ctx, c["page"]), 0)
    table = _tables(g, held, max_pages, c["pages"])[lead].contiguous()
    return ctx, table, _refs(table, c["pages"])


def _reserve_inputs(c, g):
    B = c["steps"] + c["chunks"]
    _, starts, new = _lengths(c, g)
    ctx, table, refs = _shared(c, g, B, _max_pages(c))
    k = v = None
    if c["layers"]:
        shape = (c["layers"], c["pages"], c["kv"], c["page"], c["dim"])
        k, v = (_randn(g, shape, TORCH[c["dtype"]]) for _ in range(2))
    return dict(k=k, v=v, ctx=ctx, starts=starts, new=new, table=table, refs=refs)


def _fork_inputs(c, g):
    """beams > 1: each sequence goes on from a beam of its set; else one in eight ends, one in eight goes on from another,
    one in eight is cut back."""
    B = c["batch"]
    ctx, table, refs = _shared(c, g, B, _max_pages(c))
    i = torch.arange(B, device="cuda", dtype=torch.int32)
    if c["beams"] > 1:
        parent = (i // c["beams"] * c["beams"] + _ints(g, 0, c["beams"] - 1, B)).clamp(max=B - 1)
        return dict(ctx=ctx, table=table, refs=refs, parent=parent.int(), keep=ctx[parent.long()].contiguous())
    what = _ints(g, 0, 7, B)
    parent = torch.where(what == 0, -1, torch.where(what == 1, _ints(g, 0, B - 1, B), i)).int()
    keep = torch.where(what == 2, ctx // 2, ctx[parent.long().clamp(min=0)])
    return dict(ctx=ctx, table=table, refs=refs, parent=parent, keep=keep.int())


def _compact_inputs(c, g):
    ctx = _ints(g, c["low"], c["high"], c["batch"])
    table = _tables(g, _up(ctx, c["page"]), _max_pages(c), c["pages"])
    shape = (c["layers"], c["pages"], c["kv"], c["page"], c["dim"])
    k, v = (_randn(g, shape, TORCH[c["dtype"]]) for _ in range(2))
    return dict(k=k, v=v, table=table, refs=_refs(table, c["pages"]))


INPUTS = {"attn": _attn_inputs, "write": _write_inputs, "reserve": _reserve_inputs, "fork": _fork_inputs,
          "compact": _compact_inputs}


def prepare(case, seed):
    c = dict(case)
    s = dict(c=c, plan={}, **INPUTS[c["kind"]](c, _gen(seed)))
    dev = dict(device="cuda")
    if c["kind"] == "attn":
        rows = s["q"].shape[1]
        s["host"] = s["ctx"].tolist(), s["new"].tolist()
        s["o"] = torch.zeros((rows, c["heads"] * c["dim"]), dtype=TORCH[c["dtype"]], **dev)
        s["lse"] = torch.zeros((c["heads"], rows), **dev)
    elif c["kind"] != "write":
        s["table_out"], s["refs_out"] = torch.empty_like(s["table"]), torch.empty_like(s["refs"])
        s["ctx_out"] = torch.empty_like(s["ctx"]) if "ctx" in s else None
        s["used"] = torch.empty(1, dtype=torch.int32, **dev)
    return s


# ---- the plain forms ---------------------------------------------------------------------------------------------


def _attn(s):
    c = s["c"]
    H, KV, D, page = c["heads"], c["kv"], c["dim"], c["page"]
    G, row = H // KV, 0
    o, lse = s["o"].clone(), s["lse"].clone()
    for b, (ctx, n) in enumerate(zip(*s["host"])):
        at = s["table"][b, :_up(ctx + n, page)].long()
        q = s["q"][:, row:row + n].float().view(KV, G * n, D)
        k, v = (x[at].transpose(0, 1).reshape(KV, -1, D)[:, :ctx + n].float() for x in (s["k"], s["v"]))
        hidden = torch.arange(ctx + n, device="cuda") > ctx + torch.arange(n, device="cuda")[:, None]
        for h in range(KV):  # a kv head at a time: the scores of a long chunk are large
            sc = (q[h] @ k[h].t() / math.sqrt(D)).view(G, n, -1).masked_fill(hidden, -math.inf)
            top = sc.amax(-1, keepdim=True)
            p = torch.exp(sc - top)
            total = p.sum(-1, keepdim=True)
            out = (p.view(G * n, -1) @ v[h]).view(G, n, D) / total
            o[row:row + n, h * G * D:(h + 1) * G * D] = out.transpose(0, 1).reshape(n, G * D).to(o.dtype)
            lse[h * G:(h + 1) * G, row:row + n] = (top + torch.log(total))[..., 0]
        row += n
    return o, lse


def _row_places(s):
    """The sequence, page and row in it of each new row (rows behind the last sequence: a sequence of -1)."""
    rows = s["kd"].shape[1]
    r = torch.arange(rows, device="cuda")
    if s["starts"] is None:
        b, i = r, torch.zeros_like(r)
    else:
        b = torch.searchsorted(s["starts"].long(), r, right=True) - 1
        i = r - s["starts"].long()[b]
    live = b < s["ctx"].shape[0]
    b = b.clamp(max=s["ctx"].shape[0] - 1)
    at = s["ctx"].long()[b] + i
    page = s["c"]["page"]
    entry = s["table"].long()[b, (at // page).clamp(max=s["table"].shape[1] - 1)]
    return live & (entry >= 0), entry.clamp(min=0), at % page


def _write(s):
    live, entry, row = _row_places(s)
    # rows of no sequence are sent where a row of the first one goes, with its value
    entry, row = (torch.where(live, x, x[0]) for x in (entry, row))
    for x, d in ((s["k"], s["kd"]), (s["v"], s["vd"])):
        d = torch.where(live[None, :, None], d, d[:, :1])
        x[entry, :, row] = d.transpose(0, 1)
    return s["k"], s["v"]


def _reserve(s):
    c = s["c"]
    page, table, refs = c["page"], s["table"], s["refs"]
    B, MP = table.shape
    ctx = s["ctx"].long()
    end = torch.clamp(ctx + s["new"], max=MP * page)
    first, last = ctx // page, _up(end, page)
    j = torch.arange(MP, device="cuda")
    window = (j >= first[:, None]) & (j < last[:, None])
    held = table.long().gather(1, first.clamp(max=MP - 1)[:, None])[:, 0]
    part = (end > ctx) & (ctx % page != 0) & (held >= 0)  # appends to a page that it holds
    i = torch.arange(B, device="cuda")
    rank = ((held[None] == held[:, None]) & part[None] & (i[None] < i[:, None])).sum(1)
    copies = part & (refs.long()[held.clamp(min=0)] - rank > 1)
    need = window & ((table < 0) | (copies[:, None] & (j == first[:, None])))
    nth = torch.cumsum(need.reshape(-1).long(), 0).view(B, MP) - 1
    free = refs == 0
    places = torch.where(free, torch.cumsum(free.long(), 0) - 1, c["pages"])
    pool = torch.zeros(c["pages"] + 1, dtype=torch.int64, device="cuda")
    pool.scatter_(0, places, torch.arange(c["pages"], device="cuda"))
    got = need & (nth < free.sum())
    table_out = torch.where(got, pool[nth.clamp(0, c["pages"])].int(), table)
    bins = torch.cat([refs, refs.new_zeros(1)])
    one = torch.ones_like(table).reshape(-1)
    bins.index_add_(0, torch.where(got, table_out.long(), c["pages"]).reshape(-1), one)
    left = got & (table >= 0)  # entries whose page is left to the others
    bins.index_add_(0, torch.where(left, table.long(), c["pages"]).reshape(-1), -one)
    short = torch.where(need & ~got, j[None] * page, MP * page).amin(1)
    ctx_out = torch.minimum(end, torch.maximum(ctx, short)).int()
    if c["layers"]:
        # each copying sequence's last page into its new one; the others' onto itself
        src = table.long().gather(1, (_up(ctx, page) - 1).clamp(min=0)[:, None])[:, 0].clamp(min=0)
        copied = left.any(1)
        dst = torch.where(copied, table_out.long().gather(1, first.clamp(max=MP - 1)[:, None])[:, 0], src)
        rows = torch.arange(page, device="cuda") < torch.where(copied, ctx % page, 0)[:, None]
        for x in (s["k"], s["v"]):
            x[:, dst] = torch.where(rows[None, :, None, :, None], x[:, src], x[:, dst])
    return s["k"], s["v"], table_out, bins[:c["pages"]], ctx_out


def _fork(s):
    c = s["c"]
    page, table = c["page"], s["table"]
    B, MP = table.shape
    alive = (s["parent"] >= 0) & (s["parent"] < B)
    src = s["parent"].long().clamp(0, B - 1)
    ctx_out = torch.where(alive, torch.minimum(s["keep"], s["ctx"][src]), 0).int()
    j = torch.arange(MP, device="cuda")
    table_out = torch.where(j < _up(ctx_out, page)[:, None], table[src], -1)
    bins = torch.cat([s["refs"], s["refs"].new_zeros(1)])
    one = torch.ones_like(table).reshape(-1)
    for t, sign in ((table_out, 1), (table, -1)):
        bins.index_add_(0, torch.where(t < 0, c["pages"], t).reshape(-1).long(), sign * one)
    return table_out, bins[:c["pages"]], ctx_out


def _compact(s):
    c = s["c"]
    pages, refs = c["pages"], s["refs"]
    at = torch.arange(pages, device="cuda")
    used = refs > 0
    left = used.sum()
    hole, source = ~used & (at < left), used & (at >= left)
    sources, holes = (torch.zeros(pages + 1, dtype=torch.int64, device="cuda").scatter_(
        0, torch.where(x, torch.cumsum(x.long(), 0) - 1, pages), at) for x in (source, hole))
    take = torch.where(hole, sources[(torch.cumsum(hole.long(), 0) - 1).clamp(min=0)], at)
    number = torch.where(source, holes[(torch.cumsum(source.long(), 0) - 1).clamp(min=0)], at)
    table_out = torch.where(s["table"] < 0, -1, number[s["table"].long().clamp(min=0)].int())
    refs_out = torch.where(at < left, refs[take], 0)
    for x in (s["k"], s["v"]):
        x.copy_(x[:, take])
    return s["k"], s["v"], table_out, refs_out, left.int().view(1)


# ---- the library's calls -----------------------------------------------------------------------------------------


def _own(s):
    M, c, p = _library(), s["c"], s["plan"]
    kind, ws = c["kind"], lambda n: torch.empty(max(n, 16), dtype=torch.uint8, device="cuda")
    if kind == "attn":
        if not p:
            a = M.paged_args(batch=c["steps"] + c["chunks"], rows=s["q"].shape[1], heads=c["heads"], kv_heads=c["kv"],
                             dim=c["dim"], pages=s["k"].shape[0], page=c["page"], max_pages=s["table"].shape[1],
                             max_new=c["new"], max_ctx=c["high"] + c["new"])
            p.update(a=a, ws=ws(M.attn_paged_workspace(a)))
        M.attn_paged(p["a"], s["q"], s["k"], s["v"], s["table"], s["ctx"], s["o"], p["ws"], starts=s["starts"],
                     lse=s["lse"])
        return s["o"], s["lse"]
    if not p:
        table = s["table"]
        rows = c["steps"] + c["chunks"] * c["new"] if "steps" in c else 0
        a = M.pages_args(batch=table.shape[0], rows=rows, pages=c["pages"] if "pages" in c else s["k"].shape[0],
                         page=c["page"], max_pages=table.shape[1], kv_heads=c.get("kv", 0), dim=c.get("dim", 0),
                         layers=c.get("layers", 1))
        p.update(a=a)
        if kind in ("reserve", "compact"):
            p.update(ws=ws({"reserve": M.pages_reserve_workspace, "compact": M.pages_compact_workspace}[kind](a)))
    if kind == "write":
        M.pages_write(p["a"], s["kd"], s["vd"], s["k"], s["v"], s["table"], s["ctx"], starts=s["starts"])
        return s["k"], s["v"]
    if kind == "reserve":
        M.pages_reserve(p["a"], s["k"], s["v"], s["table"], s["refs"], s["ctx"], s["table_out"], s["refs_out"],
                        s["ctx_out"], p["ws"], starts=s["starts"])
        return s["k"], s["v"], s["table_out"], s["refs_out"], s["ctx_out"]
    if kind == "fork":
        M.pages_fork(p["a"], s["table"], s["refs"], s["ctx"], s["table_out"], s["refs_out"], s["ctx_out"],
                     parent=s["parent"], keep=s["keep"])
        return s["table_out"], s["refs_out"], s["ctx_out"]
    M.pages_compact(p["a"], s["k"], s["v"], s["table"], s["refs"], s["table_out"], s["refs_out"], s["used"], p["ws"])
    return s["k"], s["v"], s["table_out"], s["refs_out"], s["used"]


def run(state):
    if own:
        return _own(state)
    return {"attn": _attn, "write": _write, "reserve": _reserve, "fork": _fork,
            "compact": _compact}[state["c"]["kind"]](state)


# ---- what a call cannot do without -------------------------------------------------------------------------------


def work(case):
    c, kind = case, case["kind"]
    page, ctx = c["page"], (c["low"] + c["high"]) / 2  # contexts uniform over [low, high]
    if kind in ("attn", "write"):
        chunk = (max(1, c["new"] // 2) + c["new"]) / 2
        rows = c["steps"] + c["chunks"] * chunk
        if kind == "write":
            return {"bytes": rows * c["kv"] * c["dim"] * 8.0, "flops": 0.0}
        D, H = c["dim"], c["heads"]
        keys = (c["steps"] + c["chunks"]) * ctx + rows
        pairs = c["steps"] * (ctx + 1) + c["chunks"] * chunk * (ctx + chunk / 2)
        return {"bytes": 4.0 * D * c["kv"] * keys + rows * H * (4.0 * D + 4), "flops": 4.0 * D * H * pairs}
    batch = c.get("batch", c.get("steps", 0) + c.get("chunks", 0))
    tables = 8.0 * batch * _max_pages(c) + 8.0 * c["pages"] + 12.0 * batch
    if kind == "fork":
        return {"bytes": tables, "flops": 0.0}
    row = 4.0 * c["kv"] * c["dim"] * max(1, c["layers"])  # a row of k and v
    if kind == "reserve":
        copies = batch * (c["beams"] - 1) / c["beams"] * (page - 1) / page if c["layers"] else 0.0
        return {"bytes": tables + copies * page / 2 * row * 2, "flops": 0.0}
    used = batch * (ctx / page + 0.5)
    moved = used * max(0.0, 1 - used / c["pages"])
    return {"bytes": tables + moved * page * row * 2, "flops": 0.0}


# ---- in 64 bits, from the definitions ----------------------------------------------------------------------------


def _exact_attn(c, x):
    H, KV, D, page = c["heads"], c["kv"], c["dim"], c["page"]
    rows = x["q"].shape[1]
    o = torch.zeros((rows, H, D), dtype=torch.float64, device="cuda")
    lse = torch.zeros((H, rows), dtype=torch.float64, device="cuda")
    row = 0
    for b, (ctx, n) in enumerate(zip(x["ctx"].tolist(), x["new"].tolist())):
        own_pages = [p for p in x["table"][b].tolist() if p >= 0]
        sees = torch.ones((n, ctx + n), dtype=torch.bool, device="cuda").tril(ctx)
        for h in range(KV):
            k, v = (torch.cat([t[p, h] for p in own_pages])[:ctx + n].double() for t in (x["k"], x["v"]))
            for g in range(h * H // KV, (h + 1) * H // KV):
                sc = torch.matmul(x["q"][g, row:row + n].double(), k.t()) * D ** -0.5
                sc[~sees] = -math.inf
                lse[g, row:row + n] = sc.logsumexp(1)
                o[row:row + n, g] = torch.softmax(sc, 1) @ v
        row += n
    return o.view(rows, H * D), lse


def _exact_write(c, x):
    row = 0
    for b, (ctx, n) in enumerate(zip(x["ctx"].tolist(), x["new"].tolist())):
        t, i = x["table"][b].tolist(), 0
        while i < n:
            at = ctx + i
            m = min(n - i, c["page"] - at % c["page"])
            for to, of in ((x["k"], x["kd"]), (x["v"], x["vd"])):
                to[t[at // c["page"]], :, at % c["page"]:at % c["page"] + m] = of[:, row + i:row + i + m]
            i += m
        row += n
    return x["k"], x["v"]


def _exact_reserve(c, x):
    page, refs, table = c["page"], x["refs"].tolist(), x["table"].tolist()
    free = [p for p, r in enumerate(refs) if r == 0][::-1]
    ctx_out = []
    for b, (ctx, n) in enumerate(zip(x["ctx"].tolist(), x["new"].tolist())):
        end, at = min(ctx + n, page * len(table[b])), ctx
        while at < end:
            j = at // page
            p, keeps = table[b][j], at % page
            shared = p >= 0 and keeps and refs[p] > 1
            if p < 0 or shared:
                if not free:
                    break
                new = free.pop()
                refs[new] = 1
                table[b][j] = new
                if shared:
                    refs[p] -= 1
                    for t in (x["k"], x["v"]):
                        if t is not None:
                            t[:, new, :, :keeps] = t[:, p, :, :keeps]
            at = min(end, (j + 1) * page)
        ctx_out.append(at)
    return x["k"], x["v"], *(torch.tensor(y, dtype=torch.int32) for y in (table, refs, ctx_out))


def _exact_fork(c, x):
    import numpy as np

    table, ctx, refs = x["table"].cpu().numpy(), x["ctx"].tolist(), x["refs"].cpu().numpy().copy()
    out, ctx_out = np.full_like(table, -1), []
    for i, (p, keep) in enumerate(zip(x["parent"].tolist(), x["keep"].tolist())):
        rows = min(keep, ctx[p]) if 0 <= p < len(ctx) else 0
        n = -(-rows // c["page"])
        out[i, :n] = table[p, :n]
        ctx_out.append(rows)
        np.add.at(refs, out[i, :n], 1)
        np.subtract.at(refs, table[i][table[i] >= 0], 1)
    return torch.from_numpy(out), torch.from_numpy(refs), torch.tensor(ctx_out, dtype=torch.int32)


def _exact_compact(c, x):
    refs, table = x["refs"].tolist(), x["table"].cpu()
    number = list(range(c["pages"]))
    used = sum(r > 0 for r in refs)
    holes = [p for p in range(used) if refs[p] == 0]
    sources = [p for p in range(used, c["pages"]) if refs[p] > 0]
    for hole, source in zip(holes, sources):
        number[source], refs[hole], refs[source] = hole, refs[source], 0
    to, of = torch.tensor(holes, device="cuda"), torch.tensor(sources, device="cuda")
    for t in (x["k"], x["v"]):
        if holes:
            t[:, to] = t[:, of]
    renamed = torch.tensor(number + [-1], dtype=torch.int32)[table.long()]
    return x["k"], x["v"], renamed, torch.tensor(refs, dtype=torch.int32), torch.tensor([used], dtype=torch.int32)


def exact(case, seed):
    x = INPUTS[case["kind"]](case, _gen(seed))
    return {"attn": _exact_attn, "write": _exact_write, "reserve": _exact_reserve, "fork": _exact_fork,
            "compact": _exact_compact}[case["kind"]](case, x)
