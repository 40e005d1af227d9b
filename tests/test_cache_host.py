"""The cache operators' host side without a GPU: what they refuse, and with which message, before touching the device; and
with a HIP runtime that runs nothing, their workspaces and launches."""
import ctypes
import re

import pytest

torch = pytest.importorskip("torch")

import mako_attn as M  # noqa: E402
from test_host_paths import events, hip, launches, tensor  # noqa: E402, F401

FAKE = ctypes.c_void_p(0x10000)  # aligned, never dereferenced: every call below fails validation first
ODD = ctypes.c_void_p(0x10008)
BIG = ctypes.c_size_t(1 << 40)


def struct(cls, base, kw):
    a = dict(base, **{f: kw.pop(f) for f, _ in cls._fields_ if f in kw})
    return ctypes.byref(cls(*[a[f] for f, _ in cls._fields_]))


def answer(rc):
    return rc, M.lib().mako_last_error().decode()


def tree_rc(**kw):
    a = struct(M.TreeArgs, dict(batch=2, n_draft=8, q_pad=16, d_pad=16, heads=8, kv_heads=2, dim=128, cap=256, max_ctx=256,
                                width=1024, scale=0.088), kw)
    p = dict(in_=M.BF16, out=M.BF16, q=FAKE, k=FAKE, v=FAKE, kd=FAKE, vd=FAKE, ctx=FAKE, nodes=None, mask=None, o=FAKE,
             ws=FAKE, bytes=BIG)
    p.update(kw)
    return answer(M.lib().mako_attn_tree(a, p["in_"], p["out"], p["q"], p["k"], p["v"], p["kd"], p["vd"], p["ctx"],
                                         p["nodes"], p["mask"], p["o"], None, p["ws"], p["bytes"], None))


@pytest.mark.parametrize("kw,code,msg", [
    (dict(dim=96), M.EUNSUPPORTED, "heads of 96"),
    (dict(in_=M.F32), M.EUNSUPPORTED, "input type"),
    (dict(out=M.F16), M.EUNSUPPORTED, "output type"),
    (dict(heads=7), M.EINVAL, "over 2 kv heads"),
    (dict(kv_heads=0), M.EINVAL, "over 0 kv heads"),
    (dict(n_draft=65, q_pad=200, d_pad=200), M.EINVAL, "65 drafts"),
    (dict(q_pad=15), M.EINVAL, "draft rows"),
    (dict(d_pad=15), M.EINVAL, "draft rows"),
    (dict(max_ctx=257), M.EINVAL, "max_ctx"),
    (dict(cap=1 << 23, max_ctx=1), M.EINVAL, "2 GiB"),
    (dict(batch=1 << 26, n_draft=1, q_pad=1 << 31, d_pad=1 << 31, heads=64, kv_heads=2), M.EINVAL, "exceed"),
    (dict(width=1020), M.EINVAL, "o rows"),
    (dict(width=1026), M.EINVAL, "o rows"),
    (dict(scale=0.0), M.EINVAL, "scale"),
    (dict(scale=float("nan")), M.EINVAL, "scale"),
    (dict(q=None), M.EINVAL, "null"),
    (dict(vd=None), M.EINVAL, "null"),
    (dict(ctx=None), M.EINVAL, "null"),
    (dict(kd=ODD), M.EINVAL, "aligned"),
    (dict(o=ODD), M.EINVAL, "aligned"),
    (dict(mask=ctypes.c_void_p(0x10004)), M.EINVAL, "mask"),
])
def test_tree_refuses(kw, code, msg):
    rc, err = tree_rc(**kw)
    assert rc == code and msg in err and err.startswith("attention_tree"), (rc, err)


def append_rc(**kw):
    a = struct(M.AppendArgs, dict(batch=2, n_draft=8, d_pad=16, kv_heads=2, dim=128, cap=256), kw)
    p = dict(in_=M.BF16, kd=FAKE, vd=FAKE, ctx=FAKE, ctx_out=FAKE, seen=FAKE, seen_out=FAKE, w=FAKE, pos=FAKE, k=FAKE,
             v=FAKE)
    p.update(kw)
    return answer(M.lib().mako_cache_append(a, p["in_"], p["kd"], p["vd"], None, None, p["ctx"], p["ctx_out"], p["seen"],
                                            p["seen_out"], p["w"], p["pos"], p["k"], p["v"], None))


@pytest.mark.parametrize("kw,code,msg", [
    (dict(dim=32), M.EUNSUPPORTED, "heads of 32"),
    (dict(in_=M.F32), M.EUNSUPPORTED, "input type"),
    (dict(kv_heads=0), M.EINVAL, "no kv heads"),
    (dict(d_pad=15), M.EINVAL, "draft rows"),
    (dict(cap=1 << 23), M.EINVAL, "2 GiB"),
    (dict(kd=None), M.EINVAL, "null"),
    (dict(ctx_out=None), M.EINVAL, "null"),
    (dict(seen=None), M.EINVAL, "need seen"),
    (dict(seen=None, pos=None), M.EINVAL, "need seen"),
    (dict(v=ODD), M.EINVAL, "aligned"),
])
def test_append_refuses(kw, code, msg):
    rc, err = append_rc(**kw)
    assert rc == code and msg in err and err.startswith("cache_append"), (rc, err)


def weights_rc(**kw):
    a = struct(M.WeightsArgs, dict(batch=2, n_q=8, q_pad=16, heads=8, kv_heads=2, dim=128, cap=256, max_ctx=256,
                                   scale=0.088, decay=1.0), kw)
    p = dict(in_=M.BF16, q=FAKE, lse=FAKE, k=FAKE, ctx=FAKE, w=FAKE, w_out=FAKE, ws=FAKE, bytes=BIG)
    p.update(kw)
    return answer(M.lib().mako_cache_weights(a, p["in_"], p["q"], p["lse"], p["k"], p["ctx"], None, None, p["w"],
                                             p["w_out"], p["ws"], p["bytes"], None))


@pytest.mark.parametrize("kw,code,msg", [
    (dict(dim=72), M.EUNSUPPORTED, "heads of 72"),
    (dict(in_=M.F32), M.EUNSUPPORTED, "input type"),
    (dict(heads=9), M.EINVAL, "kv heads"),
    (dict(q_pad=15), M.EINVAL, "queries in heads"),
    (dict(max_ctx=300), M.EINVAL, "max_ctx"),
    (dict(cap=1 << 23, max_ctx=1), M.EINVAL, "2 GiB"),
    (dict(scale=float("inf")), M.EINVAL, "scale"),
    (dict(decay=-1.0), M.EINVAL, "decay"),
    (dict(decay=float("nan")), M.EINVAL, "decay"),
    (dict(lse=None), M.EINVAL, "null"),
    (dict(w_out=None), M.EINVAL, "null"),
    (dict(q=ODD), M.EINVAL, "aligned"),
])
def test_weights_refuses(kw, code, msg):
    rc, err = weights_rc(**kw)
    assert rc == code and msg in err and err.startswith("cache_weights"), (rc, err)


def evict_rc(**kw):
    a = struct(M.EvictArgs, dict(batch=2, kv_heads=2, dim=128, cap=256, max_ctx=256, budget=64, recent=8, sinks=4), kw)
    p = dict(in_=M.BF16, k=FAKE, v=FAKE, w=FAKE, pos=FAKE, seen=FAKE, ctx=FAKE, w_out=FAKE, pos_out=FAKE, ctx_out=FAKE,
             ws=FAKE, bytes=BIG)
    p.update(kw)
    return answer(M.lib().mako_cache_evict(a, p["in_"], p["k"], p["v"], p["w"], p["pos"], p["seen"], p["ctx"],
                                           p["w_out"], p["pos_out"], p["ctx_out"], p["ws"], p["bytes"], None))


@pytest.mark.parametrize("kw,code,msg", [
    (dict(dim=512), M.EUNSUPPORTED, "heads of 512"),
    (dict(in_=M.F32), M.EUNSUPPORTED, "input type"),
    (dict(kv_heads=0), M.EINVAL, "no kv heads"),
    (dict(max_ctx=300), M.EINVAL, "max_ctx"),
    (dict(recent=61), M.EINVAL, "over the budget"),
    (dict(recent=0xFFFFFFFF), M.EINVAL, "over the budget"),
    (dict(pos=None), M.EINVAL, "go together"),
    (dict(seen=None), M.EINVAL, "go together"),
    (dict(w=None), M.EINVAL, "null"),
    (dict(pos_out=None), M.EINVAL, "null"),
    (dict(k=ODD), M.EINVAL, "aligned"),
    (dict(ws=None), M.EWORKSPACE, "workspace"),
    (dict(ws=ODD), M.EWORKSPACE, "workspace"),
    (dict(bytes=16), M.EWORKSPACE, "needed"),
])
def test_evict_refuses(kw, code, msg):
    rc, err = evict_rc(**kw)
    assert rc == code and msg in err and err.startswith("cache_evict"), (rc, err)


def test_evict_workspace_covers_the_rows_that_can_move():
    size = lambda **kw: M.cache_evict_workspace(M.evict_args(**dict(dict(batch=3, kv_heads=2, dim=64, cap=1 << 20,  # noqa: E731
                                                                         max_ctx=1 << 20, budget=1000), **kw)))
    assert size() >= 6 * 4 + 2 * 6 * 1000 * 4
    assert size(max_ctx=1300) >= 6 * 4 + 2 * 6 * 300 * 4
    assert size(max_ctx=900) < 6 * 4 * 900


# ---- with a HIP runtime that records launches and runs nothing ----


def space(nbytes, addr=0x200000):
    t = tensor(None, addr)
    t.numel, t.element_size = lambda: nbytes, lambda: 1
    t.nbytes = nbytes
    return t


X, F, I = tensor(torch.bfloat16), tensor(torch.float32), tensor(torch.int32)


def tree_call(a, ws):
    M.attn_tree(a, X, X, X, X, X, I, X, ws, lse=F, stream=0x71000)


def weights_call(a, ws):
    M.cache_weights(a, X, F, X, I, F, ws, w=F, stream=0x71000)


def evict_call(a, ws):
    M.cache_evict(a, X, X, F, I, F, I, I, ws, stream=0x71000)


CALLS = {
    "tree": (tree_call, M.attn_tree_workspace,
             M.tree_args(batch=3, n_draft=9, heads=32, kv_heads=8, dim=128, cap=9000, max_ctx=9000),
             ["tree_split", "tree_merge"]),
    "weights": (weights_call, M.cache_weights_workspace,
                M.weights_args(batch=3, n_q=100, heads=32, kv_heads=8, dim=64, cap=9000, max_ctx=9000),
                ["weights_many", "weights_join"]),
    "evict": (evict_call, M.cache_evict_workspace,
              M.evict_args(batch=3, kv_heads=8, dim=128, cap=9000, max_ctx=9000, budget=5000),
              ["evict_select", "evict_move"]),
}


@pytest.mark.parametrize("name", CALLS)
def test_workspaces(hip, name):  # noqa: F811
    """The bytes that the query names are enough and all are needed; the library allocates nothing of its own."""
    call, query, a, kernels = CALLS[name]
    need = query(a)
    assert need > 0
    for ws in (None, space(need - 1), space(need, 0x200008), space(0)):
        with pytest.raises(M.MakoError, match="workspace"):
            call(a, ws)
    assert launches(hip) == []
    call(a, space(need))
    got = launches(hip)
    assert len(got) == len(kernels) and all(k in x for k, x in zip(kernels, got)), got
    assert events(hip, "alloc", "free") == []


def test_calls_that_need_no_workspace(hip):  # noqa: F811
    """Short contexts' trees and few rows' weights take one launch, and null for a workspace."""
    a = M.tree_args(batch=2, n_draft=8, heads=32, kv_heads=8, dim=128, cap=9000, max_ctx=200)
    assert M.attn_tree_workspace(a) == 0
    tree_call(a, None)
    w = M.weights_args(batch=2, n_q=8, heads=32, kv_heads=8, dim=128, cap=9000, max_ctx=9000)
    assert M.cache_weights_workspace(w) == 0
    weights_call(w, None)
    M.cache_append(M.append_args(batch=2, n_draft=8, kv_heads=8, dim=128, cap=9000), X, X, X, X, I, I, stream=0x71000)
    got = launches(hip)
    assert [k in x for k, x in zip(("tree_split", "weights_few", "append_rows"), got)] == [True] * 3 and len(got) == 3
    assert events(hip, "alloc", "free") == []


def test_empty_calls_launch_nothing(hip):  # noqa: F811
    tree = dict(batch=2, n_draft=8, heads=32, kv_heads=8, dim=128, cap=9000, max_ctx=9000)
    for kw in (dict(batch=0), dict(n_draft=0)):
        a = M.tree_args(**dict(tree, **kw))
        assert M.attn_tree_workspace(a) == 0
        tree_call(a, None)
    wts = dict(batch=2, n_q=100, heads=32, kv_heads=8, dim=128, cap=9000, max_ctx=9000)
    for kw in (dict(batch=0), dict(max_ctx=0)):
        a = M.weights_args(**dict(wts, **kw))
        assert M.cache_weights_workspace(a) == 0
        weights_call(a, None)
    M.cache_append(M.append_args(batch=0, n_draft=8, kv_heads=8, dim=128, cap=9000), X, X, X, X, I, I, stream=0x71000)
    a = M.evict_args(batch=0, kv_heads=8, dim=128, cap=9000, max_ctx=9000, budget=5000)
    evict_call(a, None)
    assert launches(hip) == []


@pytest.mark.parametrize("dim", [64, 128, 256])
@pytest.mark.parametrize("n_draft,heads,kv", [(1, 1, 1), (8, 32, 8), (16, 32, 8), (64, 16, 1), (64, 64, 1), (33, 96, 32)])
def test_tree_split_covers_its_columns(hip, dim, n_draft, heads, kv):  # noqa: F811
    """Every (range or segment, column block) has a workgroup: blocks of 32, 64 or 128 columns, ranges for at most the CUs."""
    for batch in (1, 5, 200):
        for ctx in (0, 1, 100, 5000, 70000):
            a = M.tree_args(batch=batch, n_draft=n_draft, heads=heads, kv_heads=kv, dim=dim, cap=70000, max_ctx=ctx)
            hip.fake_clear()
            tree_call(a, space(M.attn_tree_workspace(a)))
            ev = events(hip, "launch")
            nc = n_draft * heads // kv
            ng = 1 if nc <= 32 else 2 if nc <= 64 else 4
            ncb = -(-nc // (32 * ng))
            grid = int(re.match(r"\d+", ev[0][2]).group())
            if len(ev) == 1:
                assert grid >= batch * kv * ncb
            else:
                assert ncb <= grid <= max(256 + 8 * ncb, 8 * ncb)
                items = batch * n_draft * heads
                assert int(re.match(r"\d+", ev[1][2]).group()) in (items, -(-items // 4))
