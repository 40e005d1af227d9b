"""The cache operators' host side without a GPU: what they refuse, and with which message, before touching the device."""
import ctypes

import pytest

import mako_attn as M

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
