"""The operators of a cache kept in pages without a GPU: csrc/pages.hip's kernels run on the CPU (tests/cpp/pages_cpu.cpp),
also over malformed tables, and so does the attention's split (tests/cpp/paged_split_cpu.cpp); what the entry points refuse, and with which message, before touching the device."""
import ctypes
import os
import subprocess

import pytest

pytest.importorskip("torch")

import mako_attn as M  # noqa: E402
from conftest import ROOT  # noqa: E402

CPP = os.path.join(ROOT, "tests", "cpp")
FAKE = ctypes.c_void_p(0x10000)  # aligned, never dereferenced: every call below fails validation first
ODD = ctypes.c_void_p(0x10008)
BIG = ctypes.c_size_t(1 << 40)


@pytest.mark.parametrize("name", ["pages_cpu", "paged_split_cpu"])
def test_on_the_cpu(name):
    subprocess.run(["make", "-s", "-C", CPP, f"bin/{name}"], check=True)
    r = subprocess.run([os.path.join(CPP, "bin", name)], capture_output=True, text=True, timeout=600)
    assert r.returncode == 0 and "all passed" in r.stdout, r.stdout + r.stderr


def struct(cls, base, kw):
    a = dict(base, **{f: kw.pop(f) for f, _ in cls._fields_ if f in kw})
    return ctypes.byref(cls(*[a[f] for f, _ in cls._fields_]))


def answer(rc):
    return rc, M.lib().mako_last_error().decode()


def paged_rc(**kw):
    a = struct(M.PagedArgs, dict(batch=2, rows=16, q_pad=16, heads=8, kv_heads=2, dim=128, pages=8, page=64, max_pages=4,
                                 max_new=8, max_ctx=256, width=1024, scale=0.088), kw)
    p = dict(in_=M.BF16, out=M.BF16, q=FAKE, k=FAKE, v=FAKE, table=FAKE, starts=FAKE, ctx=FAKE, o=FAKE, ws=FAKE, bytes=BIG)
    p.update(kw)
    return answer(M.lib().mako_attn_paged(a, p["in_"], p["out"], p["q"], p["k"], p["v"], p["table"], p["starts"], p["ctx"],
                                          p["o"], None, p["ws"], p["bytes"], None))


@pytest.mark.parametrize("kw,code,msg", [
    (dict(dim=96), M.EUNSUPPORTED, "heads of 96"),
    (dict(in_=M.F32), M.EUNSUPPORTED, "input type"),
    (dict(out=M.F16), M.EUNSUPPORTED, "output type"),
    (dict(heads=7), M.EINVAL, "over 2 kv heads"),
    (dict(kv_heads=0), M.EINVAL, "over 0 kv heads"),
    (dict(page=16), M.EINVAL, "pages of 16 rows"),
    (dict(page=96), M.EINVAL, "pages of 96 rows"),
    (dict(page=8192), M.EINVAL, "pages of 8192 rows"),
    (dict(max_ctx=257), M.EINVAL, "max_ctx 257"),
    (dict(max_ctx=1 << 31, max_pages=1 << 26), M.EINVAL, "max_ctx"),
    (dict(kv_heads=1 << 13, heads=1 << 13, dim=64, page=4096), M.EINVAL, "4 GiB"),
    (dict(rows=17), M.EINVAL, "query heads of 16"),
    (dict(max_new=17), M.EINVAL, "17 of a sequence"),
    (dict(starts=None, batch=17), M.EINVAL, "a row each of 17"),
    (dict(width=1020), M.EINVAL, "o rows"),
    (dict(width=1026), M.EINVAL, "o rows"),
    (dict(width=1 << 20), M.EINVAL, "o rows"),
    (dict(scale=0.0), M.EINVAL, "scale"),
    (dict(scale=float("nan")), M.EINVAL, "scale"),
    (dict(q=None), M.EINVAL, "null"),
    (dict(table=None), M.EINVAL, "null"),
    (dict(ctx=None), M.EINVAL, "null"),
    (dict(v=ODD), M.EINVAL, "aligned"),
    (dict(o=ODD), M.EINVAL, "aligned"),
    (dict(rows=1 << 26, q_pad=1 << 26, heads=64, width=8192), M.EINVAL, "too many"),
    (dict(rows=1 << 22, q_pad=1 << 22, max_ctx=1 << 30, max_pages=1 << 24), M.EINVAL, "too many"),
    (dict(rows=1 << 21, q_pad=1 << 21, max_new=1 << 21), M.EINVAL, "too many"),  # (new rows far past max_ctx)
])
def test_attention_refuses(kw, code, msg):
    rc, err = paged_rc(**kw)
    assert rc == code and msg in err and err.startswith("attention_paged"), (rc, err)


PAGES = dict(batch=2, rows=16, d_pad=16, pages=8, page=64, max_pages=4, kv_heads=2, dim=128, layers=1)


def write_rc(**kw):
    a = struct(M.PagesArgs, PAGES, kw)
    p = dict(kd=FAKE, vd=FAKE, table=FAKE, starts=FAKE, ctx=FAKE, k=FAKE, v=FAKE)
    p.update(kw)
    return answer(M.lib().mako_pages_write(a, p["kd"], p["vd"], p["table"], p["starts"], p["ctx"], None, p["k"], p["v"],
                                           None))


@pytest.mark.parametrize("kw,code,msg", [
    (dict(dim=32), M.EUNSUPPORTED, "heads of 32"),
    (dict(kv_heads=0), M.EINVAL, "0 kv heads"),
    (dict(page=32), M.EINVAL, "pages of 32 rows"),
    (dict(max_pages=1 << 25), M.EINVAL, "below 2^31 rows"),
    (dict(batch=1 << 20, max_pages=1 << 13), M.EINVAL, "too many"),
    (dict(d_pad=15), M.EINVAL, "kv heads of 15"),
    (dict(starts=None, batch=17), M.EINVAL, "a row each of 17"),
    (dict(kd=None), M.EINVAL, "null"),
    (dict(table=None), M.EINVAL, "null"),
    (dict(k=ODD), M.EINVAL, "aligned"),
    (dict(rows=1 << 30, d_pad=1 << 30), M.EINVAL, "exceed the grid"),
])
def test_write_refuses(kw, code, msg):
    rc, err = write_rc(**kw)
    assert rc == code and msg in err and err.startswith("pages_write"), (rc, err)


def reserve_rc(**kw):
    a = struct(M.PagesArgs, PAGES, kw)
    p = dict(table=FAKE, refs=FAKE, starts=FAKE, ctx=FAKE, to=FAKE, ro=FAKE, co=FAKE, k=FAKE, v=FAKE, ws=FAKE, bytes=BIG)
    p.update(kw)
    return answer(M.lib().mako_pages_reserve(a, p["table"], p["refs"], p["starts"], p["ctx"], p["to"], p["ro"], p["co"],
                                             p["k"], p["v"], p["ws"], p["bytes"], None))


@pytest.mark.parametrize("kw,code,msg", [
    (dict(batch=4097, rows=5000), M.EINVAL, "4097 sequences"),
    (dict(dim=32), M.EUNSUPPORTED, "heads of 32"),
    (dict(page=100), M.EINVAL, "pages of 100 rows"),
    (dict(starts=None, batch=17), M.EINVAL, "a row each of 17"),
    (dict(v=None), M.EINVAL, "go together"),
    (dict(layers=0), M.EINVAL, "no layers"),
    (dict(k=ODD), M.EINVAL, "aligned"),
    (dict(refs=None), M.EINVAL, "null"),
    (dict(co=None), M.EINVAL, "null"),
    (dict(bytes=40), M.EWORKSPACE, "workspace of 40"),
    (dict(ws=None), M.EWORKSPACE, "workspace"),
    (dict(ws=ODD), M.EWORKSPACE, "workspace"),
])
def test_reserve_refuses(kw, code, msg):
    rc, err = reserve_rc(**kw)
    assert rc == code and msg in err and err.startswith("pages_reserve"), (rc, err)


def fork_rc(**kw):
    a = struct(M.PagesArgs, dict(PAGES, kv_heads=0, dim=0, layers=0), kw)
    p = dict(table=FAKE, refs=FAKE, ctx=FAKE, to=FAKE, ro=FAKE, co=FAKE, ws=FAKE, bytes=BIG)
    p.update(kw)
    return answer(M.lib().mako_pages_fork(a, None, None, p["table"], p["refs"], p["ctx"], p["to"], p["ro"], p["co"],
                                          p["ws"], p["bytes"], None))


@pytest.mark.parametrize("kw,code,msg", [
    (dict(page=0), M.EINVAL, "pages of 0 rows"),
    (dict(to=ODD), M.EINVAL, "in place, or neither"),
    (dict(co=ODD), M.EINVAL, "in place, or neither"),
    (dict(table=None), M.EINVAL, "null"),
    (dict(bytes=39), M.EWORKSPACE, "workspace of 39 bytes, 40 needed"),
    (dict(ws=None), M.EWORKSPACE, "workspace"),
    (dict(batch=1 << 24, max_pages=1), M.EINVAL, "exceed the grid"),
])
def test_fork_refuses(kw, code, msg):
    rc, err = fork_rc(**kw)
    assert rc == code and msg in err and err.startswith("pages_fork"), (rc, err)


def compact_rc(**kw):
    a = struct(M.PagesArgs, PAGES, kw)
    p = dict(table=FAKE, refs=FAKE, to=FAKE, ro=FAKE, used=FAKE, k=FAKE, v=FAKE, ws=FAKE, bytes=BIG)
    p.update(kw)
    return answer(M.lib().mako_pages_compact(a, p["table"], p["refs"], p["to"], p["ro"], p["used"], None, p["k"], p["v"],
                                             p["ws"], p["bytes"], None))


@pytest.mark.parametrize("kw,code,msg", [
    (dict(dim=32), M.EUNSUPPORTED, "heads of 32"),
    (dict(pages=1 << 31), M.EINVAL, "too many"),
    (dict(v=None), M.EINVAL, "go together"),
    (dict(layers=0), M.EINVAL, "no layers"),
    (dict(v=ODD), M.EINVAL, "aligned"),
    (dict(used=None), M.EINVAL, "null"),
    (dict(bytes=100), M.EWORKSPACE, "workspace of 100"),
    (dict(ws=ODD), M.EWORKSPACE, "workspace"),
])
def test_compact_refuses(kw, code, msg):
    rc, err = compact_rc(**kw)
    assert rc == code and msg in err and err.startswith("pages_compact"), (rc, err)
