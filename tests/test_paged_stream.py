"""CPU checks of the instruction streams of attention over a cache in pages (mako-common_amd/csrc/gen_attn_paged.py): every
register they name is one their clobber lists reserve; no gfx950 software hazard; and on the emulator, whole items and pieces
of their tiles against a softmax in 64 bits: pages of one tile and of several, missing pages, NaN wherever no row lies, waves
whose rows end tiles apart, scores that send tiles down the exact path. The emulator refuses page numbers read past the
table row and counts LDS reads of bytes that have not landed; planted mistakes show that it does."""
import os
import sys

import pytest

HERE = os.path.dirname(os.path.abspath(__file__))
sys.path.insert(0, os.path.join(os.path.dirname(HERE), "mako-common_amd", "csrc"))
import fwd64_emu as E  # noqa: E402
import fwd64_hazards as Hz  # noqa: E402
import gen_attn_fwd64 as G  # noqa: E402
import gen_attn_fwd_r32 as G32  # noqa: E402
import gen_attn_paged as P  # noqa: E402
import paged_run as R  # noqa: E402


def test_registers_and_hazards():
    names = []
    for name, lines in P.streams():
        names.append(name)
        assert Hz.check(lines, name) == 0
    assert len(set(names)) == 24


def test_other_streams_are_as_before():
    """The dense and block-sparse streams know nothing of pages."""
    assert G.PAGED is False and G32.PAGED is False
    for lines in (G.body("bf16", "f32"), G.body("f16", "f16", sparse=True), G32.body("bf16", "bf16")):
        assert not any("%[pg" in ln or "npages" in ln or "s_mul_hi" in ln for ln in lines)


CASES = [
    dict(heads=4, kv=1, n=1, ctx=0, page=64, d=128),
    dict(heads=4, kv=1, n=1, ctx=700, page=128, d=128),
    dict(heads=8, kv=2, n=65, ctx=130, page=64, d=128, ind="f16", outd="f16"),
    dict(heads=1, kv=1, n=256, ctx=70, page=64, d=128, outd="bf16"),
    dict(heads=2, kv=1, n=100, ctx=191, page=256, d=128, missing=(0,)),
    dict(heads=4, kv=1, n=40, ctx=400, page=64, d=128, ind="f16", kgrow=1.5),
    dict(heads=4, kv=1, n=3, ctx=800, page=64, d=128, cut=(0, 5)),
    dict(heads=4, kv=1, n=3, ctx=800, page=128, d=128, cut=(3, 9)),
    dict(heads=4, kv=1, n=20, ctx=800, page=64, d=128, cut=(11, 13), ind="f16"),
    dict(heads=4, kv=2, n=150, ctx=200, page=128, d=64, missing=(1,)),
    dict(heads=1, kv=1, n=250, ctx=66, page=64, d=64, outd="bf16"),
    dict(heads=4, kv=1, n=2, ctx=600, page=64, d=64, cut=(4, 10), kgrow=0.5),
    # 32 rows a wave
    dict(heads=4, kv=1, n=1, ctx=0, page=64, d=128, wave_rows=32),
    dict(heads=4, kv=1, n=1, ctx=700, page=128, d=128, wave_rows=32, ind="f16", outd="f16"),
    dict(heads=4, kv=1, n=20, ctx=600, page=64, d=128, wave_rows=32, missing=(3,), outd="bf16"),
    dict(heads=2, kv=1, n=60, ctx=100, page=64, d=128, wave_rows=32),
    dict(heads=1, kv=1, n=128, ctx=70, page=64, d=128, wave_rows=32),
    dict(heads=4, kv=1, n=5, ctx=400, page=64, d=128, wave_rows=32, ind="f16", kgrow=1.5),
    dict(heads=4, kv=1, n=3, ctx=800, page=128, d=128, wave_rows=32, cut=(3, 9)),
    dict(heads=4, kv=1, n=3, ctx=800, page=64, d=128, wave_rows=32, cut=(12, 13)),
    dict(heads=4, kv=1, n=9, ctx=300, page=64, d=64, wave_rows=32, outd="bf16"),
    dict(heads=1, kv=1, n=100, ctx=500, page=256, d=64, wave_rows=32, ind="f16", outd="f16"),
    dict(heads=4, kv=2, n=2, ctx=600, page=64, d=64, wave_rows=32, kgrow=0.5),
    dict(heads=4, kv=1, n=1, ctx=63, page=64, d=256),
    dict(heads=4, kv=1, n=33, ctx=300, page=128, d=256, outd="bf16", missing=(1,)),
    dict(heads=1, kv=1, n=128, ctx=64, page=64, d=256, ind="f16", outd="f16"),
    dict(heads=2, kv=1, n=5, ctx=500, page=64, d=256, cut=(2, 8)),
    dict(heads=4, kv=1, n=5, ctx=500, page=64, d=256, cut=(7, 8)),
    dict(heads=4, kv=1, n=10, ctx=350, page=64, d=256, ind="f16", kgrow=1.5),
    # tiles of 32 keys
    dict(heads=4, kv=1, n=1, ctx=0, page=64, d=256, wave_rows=32),
    dict(heads=4, kv=1, n=1, ctx=31, page=64, d=256, wave_rows=32, outd="bf16"),
    dict(heads=4, kv=1, n=33, ctx=300, page=128, d=256, wave_rows=32, outd="bf16", missing=(1,)),
    dict(heads=1, kv=1, n=128, ctx=64, page=64, d=256, wave_rows=32, ind="f16", outd="f16"),
    dict(heads=2, kv=1, n=5, ctx=500, page=64, d=256, wave_rows=32, cut=(2, 8)),
    dict(heads=4, kv=1, n=5, ctx=500, page=64, d=256, wave_rows=32, cut=(7, 8)),
    dict(heads=4, kv=1, n=10, ctx=350, page=64, d=256, wave_rows=32, ind="f16", kgrow=1.5),
    # two heads a wave
    dict(heads=8, kv=1, n=1, ctx=300, page=64, d=128),
    dict(heads=8, kv=1, n=40, ctx=130, page=64, d=128, outd="bf16"),
    dict(heads=16, kv=2, n=33, ctx=70, page=64, d=64, ind="f16", outd="f16"),
    dict(heads=8, kv=1, n=1, ctx=700, page=128, d=128, wave_rows=32, outd="bf16"),
    dict(heads=8, kv=1, n=15, ctx=300, page=64, d=128, wave_rows=32, missing=(2,)),
    dict(heads=8, kv=1, n=3, ctx=300, page=64, d=64, wave_rows=32),
    dict(heads=8, kv=1, n=16, ctx=100, page=64, d=64, wave_rows=32, ind="f16", outd="f16"),
    dict(heads=8, kv=1, n=17, ctx=100, page=64, d=256),
    dict(heads=8, kv=1, n=1, ctx=200, page=64, d=256, outd="bf16"),
    dict(heads=8, kv=1, n=1, ctx=500, page=64, d=256, cut=(2, 6)),
    dict(heads=8, kv=1, n=9, ctx=200, page=64, d=256, wave_rows=32),
    dict(heads=8, kv=1, n=16, ctx=200, page=64, d=256, wave_rows=32, ind="f16", outd="f16"),
]


@pytest.mark.parametrize("case", CASES, ids=lambda c: "-".join(f"{k}{v}" for k, v in c.items()))
def test_stream(case, monkeypatch):
    monkeypatch.setattr(E, "POISON", [True])  # registers start as garbage
    taken = E.EXACT_COUNT[0]
    r = R.run(**case, seed=3)
    assert r["out_bad"] == 0 and r["lse_bad"] == 0 and r["early_reads"] == 0, r
    if case.get("kgrow"):
        assert E.EXACT_COUNT[0] > taken  # the exact path ran


@pytest.mark.parametrize("d,rows", [(128, 64), (128, 32), (256, 64), (256, 32)])
def test_planted_page_of_another_tile_is_found(d, rows, monkeypatch):
    """Every tile from the page read before: the outputs are off."""
    of = G.page_load
    monkeypatch.setattr(G, "page_load", lambda page, tile, t: of(page, tile, t)[:3] + ["s_nop 0"])
    assert R.run(heads=4, kv=1, n=3, ctx=600, page=64, d=d, wave_rows=rows)["out_bad"] > 0


def test_planted_look_past_the_table_is_found(monkeypatch):
    of = G.page_load
    monkeypatch.setattr(G, "page_load", lambda page, tile, t: [f"s_mov_b32 {t}, {tile}"] + of(page, tile, t)[1:])
    with pytest.raises(AssertionError, match="past the table row"):
        R.run(heads=4, kv=1, n=3, ctx=600, page=64, d=128)
