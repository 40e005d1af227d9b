"""CPU checks of the streams of attention over a cache in pages (mako-common_amd/csrc/gen_attn_paged.py) in pieces whose bytes
of K pass 32 bits: the first tiles of such a piece on the emulator (paged_run.py), against a softmax in 64 bits."""
import pytest

import paged_run as R


@pytest.mark.parametrize("past", [1, 100])
@pytest.mark.parametrize("d,rows,kt", [(64, 64, 64), (64, 32, 64), (128, 64, 64), (128, 32, 64), (256, 64, 64), (256, 32, 32)])
def test_first_tiles(d, rows, kt, past, monkeypatch):
    """A piece of 2^32 bytes of K and `past` keys, in whose first three tiles of 64 keys the waves' products end."""
    class Emu(R.Emu):
        def run_wg(self, waves):
            for w in waves:
                keys = (1 << 32) // (2 * d) + past
                w.s[R.SREG["kn"]] = keys * 2 * d & 0xFFFFFFFF
                w.s[R.SREG["tlast"]] = int(w.s[R.SREG["t0"]]) + (keys - 1) // kt
            super().run_wg(waves)

    monkeypatch.setattr(R, "Emu", Emu)
    r = R.run(heads=1, kv=1, n=3, ctx=900, page=64, d=d, wave_rows=rows, cut=(0, 3), seed=3)
    assert r["out_bad"] == 0 and r["lse_bad"] == 0 and r["early_reads"] == 0, r


@pytest.mark.parametrize("d,rows,kt", [(64, 64, 64), (64, 32, 64), (128, 64, 64), (128, 32, 64), (256, 64, 64), (256, 32, 32)])
@pytest.mark.parametrize("keys", [1, 33])
def test_last_tiles(d, rows, kt, keys, monkeypatch):
    """The last tiles of a piece, of `keys` keys in the last one, whose count has passed 2^32 bytes: three tiles from there on."""
    class Emu(R.Emu):
        def run_wg(self, waves):
            for w in waves:
                assert int(w.s[R.SREG["kn"]]) == (2 * 64 + keys) * 2 * d  # (2^32 bytes before them leave it)
            super().run_wg(waves)

    monkeypatch.setattr(R, "Emu", Emu)
    r = R.run(heads=1, kv=1, n=1, ctx=8 * 64 + keys - 1, page=64, d=d, wave_rows=rows, cut=(6, 9), seed=3)
    assert r["out_bad"] == 0 and r["lse_bad"] == 0 and r["early_reads"] == 0, r
