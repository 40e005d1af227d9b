#!/usr/bin/env python3
"""Writes the instruction streams of attention over a cache in pages (attn_paged.hip): those of flash_fwd_r64 and
flash_fwd_r32 with tiles that come from the pages of a table (gen_attn_fwd64.py, gen_attn_fwd_r32.py: PAGED). They go to the
file named on the command line, which the build makes beside its objects.

Run: python3 gen_attn_paged.py FILE
"""
import sys

import gen_attn_fwd64 as G
import gen_attn_fwd_r32 as R


def streams():
    """(macro name, lines) of every stream."""
    for d in (128, 64, 256):
        for form in ("MANY", "FEW"):  # rows a wave: 64 (heads of 256: 32, by flash_fwd_r32's stream), 32
            for ind in ("bf16", "f16"):
                for outd in ("f32", ind):
                    r32 = d == 256 and form == "MANY"
                    lines = R.body(ind, outd, paged=True) if r32 else \
                        G.body(ind, outd, d=d, paged=True, rows=64 if form == "MANY" else 32)
                    (R if r32 else G).check_registers(lines, paged=True)
                    yield f"MAKO_PAGED_D{d}_{form}_{ind.upper()}_{outd.upper()}", lines


def main(path):
    out = ["// Generated by gen_attn_paged.py.", "#pragma once", ""]
    for name, lines in streams():
        out += [f"#define {name} \\"] + [f'    "{ln}\\n" \\' for ln in lines] + ['    ""', ""]
    out += [f"#define MAKO_PAGED_CLOBBERS {G.clobbers(paged=True)}",
            f"#define MAKO_PAGED_R32_CLOBBERS {R.clobbers(paged=True)}", ""]
    with open(path, "w") as f:
        f.write("\n".join(out))


if __name__ == "__main__":
    main(sys.argv[1])
