"""Runs the streams of attention over a cache in pages (gen_attn_paged.py) on the emulator (fwd64_emu.py) for a small
sequence, with the operands attn_paged.hip computes restated here, over all of its keys or a piece of its tiles, and compares
the outputs and log-sums with a softmax in 64 bits."""
import os
import sys

import numpy as np

HERE = os.path.dirname(os.path.abspath(__file__))
sys.path.insert(0, os.path.join(os.path.dirname(HERE), "mako-common_amd", "csrc"))
import fwd64_emu as E  # noqa: E402
import fwd64_run as R64  # noqa: E402
import fwd_r32_run as R32  # noqa: E402
import gen_attn_fwd64 as G  # noqa: E402
import gen_attn_fwd_r32 as G32  # noqa: E402
import oracle as O  # noqa: E402

SOPS = {'qrs': 's[0:3]', 'ors': 's[4:7]', 'lrs': 's[8:11]', 'ent': 's[12:13]'}
SOPS.update({n: f's{14 + i}' for i, n in enumerate(
    ['c', 'ntw', 'nt', 'lmin', 'has_lse', 'ogs', 'kb0', 'kb1', 'kn', 'vb0', 'vb1', 'skww', 'skw', 'svww', 't0', 'tlast',
     'npages', 'pstride', 'pmask', 'pshift', 'pg0', 'pg1', 'pg2', 'pg3', 'ogs2', 'qo1'])})
SREG = {n: int(r[2:].split(':')[0]) if r[1] == '[' else int(r[1:]) for n, r in SOPS.items()}


VREG64 = {**R64.VREG, 'vdo': f'v{G.CLOBBER_V + len(R64.VREG)}'}


class Emu(E.Emu):
    """The emulator with the scalar instructions that the page look-ups add; a scalar load must lie in the table's row."""
    row = (0, 0)

    def step(self, w):
        op = self.prog[w.pc]
        mn, A = op.mn, op.args
        if mn == 's_load_dword':
            b = E.parse_reg(A[1])[1]
            at = (int(w.s[b]) | (int(w.s[b + 1]) << 32)) + self.sread(w, A[2])
            assert self.row[0] <= at and at + 4 <= self.row[1], 'a page number past the table row is read'
        if mn not in ('s_mul_hi_u32', 's_mul_i32', 's_min_u32', 's_lshr_b32', 's_cmp_lt_u32', 's_and_b32'):
            return super().step(w)
        w.pc += 1
        self.count += 1
        if mn == 's_cmp_lt_u32':
            w.scc = int(self.sread(w, A[0]) < self.sread(w, A[1]))
            return None
        a, b = self.sread(w, A[1]), self.sread(w, A[2])
        r = {'s_mul_hi_u32': a * b >> 32, 's_mul_i32': a * b & 0xFFFFFFFF, 's_min_u32': min(a, b), 's_lshr_b32': a >> (b & 31),
             's_and_b32': a & b}[mn]
        w.s[E.parse_reg(A[0])[1]] = r
        if mn == 's_min_u32':
            w.scc = int(a < b)
        elif mn in ('s_lshr_b32', 's_and_b32'):
            w.scc = int(r != 0)
        return None


def program(ind, outd, d, lines=None, wave_rows=64):
    r32 = d == 256 and wave_rows != 32
    lines = lines or (G32.body(ind, outd, paged=True) if r32 else G.body(ind, outd, d=d, paged=True, rows=wave_rows))
    vreg = R32.VREG if r32 else VREG64
    out = []
    for ln in lines:
        ln = ln.replace('%=', '0')
        for names in (vreg, SOPS):
            for n, r in sorted(names.items(), key=lambda x: -len(x[0])):
                ln = ln.replace(f'%[{n}]', r)
        out.append(ln)
    return E.parse(out)


def run(heads, kv, n, ctx, page, d, ind='bf16', outd='f32', cut=None, seed=0, kgrow=0.0, missing=(), lines=None, wave_rows=64):
    """n new rows behind ctx; cut = (ta, tb): the piece of tiles [ta, tb) (one item only); wave_rows: 64 or 32 (heads of 256: the stream of
    32-key tiles). Returns the worst errors."""
    rng = np.random.default_rng(seed)
    conv = O.to_bf16_bits if ind == 'bf16' else O.to_f16_bits
    dt = O.BF16 if ind == 'bf16' else O.F16
    val = lambda b: O.bits_to_f32(b, dt).astype(np.float64)  # noqa: E731
    keys = ctx + n
    held = -(-keys // page)
    pages = held + 3
    order = rng.permutation(pages)[:held]
    kf = rng.standard_normal((kv, held * page, d), dtype=np.float32)
    kf *= (1 + kgrow * (np.arange(held * page) // 64))[None, :, None].astype(np.float32)
    vf = rng.standard_normal((kv, held * page, d), dtype=np.float32)
    kb, vb, qb = conv(kf), conv(vf), conv(rng.standard_normal((heads, n, d), dtype=np.float32))
    pool = [np.full((pages, kv, page, d), 0x7FC0 if ind == 'bf16' else 0x7E00, np.uint16) for _ in range(2)]  # NaN
    for x, b in zip(pool, (kb, vb)):
        for j, e in enumerate(order):
            x[e] = b[:, j * page:(j + 1) * page]
            if j == held - 1 and keys % page:
                x[e, :, keys % page:] = 0x7FC0 if ind == 'bf16' else 0x7E00
    table = order.astype(np.uint32)
    kv_val = [val(kb)[:, :keys].copy(), val(vb)[:, :keys].copy()]
    for j in missing:
        table[j] = pages + 5 if j % 2 else 0xFFFFFFFF
        for x in kv_val:
            x[:, j * page:(j + 1) * page] = 0
    so = 4 if outd == 'f32' else 2
    width = heads * d
    arrays = [qb, pool[0], pool[1], table]
    offs = np.cumsum([8192] + [(a.nbytes + 4095) // 4096 * 4096 for a in arrays] + [n * width * so + 4096])
    Q0, K0, V0, T0, O0, L0 = [int(x) for x in offs]
    mem = E.Mem(L0 + heads * n * 4 + 8192)
    for at, a in zip((Q0, K0, V0, T0), arrays):
        mem.b[at:at + a.nbytes] = np.ascontiguousarray(a).view(np.uint8).ravel()
    mem.b[O0:O0 + n * width * so] = 0xAB
    prog, labels = program(ind, outd, d, lines, wave_rows)
    r32 = d == 256 and wave_rows != 32
    RW = 32 if r32 else wave_rows
    K_ROW, KT = 2 * d + 16, 32 if d == 256 and not r32 else 64
    K_TILE, V_TILE = -(-KT * K_ROW // 1024) * 1024, 2 * KT * d
    NKP = (K_TILE // 1024 - 1) // 4
    nbuf = 2 if r32 else G.NBUF
    group = heads // kv
    hq = 8 if group % 8 == 0 else 4 if group % 4 == 0 else 2 if group % 2 == 0 else 1
    hpw = 2 if hq == 8 else 1  # heads a wave
    R = RW * 4 // hq
    c = np.float32(1.0 / np.sqrt(float(d))) * np.float32(1.4426950408889634)
    lane = np.arange(64)
    g, c32 = lane >> 5, lane & 31
    vbase = nbuf * K_TILE
    early = 0
    row_b = 2 * d
    for hg in range(heads // hq):
        for qb_i in range(-(-n // R)):
            rows = min(R, n - qb_i * R)
            item_keys = ctx + qb_i * R + rows
            ta, tb = cut or (0, -(-item_keys // 64))
            ks = 64 * ta
            n_keys = min(64 * tb, item_keys) - ks
            emu = Emu(prog, labels, mem, nbuf * (K_TILE + V_TILE))
            emu.row = (T0, T0 + 4 * held)
            waves = []
            for w in range(4):
                W = E.Wave(w)
                h = hg * hq + w % (hq // hpw) * hpw
                kvh = hg * hq // group
                q0 = (w // (hq // hpw)) * (RW // hpw)
                row, hh = q0 + c32 // hpw, c32 % hpw
                row1 = row + 32 // hpw
                live = q0 < rows
                w_lim = ctx + qb_i * R + min(q0 + RW // hpw, rows)
                ntw = -(-min(n_keys, w_lim - ks) // KT) if live else 0
                p0 = ctx + qb_i * R + q0
                lim = [np.minimum(p0 + 32 // hpw * i + c32 // hpw + 1, keys) - ks - 8 * g for i in range(2)]
                kr = c32 * K_ROW + 16 * g

                def kd_of(i):
                    b = 1024 * i + 16 * lane
                    rr, ch = b // K_ROW, (b % K_ROW) // 16
                    at = np.array([R64.slot_of(int(r)) for r in rr]) * row_b + 16 * np.where(ch < d // 8, ch, 0)
                    return np.where(rr < KT, at, 0)
                orow = d * so
                lpr = orow // 16
                obase = w * RW * orow
                ew = obase + c32 * orow + (16 * ((c32 & 7) ^ g) if so == 4 else 8 * g + 16 * (c32 & 7))
                oc = lane // lpr
                vals = dict(kr=kr, qo=((hh * n + row) * d + 8 * g) * 2, swp=(lane ^ 32) * 4, ew=ew, lim0=lim[0],
                            er=obase + (lane // lpr) * orow + 16 * ((lane % lpr) ^ (lane // lpr)),
                            og=(q0 + oc // hpw) * width * so + (h + oc % hpw) * orow + 16 * (lane % lpr),
                            lo0=np.where(row < rows, ((h + hh) * n + qb_i * R + row) * 4, 0xffffffff))
                if r32:
                    hh, ii = (lane >> 4) & 1, lane & 15
                    vals.update({f'vr{x}': vbase + (8 * g + ii // 4) * 2 * d + 8 * (ii % 4) +
                                 32 * np.array([G32.v_unit(2 * x + int(a), int(b) // 4) for a, b in zip(hh, ii)])
                                 for x in range(4)})
                    vd, vdo = ((V_TILE // 4) * w + R32.vd_lane(lane, r) for r in (0, 2))
                    vals.update(vd=vd, vdo=vdo, vd2=vd + 4096, vdo2=vdo + 4096)
                    vals.update({f'kd{m}': kd_of(w + 4 * m if m < NKP else 4 * NKP) for m in range(NKP + 1)})
                    vreg = R32.VREG
                else:
                    vr = R64.v_read_regs(vbase, d, lane)
                    rr, pos = 16 * lane // (2 * d), 16 * lane % (2 * d)
                    vd, vdo = ((V_TILE // 4) * w + rr * 2 * d + 16 * ((pos // 16) & 1) +
                               32 * np.array([G.v_unit(int(u), int(r) + r0) for u, r in zip(pos // 32, rr)]) for r0 in (0, 2))
                    vals.update(vr0=vr[0], vr1=vr[1], kr0=kr, lim1=lim[1], vd=vd, vdo=vdo,
                                lo1=np.where(row1 < rows, ((h + hh) * n + qb_i * R + row1) * 4, 0xffffffff))
                    vals.update({f'kd{m}': kd_of(w + 4 * m) if m < NKP else 0 for m in range(4)}, kd4=kd_of(4 * NKP))
                    vreg = VREG64
                for name, x in vals.items():
                    W.v[int(vreg[name][1:])] = np.broadcast_to(np.asarray(x, np.int64), 64).astype(np.uint32)
                for name, base, nbytes in (('qrs', Q0 + (h * n + qb_i * R) * row_b, ((hpw - 1) * n + rows) * row_b),
                                           ('ors', O0 + qb_i * R * width * so, rows * width * so),
                                           ('lrs', L0, heads * n * 4)):
                    W.s[SREG[name]:SREG[name] + 4] = [base & 0xFFFFFFFF, base >> 32, nbytes, 0x20000]
                W.s[SREG['ent']:SREG['ent'] + 2] = [T0 & 0xFFFFFFFF, T0 >> 32]
                kbase, vb0 = (x + kvh * page * row_b for x in (K0, V0))
                per, t0, last = page // KT, ks // KT, ks // KT + -(-n_keys // KT) - 1
                pg = [int(table[min(t0 + i, last) // per]) for i in range(4)]
                step = 64 // lpr // hpw * width * so if 64 // lpr >= hpw else orow
                sv = dict(c=int(c.view(np.uint32)), nt=-(-n_keys // KT), ntw=ntw, lmin=min(p0 + 1, keys) - ks, has_lse=1,
                          ogs=step, ogs2=2 * step if step != orow or hpw == 1 else width * so, qo1=64 // hpw * d, kb0=kbase & 0xFFFFFFFF, kb1=kbase >> 32, kn=n_keys * row_b,
                          vb0=vb0 & 0xFFFFFFFF, vb1=vb0 >> 32, skw=0, skww=1024 * w, svww=vbase + (V_TILE // 4) * w, t0=t0,
                          tlast=last, npages=pages, pstride=kv * page * row_b, pmask=per - 1,
                          pshift=per.bit_length() - 1, pg0=pg[0], pg1=pg[1], pg2=pg[2], pg3=pg[3])
                for name, x in sv.items():
                    W.s[SREG[name]] = x & 0xFFFFFFFF
                waves.append(W)
            emu.run_wg(waves)
            early += emu.early
    raw = mem.b[O0:O0 + n * width * so]
    o = raw.view(np.float32).astype(np.float64) if so == 4 else O.bits_to_f32(raw.view(np.uint16), dt).astype(np.float64)
    o = o.reshape(n, heads, d)
    lse = mem.b[L0:L0 + heads * n * 4].view(np.float32).reshape(heads, n).astype(np.float64)
    out_bad = lse_bad = 0
    worst = 0.0
    lo, hi = (64 * cut[0], 64 * cut[1]) if cut else (0, keys)
    for h in range(heads):
        s = val(qb)[h] @ kv_val[0][h // group].T * float(c) * np.log(2)
        j = np.arange(keys)
        seen = (j <= ctx + np.arange(n)[:, None]) & (j >= lo) & (j < hi)
        s = np.where(seen, s, -np.inf)
        top = s.max(1, keepdims=True)
        p = np.exp(s - top)
        want = (p @ kv_val[1][h // group]) / p.sum(1, keepdims=True)
        err = np.abs(o[:, h] - want)
        worst = max(worst, float(err.max()))
        out_bad += int((~(err <= 2e-3 + 1e-2 * np.abs(want))).sum())
        lse_bad += int((~(np.abs(lse[h] - (top[:, 0] + np.log(p.sum(1)))) <= 1e-3)).sum())
    return dict(out_bad=out_bad, lse_bad=lse_bad, max_err=worst, early_reads=early)
