"""Plain forms of the operators of a cache kept in pages, in 64 bits, and the error their kernels may make.

The attention's kernels round the probabilities to the input type for the product with V: p (1 + e), |e| <= h, half a step of
the type (bf16 2^-8, f16 2^-11). Rows that see fewer than 64 keys (heads of 256: 32) get bf16 probabilities as a sum of two
bf16 values: the second is off by h of what the first left, h p, so |e| <= h^2. Below f16's smallest normal value, 2^-14, f16 probabilities
are off by up to half a step there, 2^-25, against a sum of at least 1 (the running maximum
is a score that was met). So an output is off by at most |e| sum_j w_j |v_j| + 2^-25 sum_j |v_j| (f16), by what the
scores' errors make of the weights (a score off by ds moves each weight by at most a factor exp(2 ds)), and by its own
rounding. A score is a sum of dim products in 32 bits: ds <= 2^-24 ((dim + 2) scale sum |q k| + |score| + 8)."""
import math

import torch


def half_step(dtype):
    return torch.finfo(dtype).eps / 2


def rows_of(pool, table, n, kvh):
    """Rows [0, n) of a sequence from its pages (a page that the table does not name: zeros)."""
    pages, _, page, dim = pool.shape
    out = torch.zeros((-(-n // page) * page, dim), dtype=torch.float64, device=pool.device)
    for j in range(-(-n // page)):
        e = int(table[j]) & 0xFFFFFFFF
        if e < pages:
            out[j * page:(j + 1) * page] = pool[e, kvh].double()
    return out[:n]


def attention(q, k, v, table, ctx, new, starts, *, scale, max_ctx, max_new, out_dtype):
    """q [heads][q_pad][dim]; lists ctx, new and starts. For each row of a sequence and head: output, log-sum and the
    errors allowed; {(row): (o [heads][dim], lse [heads], o_tol, lse_tol)} by sequence as stacked tensors."""
    H, KV, D = q.shape[0], k.shape[1], q.shape[2]
    res = []
    for b, (c, n, s0) in enumerate(zip(ctx, new, starts)):
        c, n = min(c, max_ctx), min(n, max_new)
        if n == 0:
            continue
        keys = min(c + n, max_ctx)
        o = torch.zeros((n, H, D), dtype=torch.float64, device=q.device)
        tol, lse, ltol = torch.zeros_like(o), torch.zeros((n, H), dtype=torch.float64, device=q.device), None
        ltol = torch.zeros_like(lse)
        seen = torch.clamp(torch.arange(n, device=q.device) + c + 1, max=max_ctx)
        hidden = torch.arange(keys, device=q.device) >= seen[:, None]
        e = half_step(q.dtype)
        f16 = q.dtype == torch.float16
        p_err = torch.where(seen < (32 if D == 256 else 64), e if f16 else e * e, e)[:, None]
        for h in range(H):
            kk, vv = rows_of(k, table[b], keys, h * KV // H), rows_of(v, table[b], keys, h * KV // H)
            qq = q[h, s0:s0 + n].double()
            sc = torch.matmul(qq, kk.t().contiguous()) * scale
            size = torch.matmul(qq.abs(), kk.abs().t().contiguous()) * scale
            sc[hidden], size[hidden] = -math.inf, 0.0
            w = torch.softmax(sc, 1)
            ds = 2.0 ** -24 * ((D + 2) * size.amax(1, keepdim=True) + sc.masked_fill(hidden, 0).abs().amax(1, keepdim=True) + 8)
            o[:, h] = torch.matmul(w, vv)
            tol[:, h] = torch.matmul(w, vv.abs()) * (p_err + 2.5 * ds + keys * 2.0 ** -24)
            if f16:
                tol[:, h] += 2.0 ** -25 * torch.matmul((~hidden).double(), vv.abs())
            lse[:, h] = torch.logsumexp(sc, 1)
            # the sums: at most a chain of a tile's 32 terms a lane and the tiles, then the logarithm
            ltol[:, h] = ds[:, 0] + (64 + keys / 64) * 2.0 ** -24 + 2.0 ** -22 * (lse[:, h].abs() + 4)
        # the output's rounding: half a step of the value; f16 outputs below 2^-14 lie on multiples of 2^-24, so off by 2^-25
        tol += half_step(out_dtype) * o.abs() * 1.01 + (2.0 ** -25 if out_dtype == torch.float16 else 1e-30)
        res.append((b, s0, n, o, lse, tol, ltol))
    return res


def write(k, v, kd, vd, table, ctx, new, starts, end=None):
    """Lists ctx, new, starts (and end); pools [pages][kv][page][dim] changed in place."""
    pages, _, page, _ = k.shape
    for b, (c, n, s0) in enumerate(zip(ctx, new, starts)):
        for i in range(n):
            at = c + i
            if at // page >= len(table[b]) or (end is not None and at >= end[b]):
                continue
            e = table[b][at // page]
            if 0 <= e < pages:
                k[e, :, at % page], v[e, :, at % page] = kd[:, s0 + i], vd[:, s0 + i]


def reserve(table, refs, ctx, new, page, pages):
    """Lists; returns table, refs, ctx afterwards and the pages copied as (source, target, rows)."""
    table, refs, out, moves = [list(t) for t in table], list(refs), [], []
    free = [p for p in range(pages) if refs[p] == 0][::-1]
    last, count, held = {}, {}, list(refs)
    for b, (c, n) in enumerate(zip(ctx, new)):
        if n and c % page and c < page * len(table[b]):
            e = table[b][c // page]
            last[e], count[e] = b, count.get(e, 0) + 1
    for b, (c, n) in enumerate(zip(ctx, new)):
        at, end = c, min(c + n, page * len(table[b]))
        while at < end:
            j, part = at // page, at % page
            e = table[b][j]
            shared = part and 0 <= e < pages and held[e] > 1 and (held[e] > count[e] or last[e] != b)
            if not 0 <= e < pages or shared:
                if not free:
                    break
                new_page = free.pop()
                refs[new_page] = 1
                if shared:
                    refs[e] -= 1
                    moves.append((e, new_page, part))
                table[b][j] = new_page
            at = min(end, (j + 1) * page)
        out.append(at)
    return table, refs, out, moves


def fork(table, refs, ctx, parent, keep, page):
    refs, B = list(refs), len(table)
    new, out = [], []
    for i in range(B):
        p = parent[i] if parent is not None else i
        c = min(ctx[p], keep[i] if keep is not None else ctx[p]) if 0 <= p < B else 0
        n = -(-c // page)
        new.append(list(table[p][:n]) + [-1] * (len(table[i]) - n) if n else [-1] * len(table[i]))
        out.append(c)
    for t, sign in ((new, 1), (table, -1)):
        for row in t:
            for e in row:
                if e >= 0:
                    refs[e] += sign
    return new, refs, out


def compact(table, refs):
    """Returns table, refs, the number of used pages, and each page's new number (-1: free)."""
    used = sum(r > 0 for r in refs)
    number = [p if r > 0 else -1 for p, r in enumerate(refs)]
    out = list(refs)
    holes = iter([p for p in range(used) if refs[p] == 0])
    for p in range(used, len(refs)):
        if refs[p] > 0:
            number[p] = next(holes)
            out[number[p]], out[p] = refs[p], 0
    return [[number[e] if e >= 0 else -1 for e in row] for row in table], out, used, number
