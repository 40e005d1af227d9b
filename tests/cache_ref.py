"""The cache operators in 64 bits, one row at a time from their definitions (numpy), and the error bounds of the kernels.

Bounds: u(t) is half a step of type t relative to the value (torch.finfo(t).eps / 2). With S = sum_d |q_d k_d| scale:
  a score       its dim products are exact in f32 and summed there: dim u(f32) S, and 3 u(f32) |s| for the scaling and the
                offset: ds
  exp           relative ds + 4 u(f32) (v_exp_f32 is off by at most one step, its argument by u(f32) of it, see |s| above)
  a sum of n    (n + 2) u(f32) of the sum of the magnitudes
  P for P V     u(f16) for f16 tiles and output; else two values of the type: u(t)^2 of P
  the output    u(out) of the value; f16's smallest step is 2^-24, and P below it is lost: 2^-25 a key (P is at most
                2^8, where the running maximum lags)
"""
import numpy as np
import torch

U32F = 2.0 ** -24
HALF = {torch.float32: 2.0 ** -24, torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}


def f64(t):
    return t.detach().cpu().double().numpy()


def tree(q, k, v, kd, vd, ctx, nodes, mask, *, n, scale, out, in_dtype):
    """(o [B n][H D], lse [H][B n], tolerance of o, of lse), rows past nodes NaN. Arrays: float64 of the tensors' values;
    mask: [B][n] ints, or None for the chain."""
    B, KV, _, D = k.shape
    H = q.shape[0]
    o = np.full((B * n, H * D), np.nan)
    tol = np.zeros_like(o)
    lse = np.full((H, B * n), np.nan)
    ltol = np.zeros_like(lse)
    up = HALF[torch.float16] if in_dtype == torch.float16 and out == torch.float16 else HALF[in_dtype] ** 2
    tiny = 2.0 ** -25 if in_dtype == torch.float16 else 0.0
    for b in range(B):
        for r in range(nodes[b]):
            row = b * n + r
            m = (2 << r) - 1 if mask is None else int(mask[b][r])
            js = [j for j in range(nodes[b]) if m >> j & 1]
            for h in range(H):
                g = h // (H // KV)
                kk = np.concatenate([k[b, g, :ctx[b]], kd[g, b * n:b * n + n][js]])
                vv = np.concatenate([v[b, g, :ctx[b]], vd[g, b * n:b * n + n][js]])
                cols = slice(h * D, (h + 1) * D)
                if len(kk) == 0:
                    o[row, cols], lse[h, row] = 0.0, -np.inf
                    continue
                s = kk @ q[h, row] * scale
                ds = (D * np.abs(kk) @ np.abs(q[h, row]) * scale + 3 * np.abs(s)) * U32F
                top = s.max()
                p = np.exp(s - top)
                total = p.sum()
                p /= total
                o[row, cols], lse[h, row] = p @ vv, top + np.log(total)
                rel = 2 * ds.max() + 8 * U32F + (len(s) + 2) * U32F
                # f16's denormal P, against a maximum that may lag the row's by 8 (base 2): as if all keys were there
                mag = p @ np.abs(vv)
                tol[row, cols] = HALF[out] * np.abs(o[row, cols]) + (rel * 2 + up) * mag \
                    + tiny * np.abs(vv).sum(0) / total + (2.0 ** -25 if out == torch.float16 else 0.0)
                ltol[h, row] = ds.max() + (len(s) + 8) * U32F + 4 * U32F * abs(lse[h, row])
    return o, lse, tol, ltol


def weights(q_rows, lse_rows, k, ctx, rows, w, *, heads, scale, decay):
    """(w_out [B][KV][cap], tolerance), rows past ctx NaN. q_rows(b, h, r) / lse_rows(b, h, r) give a query; rows[b]: the
    list of query indices of sequence b, in order (None: no query)."""
    B, KV, cap, D = k.shape
    out = np.full((B, KV, cap), np.nan)
    tol = np.zeros_like(out)
    for b in range(B):
        c, n = ctx[b], len(rows[b])
        for g in range(KV):
            got, off, terms = np.zeros(c), np.zeros(c), 0
            for i, r in enumerate(rows[b]):
                if r is None:
                    continue
                sees = np.arange(c) <= c - n + i
                for h in range(g * heads // KV, (g + 1) * heads // KV):
                    l = lse_rows(b, h, r)
                    if np.isinf(l):  # -inf saw nothing; exp(s - inf) is 0
                        continue
                    kk = np.where(sees[:, None], k[b, g, :c], 0.0)
                    s = kk @ q_rows(b, h, r) * scale
                    ds = (D * np.abs(kk) @ np.abs(q_rows(b, h, r)) * scale + 3 * np.abs(s) + 3 * abs(l)) * U32F
                    e = np.where(sees, np.exp(s - l), 0.0)
                    got += e
                    off += e * (ds + 8 * U32F)
                    terms += 1
            old = np.zeros(c) if w is None or decay == 0 else decay * w[b, g, :c]
            out[b, g, :c] = old + got
            tol[b, g, :c] = off + (terms + 4) * U32F * (got + np.abs(old))
    return out, tol


def evict_keep(w, pos, seen, budget, recent, sinks):
    """The rows of a list that stay, ascending."""
    n = len(w)
    if n <= budget:
        return list(range(n))
    key = lambda j: (not (pos[j] < sinks or pos[j] >= seen - recent),  # noqa: E731
                     -(-np.inf if np.isnan(w[j]) else float(w[j])), j)
    return sorted(sorted(range(n), key=key)[:budget])


def evict_rows(w, pos, seen, budget, recent, sinks):
    """For each row of the list afterwards, the row that is in it."""
    keep = evict_keep(w, pos, seen, budget, recent, sinks)
    n = min(len(w), budget)
    left = list(range(n))
    holes = sorted(set(left) - set(keep))
    for to, src in zip(holes, [j for j in keep if j >= n]):
        left[to] = src
    return left
