"""64-bit plain forms of the paged-cache operators, on the CPU, one token and one head at a time."""
import math

import numpy as np
import torch


def cached_rows(cache, table_row, page, L):
    """[L, width] rows of one sequence."""
    return torch.stack([cache[int(table_row[r // page]), r % page] for r in range(L)]) if L else cache[0, :0]


def attention(q, k_cache, v_cache, table, ctx, cu, Hq, Hkv, hd, scale, mask=None):
    """(out, absolute) fp64 [T, Hq*hd]: the attention and sum_i p_i |v_i| (what a rounding of p can move); rows that no
    sequence owns are NaN.  Pages out of range are rows that nobody sees."""
    T, page, n_pages = q.shape[0], k_cache.shape[1], k_cache.shape[0]
    out = torch.full((T, Hq, hd), math.nan, dtype=torch.float64)
    mag = torch.zeros((T, Hq, hd), dtype=torch.float64)
    G = Hq // Hkv
    for b, L in enumerate(ctx):
        n = cu[b + 1] - cu[b]
        t = torch.arange(L)
        pg = table[b].long()[t // page]
        good = (pg >= 0) & (pg < n_pages)
        k = k_cache[pg.clamp(0, n_pages - 1), t % page].double().view(L, Hkv, hd)
        v = v_cache[pg.clamp(0, n_pages - 1), t % page].double().view(L, Hkv, hd)
        for i in range(n):
            row = cu[b] + i
            seen = good & (t < L - n)
            for j in range(n):
                if L - n + j >= 0 and ((j <= i) if mask is None else (
                        j // 64 < mask.shape[1] and (int(mask[row, j // 64]) >> (j % 64)) & 1)):
                    seen[L - n + j] = good[L - n + j]
            if not seen.any():
                out[row] = 0.0
                continue
            qq = q[row].double().view(Hkv, G, hd)
            s = torch.einsum("kgd,lkd->kgl", qq, k[seen]) * scale
            p = torch.softmax(s, -1)
            out[row] = torch.einsum("kgl,lkd->kgd", p, v[seen]).reshape(Hq, hd)
            mag[row] = torch.einsum("kgl,lkd->kgd", p, v[seen].abs()).reshape(Hq, hd)
    return out.flatten(1), mag.flatten(1)


def rotate(x, cos, sin, interleaved):
    """x fp64 [..., hd], cos / sin fp64 [rot/2]."""
    y = x.clone()
    h = cos.shape[0]
    for m in range(h):
        i, j = (2 * m, 2 * m + 1) if interleaved else (m, m + h)
        y[..., i] = x[..., i] * cos[m] - x[..., j] * sin[m]
        y[..., j] = x[..., j] * cos[m] + x[..., i] * sin[m]
    return y


def sample_row(x, u, T=1.0, k=0, p=1.0, mp=0.0):
    """(token, log-probability) of one row by sorting it; weights in 64 bits, their running sum in 80; settings as fp32
    values."""
    x = np.asarray(x, dtype=np.float64)
    if np.isnan(x).any():
        return -1, math.nan
    order = np.argsort(-x, kind="stable")
    order = order[x[order] != -math.inf]
    if not order.size:
        return -1, -math.inf
    top = x[order[0]]
    if not T > 0:
        return int(order[0]), 0.0
    T = min(T, 2.0 ** 20)
    with np.errstate(invalid="ignore"):
        w = np.where(x[order] == top, 1.0, np.exp((x[order] - top) / T))
    run = np.cumsum(w.astype(np.longdouble))
    n = min(w.size, k) if k > 0 else w.size
    if p < 1:
        n = min(n, max(1, int(np.searchsorted(run[:n], p * run[n - 1], side="left")) + 1))
    if mp > 0:
        n = max(1, min(n, int((w >= mp).sum())))
    goal = min(max(u, 0.0), 1 - 2.0 ** -24) * run[n - 1]
    r = int(np.searchsorted(run[:n], goal, side="right"))
    return int(order[r]), math.log(w[r]) - float(np.log(run[n - 1]))
