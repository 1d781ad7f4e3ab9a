"""Plain 64-bit CPU forms of the serving operators of a kept full-attention layer: causal attention of packed prompts,
and a cache of e4m3 codes in pages with one power-of-two scale per (page, KV head).  Written from the definitions; the
tests compare the CUDA path with them."""
import math

import torch


def e4m3(x):
    """x (float64) on the e4m3 grid: nearest, ties to even; saturating at 448; NaN stays."""
    a = x.abs().clamp(min=2.0 ** -6, max=448.0)
    step = 2.0 ** (torch.frexp(a)[1].double() - 4)
    r = torch.round(x.clamp(-448.0, 448.0) / step) * step
    return torch.where(torch.isnan(x), x, r.clamp(-448.0, 448.0))


def page_scale(x):
    """The smallest power of two s >= 2^-64 with amax / s <= 448, over the finite values of x."""
    fin = x[torch.isfinite(x)]
    amax = float(fin.abs().max()) if fin.numel() else 0.0
    e = -64
    while amax > 448.0 * 2.0 ** e:
        e += 1
    return 2.0 ** e


def append(codes, scale, table_row, length, x):
    """Write x [n,G,D] to the positions length - n .. length - 1.  codes [P,G,L,D], scale [P,G] float64, in place."""
    L, n = codes.shape[2], x.shape[0]
    start = max(length - n, 0)
    x = x[n - (length - start):].double()
    for p in range(start // L, -(-length // L)):
        page = int(table_row[p]) if p < len(table_row) else -1
        if page < 0 or page >= codes.shape[0]:
            continue
        lo, hi = max(start, p * L), min(length, p * L + L)
        had = lo - p * L
        for g in range(codes.shape[1]):
            rows = x[lo - start:hi - start, g]
            s = page_scale(rows)
            if had:
                s = max(s, float(scale[page, g]))
                codes[page, g, :had] = e4m3(codes[page, g, :had] * (float(scale[page, g]) / s))
            codes[page, g, had:hi - p * L] = e4m3(rows / s)
            scale[page, g] = s


def softmax_attend(q, k, v, seen, scale):
    """q [n,D], k, v [m,D], seen [n,m]: (o, lse, sum p|v|, per row the largest scale * sum |q k| of a seen key), float64.
    A key that a row does not see has no part in it, whatever it holds."""
    o = torch.zeros(q.shape, dtype=torch.float64)
    mag, big = torch.zeros_like(o), torch.zeros(q.shape[0], dtype=torch.float64)
    lse = torch.full((q.shape[0],), -math.inf, dtype=torch.float64)
    q, k, v = q.double(), k.double(), v.double()
    for i in range(q.shape[0]):
        kk, vv = k[seen[i]], v[seen[i]]
        if kk.shape[0]:
            s = kk @ q[i] * scale
            lse[i] = torch.logsumexp(s, 0)
            p = torch.exp(s - lse[i])
            o[i], mag[i] = p @ vv, p @ vv.abs()
            big[i] = (kk.abs() @ q[i].abs() * scale).max()
    return o, lse, mag, big


def prompt_attention(q, k, v, cu, cuk=None, scale=None):
    """q [T,H,D], k, v [Tk,G,D], lists cu, cuk: (o [T,H,D], lse [H,T], sum p|v| [T,H,D], score size [T,H])."""
    T, H, D = q.shape
    R = H // k.shape[1]
    cuk = cu if cuk is None else cuk
    scale = D ** -0.5 if scale is None else scale
    o, lse = torch.zeros(q.shape, dtype=torch.float64), torch.full((H, T), -math.inf, dtype=torch.float64)
    mag, big = torch.zeros_like(o), torch.zeros(T, H, dtype=torch.float64)
    for b in range(len(cu) - 1):
        nq, nk = cu[b + 1] - cu[b], cuk[b + 1] - cuk[b]
        seen = torch.arange(nk)[None] <= torch.arange(nq)[:, None] + nk - nq
        rows, keys = slice(cu[b], cu[b + 1]), slice(cuk[b], cuk[b + 1])
        for h in range(H):
            o[rows, h], lse[h, rows], mag[rows, h], big[rows, h] = softmax_attend(q[rows, h], k[keys, h // R], v[keys, h // R],
                                                                                seen, scale)
    return o, lse, mag, big


def attend(kc, ks, vc, vs, table_row, length, q, scale=None):
    """q [t,H,D] at the positions length - t ..; codes [P,G,L,D] and scales [P,G] float64: (o, lse [H,t], mag, big)."""
    t, H, D = q.shape
    G, L = kc.shape[1], kc.shape[2]
    scale = D ** -0.5 if scale is None else scale
    n = max(length, 0)
    pages = [int(table_row[p]) if p < len(table_row) else -1 for p in range(-(-n // L))]
    ok = [0 <= p < kc.shape[0] for p in pages]
    there = torch.tensor([ok[j // L] for j in range(n)], dtype=torch.bool)
    use = torch.tensor([p if o else 0 for p, o in zip(pages, ok)], dtype=torch.long)
    o, lse = torch.zeros(q.shape, dtype=torch.float64), torch.full((H, t), -math.inf, dtype=torch.float64)
    mag, big = torch.zeros_like(o), torch.zeros(t, H, dtype=torch.float64)
    seen = (torch.arange(n)[None] <= torch.arange(length - t, length)[:, None]) & there[None]
    for h in range(H):
        g = h // (H // G)
        k = (kc[use, g] * ks[use, g][:, None, None]).reshape(-1, D)[:n]
        v = (vc[use, g] * vs[use, g][:, None, None]).reshape(-1, D)[:n]
        o[:, h], lse[h], mag[:, h], big[:, h] = softmax_attend(q[:, h], k, v, seen, scale)
    return o, lse, mag, big
