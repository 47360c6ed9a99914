"""The paged key/value operators in 64 bits, one row at a time, with the error that a kernel
of a given type may have.

Rounding of a value to type t is off by at most u = eps(t) / 2 of it; fp32 by w = 2^-24.
With A = sum_j p_j |v_j| (p the exact weights) an attention output may differ by
  u |o|                 rounding of the output,
  u A                   rounding of the weights before the product with v (16-bit types),
  2 (d + e) A           errors of the weights: d = largest error of a score, e of the exponential,
where a score of n products in fp32 is off by at most
  d = w ((dim + 4) scale sum |q k| + 8 |z|)
(dim + 4 roundings: the products' sum, the scale, cap and bias; |z| after them for the
change to powers of two, the subtraction of the maximum and the argument's rounding), and the
exponential by e: 2^-21 for fp32 (the argument's and the result's last places), u / 8 for
16-bit types.  The sums over n keys add at most 2 n w A for any order.
"""
import math

import torch


def unit(dtype):
    return torch.finfo(dtype).eps / 2


def gather(pages, table, seq, n):
    """[kv_heads, n, dim] in 64 bits; pages outside the pool are zeros."""
    ps, count = pages.shape[2], pages.shape[0]
    rows = []
    for i in range(-(-n // ps)):
        page = int(table[seq, i])
        rows.append(pages[page] if 0 <= page < count else torch.zeros_like(pages[0]))
    x = torch.cat(rows, 1)[:, :n] if rows else pages[0][:, :0]
    return x.double()


def attend(q, k, v, positions, scale, window=0, prefix=0, cap=0.0, slopes=None, dtype=torch.float32):
    """q [rows, heads, dim] at `positions`, k and v [kv_heads, n, dim]: (out, lse, bound of out,
    bound of lse) in 64 bits."""
    rows, heads, dim = q.shape
    kv, n = k.shape[:2]
    out = torch.zeros(rows, heads, dim, dtype=torch.float64, device=q.device)
    lse = torch.full((rows, heads), -math.inf, dtype=torch.float64, device=q.device)
    tol, tol_l = torch.zeros_like(out), torch.zeros_like(lse)
    u, w = unit(dtype), 2.0 ** -24
    wide = dtype == torch.float32
    e = 2.0 ** -21 if wide else u / 8
    j = torch.arange(n, device=q.device)
    for r in range(rows):
        p = int(positions[r])
        seen = j <= p
        if window:
            seen &= p - j < window
        seen |= j < prefix
        seen = seen.nonzero().flatten()
        if not len(seen):
            continue
        for h in range(heads):
            kk, vv = k[h // (heads // kv), seen], v[h // (heads // kv), seen]
            x = q[r, h].double()
            z = (kk @ x) * scale
            size = (kk.abs() @ x.abs()) * abs(scale)
            if cap:
                z = cap * torch.tanh(z / cap)
            if slopes is not None:
                z = z - float(slopes[h]) * (p - seen).abs()
                size = size + abs(float(slopes[h])) * (p - seen).abs()
            m = z.max()
            pr = torch.exp(z - m)
            total = pr.sum()
            pr = pr / total
            out[r, h] = pr @ vv
            lse[r, h] = m + torch.log(total)
            a = pr @ vv.abs()
            d = float((w * ((dim + 4) * size + 8 * (z.abs() + m.abs()))).max())
            rel = (0 if wide else u) + 2 * (d + e) + 2 * len(seen) * w
            tol[r, h] = u * out[r, h].abs() + rel * a + torch.finfo(dtype).tiny
            tol_l[r, h] = d + e + len(seen) * w + 4 * w * (abs(float(lse[r, h])) + 1)
    return out, lse, tol, tol_l


def rotate(x, cos, sin, interleaved):
    """Rotary positions of x [rows, heads, dim] in 64 bits with cos, sin [rows, dims / 2], and
    the bound of an fp32 evaluation: two products and a sum, each rounded once."""
    x, cos, sin = x.double(), cos.double()[:, None], sin.double()[:, None]
    dims = 2 * cos.shape[-1]
    out, tol = x.clone(), torch.zeros_like(x)
    ia = torch.arange(0, dims, 2) if interleaved else torch.arange(dims // 2)
    ib = ia + 1 if interleaved else ia + dims // 2
    a, b = x[..., ia], x[..., ib]
    out[..., ia] = a * cos - b * sin
    out[..., ib] = a * sin + b * cos
    w = 2.0 ** -24
    tol[..., ia] = 2 * w * ((a * cos).abs() + (b * sin).abs())
    tol[..., ib] = 2 * w * ((a * sin).abs() + (b * cos).abs())
    return out, tol


def capped(q, k, v, positions, scale, cap, slopes=None, dtype=torch.float32):
    """`attend` under a cap, with the bound that holds where scores pass it: a product that is off
    by w (dim + 4) scale sum |q k| moves the capped score by no more than tanh moves over that
    interval (nothing, where it is flat).  tanh by 1 - 2 / (1 + 2^y) is off by at most 10 w of
    itself where it starts, at 0.54 (2^y: 4 w, and 2 w for y; the quotient: 4 w; of 0.46, and w
    for the difference), less after it and below, so that z is off by 10 w |z|, and by 8 w |z| as
    there.  (out, tol)"""
    rows, heads, dim = q.shape
    kv = k.shape[0]
    out = torch.zeros(rows, heads, dim, dtype=torch.float64, device=q.device)
    tol = torch.zeros_like(out)
    u, w = unit(dtype), 2.0 ** -24
    wide = dtype == torch.float32
    for r in range(rows):
        p = int(positions[r])
        for h in range(heads):
            kk, vv = k[h // (heads // kv), :p + 1], v[h // (heads // kv), :p + 1]
            x = q[r, h].double()
            z = (kk @ x) * scale
            off = w * (dim + 4) * (kk.abs() @ x.abs()) * abs(scale)
            low, z, high = (cap * torch.tanh(y / cap) for y in (z - off, z, z + off))
            d = torch.maximum((high - z).abs(), (z - low).abs()) + 18 * w * z.abs()
            if slopes is not None:
                bias = float(slopes[h]) * (p - torch.arange(p + 1, device=q.device))
                z, d = z - bias, d + 8 * w * bias.abs()
            m = z.max()
            pr = torch.exp(z - m)
            pr = pr / pr.sum()
            out[r, h] = pr @ vv
            rel = 2 * (8 * w * m.abs() + (2.0 ** -21 if wide else u / 8)) + 2 * (p + 1) * w + (0 if wide else u)
            # a weight is off by its score's error and by the sum's, the weights' mean of them all
            tol[r, h] = u * out[r, h].abs() + 2 * (pr * d.expm1()) @ vv.abs() + ((pr * d.expm1()).sum() * 2 + rel) * (pr @ vv.abs())
    return out, tol + torch.finfo(dtype).tiny
