"""64-bit evaluation of the paged-cache operators from their definition -- TEST INFRASTRUCTURE ONLY.

`attention` also returns, for every output element, how far a correct kernel may be off. With P the
normalised weights and u the rounding of a probability that is fed to the tensor cores in the input
type (half a step, relative: finfo.eps / 2; 0 for float32 inputs):
  |dO| <= (u + 2 ds) (P |V|) + u_out |O| + half the smallest step of the output type
(float16 values below 2^-14 stand 2^-24 apart whatever their size, so their rounding is off by up to 2^-25)
where ds bounds the error of a score (and so the relative error of an exponential, in numerator and
denominator alike): products and sums of D terms in float32, (D + 8) 2^-24 scale sum |q_d k_d|, the
cap's tanh 2^-20 cap, the bias 2^-22 |slope rel|, and 2^-18 for exponentials, running sums and joins.
"""
from __future__ import annotations

import math

import torch

U = {torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8, torch.float32: 2.0 ** -24}
STEP = {torch.float16: 2.0 ** -25, torch.bfloat16: 2.0 ** -134, torch.float32: 2.0 ** -150}


def rows_of(cache, pages, n):
    """The first n tokens stored in `pages`, as float64 [n, Hk, D]."""
    if n == 0:
        return cache.new_zeros((0, *cache.shape[2:])).double()
    idx = torch.arange(n, device=cache.device)
    return cache[pages.long()[idx // cache.shape[1]], idx % cache.shape[1]].double()


def attention(q, k_cache, v_cache, table, lens, scale, causal=False, starts=None, cap=0.0, window=None, slopes=None,
              prefix_table=None, prefix_len=0, out_dtype=None):
    """(O, LSE, tolerance of O, tolerance of LSE) in float64; rows of no request are NaN."""
    dev, (rows, hq, d) = q.device, q.shape
    hk = k_cache.shape[2]
    starts = list(range(len(lens) + 1)) if starts is None else starts
    out = torch.full((rows, hq, d), math.nan, dtype=torch.float64, device=dev)
    tol = torch.zeros_like(out)
    lse = torch.full((hq, rows), math.nan, dtype=torch.float64, device=dev)
    lse_tol = torch.zeros_like(lse)
    u_p = 0.0 if q.dtype == torch.float32 else U[q.dtype]
    u_out, step = U[out_dtype or q.dtype], STEP[out_dtype or q.dtype]
    for i, n in enumerate(lens):
        a, b = starts[i], starts[i + 1]
        if a == b:
            continue
        k, v = rows_of(k_cache, table[i], n), rows_of(v_cache, table[i], n)
        if prefix_len:
            k = torch.cat([rows_of(k_cache, prefix_table, prefix_len), k])
            v = torch.cat([rows_of(v_cache, prefix_table, prefix_len), v])
        at = torch.arange(k.shape[0], device=dev)
        pos = prefix_len + n - (b - a) + torch.arange(b - a, device=dev)
        rel = at[None] - pos[:, None]
        see = torch.ones_like(rel, dtype=torch.bool)
        if causal:
            see &= rel <= 0
        if window is not None and window[0] >= 0:
            see &= rel >= -window[0]
        if window is not None and window[1] >= 0:
            see &= rel <= window[1]
        used = see.any(0)  # slots no row sees may hold anything
        k = torch.where(used[:, None, None], k, torch.zeros_like(k))
        v = torch.where(used[:, None, None], v, torch.zeros_like(v))
        for h in range(hq):
            kh, vh, qh = k[:, h * hk // hq], v[:, h * hk // hq], q[a:b, h].double()
            x = qh @ kh.t() * scale
            ds = (d + 8) * 2.0 ** -24 * abs(scale) * (qh.abs() @ kh.abs().t()) + 2.0 ** -18
            if cap:
                x = cap * torch.tanh(x / cap)
                ds = ds + 2.0 ** -20 * cap
            if slopes is not None:
                x = x + float(slopes[h]) * rel
                ds = ds + 2.0 ** -22 * (float(slopes[h]) * rel).abs()
            x = x.masked_fill(~see, -math.inf)
            empty = ~see.any(1)
            m = torch.where(empty, torch.zeros_like(x[:, 0]) if x.shape[1] else x.new_zeros(b - a),
                            x.amax(1) if x.shape[1] else x.new_zeros(b - a))
            e = torch.exp(x - m[:, None])
            s = e.sum(1)
            p = e / torch.where(empty, torch.ones_like(s), s)[:, None]
            o = p @ vh
            off = (u_p + 2 * torch.where(see, ds, torch.zeros_like(ds)).amax(1) if x.shape[1] else x.new_zeros(b - a))
            out[a:b, h] = o
            tol[a:b, h] = off[:, None] * (p @ vh.abs()) + u_out * o.abs() + step + 1e-30
            lse[h, a:b] = torch.where(empty, torch.full_like(m, -math.inf), m + torch.log(s))
            lse_tol[h, a:b] = off - u_p + 2.0 ** -22 * (m.abs() + 1)
    return out, lse, tol, lse_tol


def assert_attention(got, ref, tol, what):
    """Every element of the rows that belong to a request within its tolerance."""
    mine = ~ref.isnan()
    g = got.double()
    assert torch.isfinite(g[mine]).all(), f"{what}: non-finite output"
    over = ((g - ref).abs() - tol)[mine]
    assert over.numel() == 0 or float(over.max()) <= 0, (
        f"{what}: worst element {float(over.max()):.3e} beyond its tolerance, "
        f"largest ratio {float(((g - ref).abs() / tol)[mine].max()):.2f}")


def plan(cached, new, table, free, page, rows, begin=0):
    """(table, seq_lens, cu, slots, positions, free_end) as Python lists."""
    table = [list(r) for r in table]
    width = len(table[0]) if table else 0
    at, cu, slots, positions = begin, [0], [], []
    for i, (c, n) in enumerate(zip(cached, new)):
        held, after = min(-(-c // page), width), min(-(-(c + n) // page), width)
        for p in range(held, after):
            table[i][p] = free[at] if at < len(free) else -1
            at += 1
        for pos in range(c, c + n):
            p = pos // page
            ok = p < width and table[i][p] >= 0
            slots.append(table[i][p] * page + pos % page if ok else -1)
            positions.append(pos)
        cu.append(cu[-1] + n)
    slots, positions = slots[:rows], positions[:rows]
    slots += [-1] * (rows - len(slots))
    positions += [0] * (rows - len(positions))
    return table, [c + n for c, n in zip(cached, new)], cu, slots, positions, min(at, len(free))


def rotate(x, positions, theta):
    """Rotate-half RoPE of [T, H, D] in float64 (a row at position None is kept)."""
    half = x.shape[-1] // 2
    inv = torch.tensor([theta ** (-2.0 * i / x.shape[-1]) for i in range(half)], dtype=torch.float64, device=x.device)
    ang = positions.double()[:, None] * inv
    c, s = ang.cos()[:, None], ang.sin()[:, None]
    a, b = x[..., :half].double(), x[..., half:2 * half].double()
    return torch.cat([a * c - b * s, a * s + b * c, x[..., 2 * half:].double()], -1)
