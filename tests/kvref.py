"""The 4-bit K/V cache and attention over it in numpy, in 64 bits, from their definitions."""
import numpy as np

GROUP = 32


def scales(x):
    """Scale of each group of 32 along the last axis (f64)."""
    g = np.asarray(x, np.float64).reshape(*x.shape[:-1], -1, GROUP)
    hi, lo = g.max(-1), g.min(-1)
    d = np.clip(np.where(hi >= -lo, hi, lo) / -8, -8160, 8160)
    m, e = np.frexp(d)
    d = np.ldexp(np.rint(np.ldexp(m, 8)), e - 8)           # 8 significant bits, ties to even
    return np.where(np.abs(d) < 2.0 ** -14, np.rint(d * 2.0 ** 24) * 2.0 ** -24, d)  # f16's subnormals


def held(x):
    """What the cache holds for finite x."""
    d = scales(x)[..., None]
    g = np.asarray(x, np.float64).reshape(*x.shape[:-1], -1, GROUP)
    q = np.clip(np.rint(g / np.where(d == 0, 1, d)), -8, 7)
    return (np.where(d == 0, 0, q) * d).reshape(x.shape)


def held_pair(k, v):
    """K and V [rows, heads, dim] as held, values that are not finite among them."""
    bad = ~(np.isfinite(k).all(-1) & np.isfinite(v).all(-1))
    gv = np.isfinite(v.reshape(*v.shape[:-1], -1, GROUP)).all(-1).repeat(GROUP, -1)
    hk = held(np.where(np.isfinite(k), k, 0))
    return np.where(bad[..., None], np.nan, hk), held(np.where(gv, v, 0))


def rows_visible(pos, length, window, causal):
    j = np.arange(max(length, 0))
    ok = np.ones(j.size, bool) if pos >= 0 else np.zeros(j.size, bool)
    if causal:
        ok &= j <= pos
    if window:
        ok &= j > pos - window
    return ok


def attention(q, k, v, scale, window=0, softcap=0.0, causal=True, absent=None):
    """q [n, q_heads, dim]: the last n tokens of the sequence whose cached rows are k, v [len, heads, dim]
    (f64).  Returns out and, for tolerances, sum_j p_j |v_j|, the relative error of p that
    roundings of f32 sums allow (from the magnitudes in the scores), and an absolute one."""
    n, hq, dim = q.shape
    length, heads, _ = k.shape
    g = hq // heads
    out, mag, eps, floor = np.zeros(q.shape), np.zeros(q.shape), np.zeros((n, hq, 1)), np.zeros(q.shape)
    for t in range(n):
        pos = length - n + t
        ok = rows_visible(pos, length, window, causal)
        if absent is not None:
            ok = ok & ~absent
        if not ok.any():
            continue
        for h in range(hq):
            kk, vv, qq = k[ok, h // g], v[ok, h // g], q[t, h].astype(np.float64)
            s = kk @ qq * scale
            # q in parts of 22 bits of the row's largest.  The products' f32 sums: a group's 32 products of codes and
            # q (exact each), and a multiplication and addition for each of dim / 32 groups
            part = np.abs(kk).sum(1) * np.abs(qq).max() * 2.0 ** -22
            add = (np.abs(kk) @ np.abs(qq)) * (dim / 32 + 16) * 2.0 ** -24
            err = (part + add) * abs(scale) + np.abs(s) * 2.0 ** -22
            if softcap:
                s = softcap * np.tanh(s / softcap)
                err = err + softcap * 2.0 ** -21 + np.abs(s) * 2.0 ** -22  # tanh and its argument
            p = np.exp(s - s.max())
            p /= p.sum()
            out[t, h] = p @ vv
            # p enters as f16 parts of p * 2^13 and more (the largest p is 2^13 at least): below f16's smallest
            # normal number an error of half of 2^-24, 2^-38 of the largest p, whatever p is
            mag[t, h] = p @ np.abs(vv)
            floor[t, h] = 2.0 ** -38 * np.abs(vv).sum(0)
            eps[t, h] = np.nanmax(err) + 2.0 ** -21  # + exp2 and p's parts
    return out, mag, eps, floor


def tolerance(out, mag, eps, floor, keys, f16):
    """|kernel - out| at most: p's relative errors enter the sum and its divisor; f32 sums of `keys` products in
    pieces of 32; with f16 operands p is rounded to 11 bits, and out is."""
    tol = floor + mag * (2 * eps + (keys / 32 + 16) * 2.0 ** -24)
    if f16:
        tol = tol + mag * 2 * 2.0 ** -11 + np.abs(out) * 2.0 ** -11 + 2.0 ** -25
    return tol + np.abs(out) * 2.0 ** -22 + 1e-30
