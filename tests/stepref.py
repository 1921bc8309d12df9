"""What stands around the K/V cache in a serving step, in numpy and 64 bits, from the definitions in include/arfq.h."""
import numpy as np

import kvref


def plan(page, add, held, pages, free, n_free, tokens):
    """Sequence after sequence, page after page.  pages and free are copied."""
    pages, free = pages.copy(), free.copy()
    batch, most = pages.shape
    n_free = min(max(int(n_free), 0), free.size)
    ceil = lambda n: -(-n // page)
    fine = [0 <= int(h) <= most * page for h in held]
    pool, freed, start = [], [0], [0]
    for b in range(batch):
        h, a = int(held[b]), int(add[b])
        if fine[b] and a <= 0:
            pool += [int(p) for p in pages[b, ceil(max(0, h + a)):ceil(h)]]
        freed.append(len(pool))
        start.append(start[-1] + max(a, 0))
    there, wanted, taken = n_free + len(pool), 0, [0]
    held_next, lens = [], []
    positions, slots = np.full(tokens, -1, np.int64), np.full(tokens, -1, np.int64)
    for b in range(batch):
        h, a = int(held[b]), int(add[b])
        new, got = max(0, h + a), 0
        ok = fine[b]
        if a > 0:
            ok = ok and start[b + 1] <= tokens and ceil(new) <= most
            if ok:
                more = ceil(new) - ceil(h)
                wanted += more
                ok = more == 0 or wanted <= there
                if ok:
                    got = more
                    for i in range(more):
                        at = taken[-1] + i
                        pages[b, ceil(h) + i] = pool[at] if at < len(pool) else free[n_free - 1 - (at - len(pool))]
                    for i, p in enumerate(range(h, new)):
                        positions[start[b] + i] = p
                        slots[start[b] + i] = int(pages[b, p // page]) * page + p % page
        taken.append(taken[-1] + got)
        held_next.append(new if ok else h)
        lens.append(new if ok else 0)
    for i in range(taken[-1], len(pool)):
        at = n_free + len(pool) - 1 - i
        if at < free.size:
            free[at] = pool[i]
    return dict(pages=pages, free=free, held_next=held_next, lens=lens, start=np.minimum(start, tokens), taken=taken, freed=freed,
                n_free_next=[min(there - taken[-1], free.size)], positions=positions, slots=slots)


def rope(x, positions, freqs, axes, neighbours, gain=1.0, inverse=False):
    """x [tokens, heads, dim].  Returns out and the |a| + |b| of each value's pair (0 where nothing turns)."""
    x = x.astype(np.float64)
    out, mag = x.copy(), np.zeros(x.shape)
    half = len(freqs)
    for i in range(half):
        w = positions[axes[i], :x.shape[0]].astype(np.float64)[:, None] * freqs[i] * (-1 if inverse else 1)
        p, q = (2 * i, 2 * i + 1) if neighbours else (i, i + half)
        a, b = x[..., p], x[..., q]
        out[..., p], out[..., q] = (a * np.cos(w) - b * np.sin(w)) * gain, (a * np.sin(w) + b * np.cos(w)) * gain
        mag[..., p] = mag[..., q] = (np.abs(a) + np.abs(b)) * abs(gain)
    return out, mag


def rope_tolerance(out, mag, angle, f16):
    """A cosine's argument is at most pi / 4, rounded twice in 32 bits (2 * 0.79 * 2^-24), its series adds 3 roundings of
    values up to 1 and leaves out 2^-27, the gain one more: 6 * 2^-24 in all, and two roundings for the products and
    their sum.  In 64 bits an angle is off by 4 roundings of 2^-53."""
    tol = mag * (8 * 2.0 ** -24 + np.abs(angle).max(initial=0.0) * 2.0 ** -51) + 1e-37
    return tol + np.abs(out) * 2.0 ** -11 + 2.0 ** -25 if f16 else tol


def lora(x, ids, a, b, scale, base):
    """Returns out and what its rounding goes by: sum_r |B| sum_k |A| |x|, sum_r |B| |h| and max |h| sum_r |B|, times
    |scale|."""
    ids, rows, n = np.asarray(ids), x.shape[0], b.shape[1]
    out = np.zeros((rows, n)) if base is None else base.astype(np.float64)
    mags = np.zeros((3, rows, n))
    for e in np.unique(ids[(ids >= 0) & (ids < a.shape[0])]):
        t = np.flatnonzero(ids == e)
        ae, be, xt = a[e].astype(np.float64), b[e].astype(np.float64), x[t].astype(np.float64)
        s = 1.0 if scale is None else float(scale[e])
        h, ab = xt @ ae.T, np.abs(be)
        out[t] += s * (h @ be.T)
        mags[0, t], mags[1, t] = abs(s) * (np.abs(xt) @ np.abs(ae).T @ ab.T), abs(s) * (np.abs(h) @ ab.T)
        mags[2, t] = abs(s) * np.abs(h).max(1)[:, None] * ab.sum(1)
    return out, mags


def lora_tolerance(out, mags, base, k, rank):
    """A_e x: at most one rounding for each product and sum of k values, in parts or not; B_e h: one for each of rank; h
    in two f16 parts keeps 22 bits of its row's largest; the scale, and the sum with base."""
    per_sum = min(k, 2048) + 64  # (parts of k: products of one accumulator, and the parts)
    own = 0.0 if base is None else np.abs(base)
    return mags[0] * per_sum * 2.0 ** -24 + mags[1] * (rank + 8) * 2.0 ** -24 + mags[2] * 2.0 ** -22 + (np.abs(out) + own) * 2.0 ** -23 + 1e-37


def bounds(k, page):
    """[blocks, heads, 2, dim] of held keys [len, heads, dim]: the largest and the smallest, NaN where a key is."""
    out = []
    for i in range(0, k.shape[0], page):
        part = k[i:i + page]
        out.append(np.stack([part.max(0), part.min(0)], 1))  # (numpy's extremes of NaN are NaN)
    return np.array(out).reshape(-1, k.shape[1], 2, k.shape[2])


def choose(q, bnd, seen, count, first, last, negative=False, absent=None):
    """Blocks that the heads q [group, dim] of a row choose of bnd [>= seen, 2, dim]."""
    if seen <= count:
        return np.arange(seen)
    q = q.astype(np.float64) * (-1 if negative else 1)
    hi, lo = bnd[:seen, 0].T, bnd[:seen, 1].T
    score = (np.where(q < 0, 0, q) @ hi + np.where(q < 0, q, 0) @ lo).max(0)
    rank = np.where(np.isnan(score), np.inf, score)
    if absent is not None:
        rank = np.where(absent[:seen], -np.inf, rank)
    rule = (np.arange(seen) < first) | (np.arange(seen) >= seen - last)
    rest = np.flatnonzero(~rule)
    best = rest[np.argsort(-rank[rest], kind="stable")][:count - first - last]
    return np.sort(np.concatenate([np.flatnonzero(rule), best]))


def attend_blocks(q, k, v, page, scale, count, first, last, softcap=0.0, absent=None, bnd=None):
    """q [n, q_heads, dim]: the last n tokens of a sequence whose held rows are k, v [len, heads, dim].  Returns what
    kvref.attention does, the most keys of a row, and the blocks [n, heads, count]."""
    n, hq, dim = q.shape
    length, heads, _ = k.shape
    g = hq // heads
    res = [np.zeros(q.shape), np.zeros(q.shape), np.zeros((n, hq, 1)), np.zeros(q.shape)]
    chosen = np.full((n, heads, count), -1, np.int64)
    bnd = bounds(k, page) if bnd is None else bnd
    for t in range(n):
        pos = length - n + t
        if pos < 0:
            continue
        seen = pos // page + 1
        for h in range(heads):
            mine = slice(h * g, (h + 1) * g)
            blocks = choose(q[t, mine], bnd[:, h], seen, count, first, last, scale < 0, absent)
            chosen[t, h, :blocks.size] = blocks
            keys = (blocks[:, None] * page + np.arange(page)).ravel()
            keys = keys[keys <= pos]
            gone = None if absent is None else absent[keys // page]
            got = kvref.attention(q[t:t + 1, mine], k[keys, h:h + 1], v[keys, h:h + 1], scale, softcap=softcap, absent=gone)
            for all_, one in zip(res, got):
                all_[t, mine] = one[0]
    return (*res, min(length, count * page), chosen)


def lora_norm_tolerance(out, base, k, rank):
    """On the norm of all errors, where x, A and B have random signs and one size.  A sum of n terms is rounded n times, by at most
    2^-24 of a partial sum each; these errors have signs of their own and partial sums are no larger than the sum in root
    mean square, so their norm is at most sqrt(n) 2^-24 of the sums'.  n is k, then rank; h in two f16 parts is off by 2^-22
    of its row's largest, at most four times its root mean square; scale and product round h twice more, the sum with base once."""
    own = out if base is None else out - base
    return np.linalg.norm(own) * ((np.sqrt(k) + np.sqrt(rank) + 4) * 2.0 ** -24 + 2.0 ** -20) + np.linalg.norm(out) * 2.0 ** -24
