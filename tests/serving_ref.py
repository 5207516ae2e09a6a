"""Plain 64-bit forms of the serving operators, with the error that each kernel's
roundings can make: |out - y| <= bound for every element.

A score s = c q.k formed with relative error e per product is off by at most
e scale sum |q_i k_i|; weights then by the factor exp(+-2 err) together with their
sum; what the weights and the output are rounded to comes on top (half a step:
2^-24 f32, 2^-8 bf16). A value v in [2^e, 2^(e+1)) split into two bf16 with the high
one cut leaves at most 2^(e-7), half a step of which (2^-8 of the power of two below
it, at most 2^(e-8)) is 2^(e-16): 2^-16."""
import math

import numpy as np

F32, BF16, SPLIT = 2.0 ** -24, 2.0 ** -8, 2.0 ** -16


def bf16_bits(x):
    u = np.ascontiguousarray(x, np.float32).view(np.uint32).astype(np.uint64)
    return ((u + 0x7fff + ((u >> 16) & 1)) >> 16).astype(np.uint16)


def bf16_value(bits):
    return (np.asarray(bits, np.uint16).astype(np.uint32) << 16).view(np.float32)


def attend(q, k, v, scale, p_step, out_step):
    """One query row [D] over keys k, v [n, D] in 64 bits: (y, bound)."""
    q, k, v = (np.asarray(x, np.float64) for x in (q, k, v))
    if k.shape[0] == 0:
        return np.zeros(v.shape[1]), np.zeros(v.shape[1])
    s = (k @ q) * scale
    err = ((k.shape[1] + 4) * F32 + SPLIT) * scale * np.abs(k * q).sum(axis=1).max() \
        + 4 * F32 * np.abs(s).max()
    w = np.exp(s - s.max())
    w /= w.sum()
    y, size = w @ v, w @ np.abs(v)
    rel = math.expm1(2 * err) + (k.shape[0] + 8) * F32 + p_step
    return y, rel * size + out_step * np.abs(y) + 1e-30


def paged_keys(pages, table, n, h):
    """Keys (or values) of a sequence's first n positions that have a page."""
    ps, rows = pages.shape[2], []
    for i, page in enumerate(table):
        if i * ps < n and 0 <= page < pages.shape[0]:
            rows.append(pages[page, h, :n - i * ps])
    return np.concatenate(rows).astype(np.float64) if rows else np.zeros((0, pages.shape[3]))


def paged_decode(q, kp, vp, table, lens, scale=None, p_step=SPLIT, out_step=F32):
    b, hq, d = q.shape
    g = hq // kp.shape[1]
    y, bound = np.zeros((b, hq, d)), np.zeros((b, hq, d))
    for i in range(b):
        for h in range(kp.shape[1]):
            n = max(0, int(lens[i]))
            k, v = paged_keys(kp, table[i], n, h), paged_keys(vp, table[i], n, h)
            for r in range(h * g, h * g + g):
                y[i, r], bound[i, r] = attend(q[i, r], k, v, scale or 1 / math.sqrt(d), p_step, out_step)
    return y, bound


def packed_prefill(q, k, v, offsets, scale=None, p_step=SPLIT, out_step=F32, rows=None):
    """(y, bound), rows outside every sequence NaN; rows: only these packed rows."""
    t, hq, d = q.shape
    g = hq // k.shape[1]
    y, bound = np.full((t, hq, d), np.nan), np.zeros((t, hq, d))
    for a, e in zip(offsets, offsets[1:]):
        for r in range(a, e):
            if rows is not None and r not in rows:
                continue
            for h in range(hq):
                y[r, h], bound[r, h] = attend(q[r, h], k[a:r + 1, h // g], v[a:r + 1, h // g],
                                              scale or 1 / math.sqrt(d), p_step, out_step)
    return y, bound


def append(pages, new, table, starts, offsets):
    """pages [P, Hkv, ps, D] with new [T, Hkv, D] written (any types that cast)."""
    out, ps = pages.copy(), pages.shape[2]
    for b, start in enumerate(starts):
        for i, row in enumerate(range(offsets[b], offsets[b + 1])):
            pos = int(start) + i
            if row < 0 or row >= new.shape[0] or pos < 0 or pos // ps >= table.shape[1]:
                continue
            page = table[b][pos // ps]
            if 0 <= page < pages.shape[0]:
                out[page, :, pos % ps] = new[row]
    return out


def sample(logits, u, t=None, k=None, p=None, m=None):
    """The token of one row, from the sorted words."""
    z = np.asarray(logits, np.float64)
    t = 1.0 if t is None else float(t)
    if np.isnan(z).any():
        return int(np.flatnonzero(np.isnan(z))[0])
    if not t > 0 or not np.isfinite(z.max()):
        return int(np.argmax(z))
    order = np.lexsort((np.arange(z.size), -z))
    if k is not None and 0 < k < z.size:
        order = order[:k]
    w = np.exp((z[order] - z[order[0]]) / t)
    w[z[order] == -np.inf] = 0.0
    if p is not None and p < 1:
        mass = np.cumsum(w)
        n = min(int(np.searchsorted(mass, max(float(p), 0.0) * mass[-1])) + 1, w.size)
        order, w = order[:n], w[:n]
    if m is not None and m > 0:
        n = max(1, int((w >= float(m)).sum()))
        order, w = order[:n], w[:n]
    mass = np.cumsum(w)
    u = min(max(float(u), 0.0), 1 - 2.0 ** -24) if u == u else 0.0
    return int(order[int(np.searchsorted(mass, u * mass[-1], side="right"))])
