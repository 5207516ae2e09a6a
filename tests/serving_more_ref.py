"""Plain 64-bit forms of the 8-bit cache, of attention behind shared prefixes and of
the logits' adjustments. Attention's bounds are serving_ref's: an 8-bit value is
(code - 128) s exactly, its score c s_k (q . codes) and its weight p s_v each take
two roundings more, and joining the records of a row a few, which 8 half steps of
f32 cover (`MORE`). Over 8-bit rows q and the weights go into the products in f16, whose
half step is 2^-11: q in parts that leave 2^-22 of an element and 2^-39 of the row's
largest, less than SPLIT of the sums of |q k|; weights in one part behind a bf16 output
(`F16`), in two, 2^-22 and so less than SPLIT, behind an f32 one. A weight p s_v is a
multiple of 2^-24 where the largest so far is 2^10 at least: half of that, 2^-35 of the
largest, for each key and at most 127 units of its code (`grain`). Behind a shared
prefix the weights of bf16 rows are one bf16 part (2^-8) for a bf16 output."""
import math

import numpy as np

import serving_ref as ref

MORE = 8 * ref.F32
F16 = 2.0 ** -11


def p_step(kind, out):
    """What weights are rounded by, beside f32's own roundings."""
    return (ref.SPLIT if out == "f32" else F16 if kind == "q8" else ref.BF16) + MORE


def grain(q, k, vs, scale):
    """Of one query row over keys k [n, D] whose values have the scales vs [n]."""
    if k.shape[0] == 0:
        return 0.0
    s = (np.asarray(k, np.float64) @ np.asarray(q, np.float64)) * scale
    w = np.exp(s - s.max())
    return k.shape[0] * 2.0 ** -35 * 127 * float((w * np.abs(vs)).max() / w.sum())


def decode8(q, kc, vc, ks, vs, table, lens, scale=None, out="f32"):
    """(y, bound) of decode attention over codes and scales."""
    step = ref.BF16 if out == "bf16" else ref.F32
    y, bound = ref.paged_decode(q, value(kc, ks), value(vc, vs), table, lens, scale, p_step("q8", out), step)
    g, c = q.shape[1] // kc.shape[1], scale or 1 / math.sqrt(q.shape[2])
    for i in range(q.shape[0]):
        for h in range(q.shape[1]):
            n = max(0, int(lens[i]))
            k = ref.paged_keys(value(kc, ks), table[i], n, h // g)
            bound[i, h] += grain(q[i, h], k, ref.paged_keys(vs[..., None], table[i], n, h // g)[:, 0], c)
    return y, bound


def encode(x):
    """Rows [..., D] f32 as (codes, scales), the encoder's rule in f32."""
    x = np.asarray(x, np.float32)
    with np.errstate(invalid="ignore", over="ignore"):
        amax = np.abs(x).max(axis=-1)
        s = np.maximum(amax, np.float32(1e-12)) / np.float32(127)
        s = np.where(np.isfinite(amax), s, np.float32(np.nan)).astype(np.float32)
        code = np.clip(np.rint(x / s[..., None]), -127, 127) + 128
    return np.where(np.isnan(s)[..., None], 128, code).astype(np.uint8), s


def value(codes, scales):
    """What codes [..., D] and scales [...] stand for, in 64 bits."""
    return (codes.astype(np.float64) - 128) * np.asarray(scales, np.float64)[..., None]


def read(pages, table, starts, offsets, total):
    """Rows [total, Hkv, D] of pages [P, Hkv, ps, D]; NaN outside every sequence."""
    _, hkv, ps, d = pages.shape
    out = np.full((total, hkv, d), np.nan)
    for b, start in enumerate(starts):
        for i, row in enumerate(range(max(offsets[b], 0), min(offsets[b + 1], total))):
            pos, out[row] = int(start) + i + max(-offsets[b], 0), 0
            if 0 <= pos and pos // ps < table.shape[1] and 0 <= table[b][pos // ps] < pages.shape[0]:
                out[row] = pages[table[b][pos // ps], :, pos % ps]
    return out


def shared(q, kp, vp, prefixes, prefix_lens, groups, table, lens, scale=None, out="f32", vs=None):
    """(y, bound) over pages of values; vs: the scales of V's codes."""
    step, weights = ref.BF16 if out == "bf16" else ref.F32, p_step("bf16" if vs is None else "q8", out)
    b, hq, d = q.shape
    g = hq // kp.shape[1]
    y, bound = np.zeros((b, hq, d)), np.zeros((b, hq, d))
    for i in range(b):
        for h in range(kp.shape[1]):
            parts = [(table[i], lens[i])]
            for n in range(len(prefixes)):
                if groups[n] <= i < groups[n + 1]:
                    parts.insert(0, (prefixes[n], prefix_lens[n]))
            k, v = (np.concatenate([ref.paged_keys(x, t, max(0, int(n)), h) for t, n in parts])
                    for x in (kp, vp))
            if vs is not None:
                scales = np.concatenate([ref.paged_keys(vs[..., None], t, max(0, int(n)), h) for t, n in parts])[:, 0]
            for r in range(h * g, h * g + g):
                c = scale or 1 / math.sqrt(d)
                y[i, r], bound[i, r] = ref.attend(q[i, r], k, v, c, weights, step)
                bound[i, r] += 0 if vs is None else grain(q[i, r], k, scales, c)
    return y, bound


def adjust(z, step, tokens=None, offsets=None, prompts=None, repetition=None, frequency=None,
           presence=None, bias_words=None, bias=None, bias_offsets=None, mask=None, mask_rows=None):
    """(y, bound): four roundings of f32 at most, each half a step of the largest value on the
    way (the quotient, n frequency + presence, the difference, the sum), and the output's."""
    y = np.asarray(z, np.float64).copy()
    size = np.abs(np.where(np.isfinite(y), y, 0))
    rows, vocab = y.shape
    for b in range(rows):
        if tokens is not None:
            words = np.asarray(tokens[max(0, offsets[b]):max(0, offsets[b + 1])])
            skip = max(0, int(prompts[b])) if prompts is not None else 0
            good = (words >= 0) & (words < vocab)
            count = np.bincount(words[skip:][good[skip:]], minlength=vocab)
            seen = np.bincount(words[good], minlength=vocab) > 0
            r = float(repetition[b]) if repetition is not None else 1.0
            if r > 0:
                with np.errstate(invalid="ignore"):
                    y[b] = np.where(seen, np.where(y[b] > 0, y[b] / r, y[b] * r), y[b])
            size[b] = np.maximum(size[b], np.abs(np.where(np.isfinite(y[b]), y[b], 0)))
            off = (count * (float(frequency[b]) if frequency is not None else 0.0)
                   + (count > 0) * (float(presence[b]) if presence is not None else 0.0))
            y[b] -= off
            size[b] += np.abs(off)
        if bias is not None:
            for e in range(max(0, bias_offsets[b]), min(max(0, bias_offsets[b + 1]), bias.size)):
                w = int(bias_words[e])
                later = [x for x in bias_words[e + 1:bias_offsets[b + 1]] if x == w]
                if 0 <= w < vocab and not later:
                    y[b, w] += float(bias[e])
                    if np.isfinite(bias[e]):
                        size[b, w] += abs(float(bias[e]))
        m = -1 if mask is None else b if mask_rows is None else int(mask_rows[b])
        if mask is not None and 0 <= m < mask.shape[0]:
            bits = np.unpackbits(np.ascontiguousarray(mask[m]).view(np.uint8), bitorder="little")
            y[b, bits[:vocab] == 0] = -np.inf
    with np.errstate(invalid="ignore"):
        return y, 4 * ref.F32 * size + step * np.where(np.isfinite(y), np.abs(y), 0) * 1.01 + 1e-30
