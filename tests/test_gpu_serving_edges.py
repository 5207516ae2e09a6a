"""The serving operators at the ends of their inputs' range, against the 64-bit forms."""
import numpy as np
import pytest

import serving_ref as ref
from test_gpu_serving import P_STEP, STEP, check, check_sample, decode, floats, make_pages, packed, prompts, sample

pytestmark = pytest.mark.gpu


# ---- sampling ---------------------------------------------------------------------

def check_min_p(rt, z, u, k, m, p=None):
    """check_sample at temperature 1, with min_p's words told by their logits: exp(-d) >= m where d <= -log m.
    (exp(-d) is below 1 for every d > 0, but 1 in 64 bits from d = 2^-54 down, so that ref.sample takes
    such words for ties of the first at m = 1.)"""
    want = []
    for row, top_k in zip(z, k):
        order = np.lexsort((np.arange(row.size), -row))
        order = order[:top_k] if 0 < top_k < row.size else order
        d = np.float64(row[order[0]]) - row[order].astype(np.float64)
        mass = np.cumsum(np.exp(-d))
        n = order.size if p is None else int(np.searchsorted(mass, np.float64(np.float32(p)) * mass[-1])) + 1
        n = max(1, min(n, int((d <= -np.log(np.float64(np.float32(m)))).sum())))
        want.append(int(order[np.searchsorted(mass[:n], min(np.float32(u), 1 - 2.0 ** -24) * mass[n - 1], side="right")]))
        if m < 1:  # (the two forms are one)
            assert want[-1] == ref.sample(row, np.float32(u), None, top_k, None if p is None else np.float32(p), np.float32(m))
    n = len(z)
    got = sample(rt, z, np.full(n, u, np.float32), k=k, m=[m] * n, p=None if p is None else [p] * n)
    assert got.tolist() == want, (u, m, p)

def short_spans(v):
    """Rows whose words to choose from are two that lie close together: the others are at -inf, or out of
    top_k's reach."""
    rng = np.random.default_rng(v)
    step = lambda x: np.nextafter(np.float32(x), np.float32(-np.inf))  # noqa: E731
    pairs = [(1.0, step(1.0)), (10.0, step(10.0)), (-7.5, step(-7.5)), (1e-30, 0.0), (0.0, -1e-30), (1e-42, 0.0),
             (1e30, step(1e30)), (3.0, 3.0 - 1e-5), (0.0, -1e-3)]
    rows, ks = [], []
    for a, b in pairs:
        near = np.full(v, -np.inf, np.float32)
        near[rng.permutation(v)[:2]] = a, b
        deep = np.where(near > -np.inf, near, np.float32(min(a, b) - abs(a) - 20))
        rows += [near, deep.astype(np.float32)]
        ks += [0, 2]
    return np.array(rows, np.float32), ks


@pytest.mark.parametrize("v", [2, 5, 1030, 151936])
def test_sample_min_p_over_a_short_span(rt, v):
    """min_p's border far behind the last word that weighs anything; rows that one and several
    workgroups share."""
    z, ks = short_spans(v)
    for u in (0.0, 0.3, 0.9, 1.0):
        for m in (0.02, 0.05, 0.1, 0.5, 0.9999999):
            check_min_p(rt, z, u, ks, m)
            check_min_p(rt, z, u, ks, m, p=0.7)


@pytest.mark.parametrize("v", [2, 5, 1030, 151936])
def test_sample_min_p_of_one(rt, v):
    """min_p = 1 leaves the first word and its ties, however near the next ones come; above 1 the first alone."""
    z, ks = short_spans(v)
    for u in (0.0, 0.3, 0.9, 1.0):
        for m in (1.0, 1.0000001, 7.0):
            check_min_p(rt, z, u, ks, m)
            check_min_p(rt, z, u, ks, m, p=0.7)


@pytest.mark.parametrize("v", [60, 3000, 30000, 151936])
def test_sample_min_p_of_one_among_many(rt, v):
    """The same with hundreds and thousands of words a hair below the first's ties."""
    rng = np.random.default_rng(v)
    near = np.where(rng.random(v) < 0.3, 1e-30, rng.uniform(0, 1e-30, v))
    z = np.stack([near, -near, np.where(rng.random(v) < 0.9, near, -5.0)]).astype(np.float32)
    for u in (0.0, 0.4, 0.9):
        for k in (0, 50, v - 1):
            check_min_p(rt, z, u, [k] * 3, 1.0)


@pytest.mark.parametrize("v", [3, 1030, 151936])
@pytest.mark.parametrize("t", [1e4, 1e7, 1e30, 3e38])
def test_sample_min_p_at_high_temperatures(rt, v, t):
    rng = np.random.default_rng(v)
    z = (2 * rng.standard_normal((6, v))).astype(np.float32)
    z[3:, 0] = -np.inf
    for u in (0.3, 0.9):
        for m in (0.05, 0.5, 0.999):
            for k in (0, 2, 7):
                check_sample(rt, z, np.full(6, u, np.float32), t=[t] * 6, k=[k] * 6, m=[m] * 6)


# ---- packed prompts ---------------------------------------------------------------

TYPES = [(64, "bf16", "bf16"), (128, "bf16", "bf16"), (256, "bf16", "bf16"), (64, "f32", "f32"), (128, "f32", "f32"),
         (256, "f32", "f32"), (128, "f32", "bf16"), (256, "bf16", "f32"), (80, "f32", "f32")]


@pytest.mark.parametrize("copies", [1, 60])
@pytest.mark.parametrize("d,qk,out", TYPES)
def test_packed_prefill_first_keys_that_weigh_nothing(rt, d, qk, out, copies):
    """Scores of -inf over a sequence's first 32 (and 64) keys and far below 0 after them: the others' softmax
    all the same, whichever kernel takes the rows. A row with nothing but -inf is 0."""
    rng = np.random.default_rng(d)
    q, k, v, offsets = prompts(rng, [130, 40, 100], 2, 1, d, qk)
    q[..., :2] = 1.0
    k[..., 1] = -256.0  # (times the scale and log2 e: some -133, -185 and -259)
    dead = {0: 32, 130: 32, 170: 64}
    for a, n in dead.items():
        k[a:a + n, :, 0] = -np.inf
    for scale in (0.36, 0.5, 0.7):
        y = packed(rt, q, qk, k, v, offsets, out, scale=scale, copies=copies)
        for a, e in zip(offsets, offsets[1:]):
            first = a + dead[int(a)]
            assert not y[a:first].any()
            for row in range(first, e):
                for h in range(2):
                    want, bound = ref.attend(q[row, h], k[first:row + 1, 0], v[first:row + 1, 0], scale, P_STEP[out], STEP[out])
                    check(y[row, h], want, bound)


@pytest.mark.parametrize("copies", [1, 60])
@pytest.mark.parametrize("d,qk,out", TYPES)
def test_packed_prefill_scores_past_the_exponent(rt, d, qk, out, copies):
    """Scores of 10^10, where half a step of f32 is past the exponents of a weight: each row's largest takes
    it all (the next is thousands below; a score is off by (d + 4) 2^-24 of its products)."""
    rng = np.random.default_rng(d)
    q, k, v, offsets = prompts(rng, [1, 1, 1, 1, 30, 40, 100], 2, 1, d, qk)
    q, k = q * np.float32(2 ** 17), k * np.float32(2 ** 17)
    y = packed(rt, q, qk, k, v, offsets, out, copies=copies)
    step = P_STEP[out] + STEP[out] + 8 * ref.F32
    seen = 0
    for a, e in zip(offsets, offsets[1:]):
        for row in range(a, e):
            for h in range(2):
                s = k[a:row + 1, 0].astype(np.float64) @ q[row, h].astype(np.float64) / np.sqrt(d)
                size = (np.abs(k[a:row + 1, 0].astype(np.float64)) @ np.abs(q[row, h].astype(np.float64))).max() / np.sqrt(d)
                top = np.sort(s)[::-1]
                if s.size > 1 and top[0] - top[1] < 1000 + 4 * (d + 4) * ref.F32 * size:
                    continue
                seen += 1
                want = v[a + int(np.argmax(s)), 0].astype(np.float64)
                check(y[row, h], want, step * np.abs(want))
    assert seen > 300


# ---- paged decode -----------------------------------------------------------------

def test_paged_decode_lengths_up_to_the_last_position(rt):
    """A table of 2^31 - 16 positions, most of them without a page, and lengths in its last tile."""
    rng, ps = np.random.default_rng(0), 8176
    entries = (2 ** 31 - 16) // ps
    assert entries * ps == 2 ** 31 - 16
    lens = [2 ** 31 - 1, 2 ** 31 - 31, 100, 0, 2 ** 31 - 32]
    table = np.full((5, entries), -1, np.int32)
    table[0, [0, 1000, entries - 1]] = 2, 0, 1
    table[1, entries - 1], table[2, 0], table[4, entries - 1] = 0, 1, 2
    q = floats(rng, (5, 4, 64), "f32")
    kp, vp = (floats(rng, (3, 1, ps, 64), "bf16") for _ in range(2))
    y = decode(rt, q, "f32", kp, vp, "bf16", table, lens)
    check(y, *ref.paged_decode(q, kp, vp, table, lens))


# ---- scales -------------------------------------------------------------------------

@pytest.mark.parametrize("d,pk", [(64, "bf16"), (128, "f32"), (256, "bf16"), (80, "f32")])
def test_small_scales(rt, d, pk):
    """A scale of 2^-120 d^-1/2 over scores that are 2^120 times as large is an ordinary softmax."""
    rng = np.random.default_rng(d)
    big, scale = np.float32(2.0 ** 60), float(np.float32(d ** -0.5)) * 2.0 ** -120
    lens = [70, 1, 200]
    q = floats(rng, (3, 4, d), "f32") * big
    kp, vp, table = make_pages(rng, lens, 2, 16, d, pk)
    y = decode(rt, q, "f32", kp * big, vp, pk, table, lens, scale=scale)
    check(y, *ref.paged_decode(q, kp * big, vp, table, lens, scale=scale))
    for copies in (1, 60):
        q, k, v, offsets = prompts(rng, [40, 100], 2, 1, d, "f32")
        y = packed(rt, q * big, "f32", k * big, v, offsets, scale=scale, copies=copies)
        check(y, *ref.packed_prefill(q * big, k * big, v, offsets, scale=scale))


@pytest.mark.parametrize("d,pk", [(64, "bf16"), (128, "f32"), (256, "bf16"), (80, "f32")])
def test_the_least_scale(rt, d, pk):
    """Under the least f32 above 0 every key that a row sees weighs the same, and no other any."""
    rng, scale = np.random.default_rng(d), float(np.finfo(np.float32).smallest_subnormal)
    lens = [70, 1, 200, 0]
    q = floats(rng, (4, 4, d), "f32")
    kp, vp, table = make_pages(rng, lens, 2, 16, d, pk)
    table[0, 1] = -1
    y = decode(rt, q, "f32", kp, vp, pk, table, lens, scale=scale)
    check(y, *ref.paged_decode(q, kp, vp, table, lens, scale=scale))
    for copies in (1, 60):
        q, k, v, offsets = prompts(rng, [40, 100], 2, 1, d, "f32")
        y = packed(rt, q, "f32", k, v, offsets, scale=scale, copies=copies)
        check(y, *ref.packed_prefill(q, k, v, offsets, scale=scale))


# ---- what f32 keeps -----------------------------------------------------------------

def cut(x, parts):
    """x >= 0 as the kernels' bf16 parts: cut ones and a rounded last one."""
    rest, total = np.asarray(x, np.float32), np.zeros(np.shape(x))
    for _ in range(parts - 1):
        high = ((np.maximum(rest.view(np.uint32), 1) - 1) & 0xffff0000).astype(np.uint32).view(np.float32)
        rest, total = rest - high, total + high
    return total + ref.bf16_value(ref.bf16_bits(rest))


def attend_exact(q, k, v, scale, weights=lambda w: w):
    """A row [D] with one element that is not 0: its scores are one product each, of three parts (two sums
    round). Scores within S of 0 and c cost a difference of two 4 2^-24 S for the sums, 2 2^-24 S for c and as
    much for its own rounding; a quotient takes twice that. Then n weights in a sum, their exponentials and
    the division."""
    s = (k.astype(np.float64) @ q.astype(np.float64)) * scale
    w = np.exp(s - s.max())
    y = weights(w) @ v / w.sum()
    rel = np.expm1(16 * ref.F32 * np.abs(s).max()) + (s.size + 8) * ref.F32
    return y, rel * (w @ np.abs(v)) / w.sum() + ref.F32 * np.abs(y)


@pytest.mark.parametrize("copies", [1, 60])
@pytest.mark.parametrize("d", [64, 128, 256])
def test_f32_rows_keep_24_bits(rt, d, copies):
    """An f32 q enters whole and an f32 output takes whole weights, on the matrix cores too: two bf16 parts
    of either would pass the bound (which the same test shows)."""
    rng = np.random.default_rng(d)
    counts, scale = [8] * 12, 0.5
    q, k, v, offsets = prompts(rng, counts, 2, 1, d, "f32")
    at = rng.integers(0, d, q.shape[:2])
    one = np.zeros_like(q)
    np.put_along_axis(one, at[..., None], rng.uniform(4, 16, at.shape + (1,)).astype(np.float32), 2)
    packed_y = packed(rt, one, "f32", k, v, offsets, scale=scale, copies=copies)
    # the last rows' queries over the same keys, one page a sequence
    last, kp, vp = offsets[1:] - 1, np.zeros((12, 1, 16, d), np.float32), np.zeros((12, 1, 16, d), np.float32)
    for b, a in enumerate(offsets[:-1]):
        kp[b, 0, :8], vp[b, 0, :8] = k[a:a + 8, 0], v[a:a + 8, 0]
    table = np.arange(12, dtype=np.int32)[:, None]
    paged_y = [decode(rt, one[last], "f32", kp, vp, pk, table, [8] * 12, scale=scale) for pk in ("bf16", "f32")]
    over = {"q": 0, "weights": 0}
    for b, a in enumerate(offsets[:-1]):
        for row in range(a, a + 8):
            for h in range(2):
                keys, vals = k[a:row + 1, 0], v[a:row + 1, 0].astype(np.float64)
                want, bound = attend_exact(one[row, h], keys, vals, scale)
                check(packed_y[row, h], want, bound)
                if row == last[b]:
                    for y in paged_y:
                        check(y[b, h], want, bound)
                    over["q"] += (np.abs(attend_exact(cut(one[row, h], 2), keys, vals, scale)[0] - want) > bound).any()
                    over["weights"] += (np.abs(attend_exact(one[row, h], keys, vals, scale, lambda w: cut(w, 2))[0] - want) > bound).any()
    assert over["q"] > 0 and over["weights"] > 0, over
