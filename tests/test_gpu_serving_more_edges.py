"""The operators over 8-bit pages and shared prefixes and the logits' adjustments at the ends of
their inputs' range, against the 64-bit forms."""
import numpy as np
import pytest

import serving_more_ref as more
import serving_ref as ref
from test_gpu_cache8 import decode8
from test_gpu_logits import I32, adjust, biases, history, masks
from test_gpu_serving import STEP, check, decode, floats, make_pages
from test_gpu_shared import call

pytestmark = pytest.mark.gpu

TYPES = [("bf16", "bf16"), ("f32", "f32"), ("f32", "bf16")]


def lay(rows, ps=16):
    """Rows [n, ...] of every kv head as pages [P, hkv, ps, ...]: position j in page j / ps."""
    n, hkv = rows.shape[:2]
    pages = np.zeros((-(-n // ps) * ps, hkv, *rows.shape[2:]), rows.dtype)
    pages[:n] = rows
    return np.ascontiguousarray(np.moveaxis(pages.reshape(-1, ps, *pages.shape[1:]), 2, 1))


def both8(rt, q, qk, k, v, out, scale=None, first=0, ps=16):
    """Decode attention over 8-bit rows k, v = (codes [n, hkv, d], scales [n, hkv]) of all sequences of
    q: the paged call's result, and the shared call's, the first `first` positions (whole pages) as a prefix."""
    n, b = k[0].shape[0], q.shape[0]
    kc, vc, ks, vs = (lay(x, ps) for x in (k[0], v[0], k[1], v[1]))
    table = np.tile(np.arange(kc.shape[0], dtype=np.int32), (b, 1))
    cut = first // ps
    y = decode8(rt, q, qk, kc, vc, ks, vs, table, [n] * b, out, scale)
    z = call(rt, q, qk, None, None, (kc, ks, vc, vs), "q8", table[:1], [cut * ps], [0, b], table[:, cut:], [n - cut * ps] * b,
             out, scale)
    return y, z


def want8(q, k, v, out, scale=None):
    """What both have to be, with its bound."""
    kc, vc, ks, vs = (lay(x) for x in (k[0], v[0], k[1], v[1]))
    table = np.tile(np.arange(kc.shape[0], dtype=np.int32), (q.shape[0], 1))
    return more.decode8(q, kc, vc, ks, vs, table, [k[0].shape[0]] * q.shape[0], scale, out)


def check8(rt, q, qk, k, v, out, scale=None, first=0):
    want = want8(q, k, v, out, scale)
    for y in both8(rt, q, qk, k, v, out, scale, first):
        check(y, *want)


def rows8(x):
    return more.encode(np.asarray(x, np.float32))


# ---- scales of V's rows ---------------------------------------------------------------

@pytest.mark.parametrize("d,ps", [(64, 16), (128, 16), (256, 16), (96, 16), (128, 7)])
@pytest.mark.parametrize("qk,out", TYPES)
def test_a_value_scale_of_zero_under_the_largest_score(rt, d, ps, qk, out):
    """Keys whose values' scale is 0, whose scores lie hundreds above those of the tiles before: they take all of
    the weight, and the row is what the others have left, next to nothing."""
    rng = np.random.default_rng(d)
    n, hkv = 400, 64  # (and 16 sequences: a wave has several tiles of each)
    k = np.zeros((n, hkv, d), np.float32)
    k[[37, 70, 203, 390], :, 0] = np.array([60, 200, 300, 90])[:, None]
    v = rows8(rng.standard_normal((n, hkv, d)))
    v[1][[37, 70, 203, 390]] = 0
    q = np.zeros((16, hkv, d), np.float32)
    q[:, :, 0] = 1
    for first in (0, 64, 208):
        for y in both8(rt, q, qk, rows8(k), v, out, 1.0, first, ps):
            assert np.isfinite(y).all() and np.abs(y).max() <= 1e-20


@pytest.mark.parametrize("d", [64, 128, 256, 96])
@pytest.mark.parametrize("qk,out", TYPES)
@pytest.mark.parametrize("large", [1e24, 1e26, 1e38])
def test_values_of_zero_beside_very_large_ones(rt, d, qk, out, large):
    """Rows of zeros (the least scale there is) weigh as much as rows of 1e38: in one tile and in tiles of several waves,
    before and behind the large ones."""
    rng = np.random.default_rng(d)
    n = 1500
    for where in (np.arange(8), n - 1 - np.arange(8), rng.permutation(n)[:8]):
        v = np.zeros((n, 1, d), np.float32)
        v[where] = large * rng.uniform(0.5, 1, (8, 1, d))
        k, q = floats(rng, (n, 1, d), "f32"), floats(rng, (1, 2, d), qk)
        check8(rt, q, qk, rows8(k), rows8(v), out, first=n // 2)


@pytest.mark.parametrize("qk,out", TYPES)
def test_values_of_zero_beside_very_large_ones_in_a_waves_tiles(rt, qk, out):
    """The same over so many keys that every wave has several tiles."""
    rng = np.random.default_rng(1)
    n, d = 150000, 128
    k, q = rows8(floats(rng, (n, 1, d), "f32")), floats(rng, (1, 1, d), qk)
    for where in (np.arange(900), n - 1 - np.arange(900), rng.permutation(n)[:900]):
        v = np.zeros((n, 1, d), np.float32)
        v[where] = 1e26 * rng.uniform(0.5, 1, (900, 1, d))
        check8(rt, q, qk, k, rows8(v), out, first=n // 2)


@pytest.mark.parametrize("d", [64, 128, 256])
@pytest.mark.parametrize("qk,out", TYPES)
def test_the_sum_keeps_light_keys_beside_very_large_values(rt, d, qk, out):
    """1500 keys of weight exp(-12), with values of 0, beside one of weight 1 and 1e38."""
    n = 1500
    for at in (0, 700, n - 1):
        k, v = np.zeros((n, 1, d), np.float32), np.zeros((n, 1, d), np.float32)
        k[at, :, 0], v[at] = 12, 1e38
        q = np.zeros((1, 4, d), np.float32)
        q[:, :, 0] = 1
        check8(rt, q, qk, rows8(k), rows8(v), out, 1.0, first=800)


# ---- scores ------------------------------------------------------------------------------

@pytest.mark.parametrize("d", [64, 128, 256, 96])
@pytest.mark.parametrize("qk,out", TYPES)
@pytest.mark.parametrize("size", [1e8, 3e9, 1e12, 1e30])
def test_8bit_scores_far_past_their_steps(rt, d, qk, out, size):
    """Scores whose steps in f32 are larger than what a scale adds to them: the largest ones, equal to each
    other, share the row. (Their weights are then the same number p, so that the row is the mean of their values but
    for what weights are rounded by, MORE, the output's step and the grain.)"""
    rng = np.random.default_rng(d)
    n = 100
    tops = [3, 40, 41, 77]
    k = np.zeros((n, 1, d), np.float32)
    k[:, :, 0] = -size * rng.uniform(0.1, 1, (n, 1))
    k[tops, :, 0] = size
    v = rng.standard_normal((n, 1, d)) * 10.0 ** rng.integers(-6, 7, (n, 1, 1))
    v[tops] = rng.standard_normal((4, 1, d)) * 10.0 ** np.array([5, 4, 5, 3])[:, None, None]
    v = rows8(v)
    q = np.zeros((1, 2, d), np.float32)
    q[:, :, 0] = 1
    value = more.value(*v)[tops, 0]
    want = value.mean(axis=0)
    bound = (more.p_step("q8", out) * np.abs(value).mean(axis=0) + STEP[out] * np.abs(want)
             + n * 2.0 ** -35 * 127 * v[1][tops].max())
    for first in (0, 32, 64):
        for y in both8(rt, q, qk, rows8(k), v, out, 1.0, first):
            check(y, np.broadcast_to(want, y.shape), np.broadcast_to(bound, y.shape))


@pytest.mark.parametrize("d", [64, 128, 256, 96])
@pytest.mark.parametrize("qk,out", TYPES)
@pytest.mark.parametrize("size", [1e-34, 1e-36, 2e-38])
def test_8bit_queries_near_0(rt, d, qk, out, size):
    """Queries of 1e-36 over keys of 1e36: scores as of any other ones."""
    rng = np.random.default_rng(d)
    n, hkv = 150, 2
    k, v = rows8(rng.standard_normal((n, hkv, d)) / (size * 10)), rows8(rng.standard_normal((n, hkv, d)))
    q = floats(rng, (2, 4, d), qk, std=size * 10)
    check8(rt, q, qk, k, v, out, first=64)


@pytest.mark.parametrize("d", [64, 128, 256, 96])
@pytest.mark.parametrize("qk,out", TYPES)
@pytest.mark.parametrize("scale", [1e34, 1e36, 1e38])
def test_8bit_scales_of_the_scores_near_the_largest(rt, d, qk, out, scale):
    """A softmax scale near f32's end, over queries as small as it is large."""
    rng = np.random.default_rng(d)
    n, hkv = 150, 2
    k, v = rows8(rng.standard_normal((n, hkv, d))), rows8(rng.standard_normal((n, hkv, d)))
    q = floats(rng, (2, 4, d), qk, std=0.2 / scale)
    check8(rt, q, qk, k, v, out, scale, first=64)


@pytest.mark.parametrize("d,ps", [(64, 16), (128, 16), (256, 16), (96, 16), (128, 7)])
@pytest.mark.parametrize("qk,out", TYPES)
def test_8bit_scales_of_the_scores_near_0(rt, d, ps, qk, out):
    """A softmax scale of 2e-38 over queries and keys of 1e19: their products pass f32 before the scale."""
    rng = np.random.default_rng(d)
    n, hkv = 150, 2
    k, v = rows8(1e19 * rng.standard_normal((n, hkv, d))), rows8(rng.standard_normal((n, hkv, d)))
    q = floats(rng, (2, 4, d), qk, std=3e18)
    want = want8(q, k, v, out, 2e-38)
    for y in both8(rt, q, qk, k, v, out, 2e-38, 64, ps):
        check(y, *want)


def shared_and_paged(rt, q, qk, k, v, kind, out, scale, first):
    """Rows k, v [n, hkv, d] of all sequences: the shared call's result, the first `first` (whole pages) as a prefix, and
    the paged call's."""
    n, b = k.shape[0], q.shape[0]
    kp, vp = lay(k), lay(v)
    table = np.tile(np.arange(kp.shape[0], dtype=np.int32), (b, 1))
    cut = first // 16
    y = call(rt, q, qk, kp, vp, None, kind, table[:1], [cut * 16], [0, b], table[:, cut:], [n - cut * 16] * b, out, scale)
    return y, decode(rt, q, qk, kp, vp, kind, table, [n] * b, out, scale)


@pytest.mark.parametrize("d", [64, 128, 256, 96])
@pytest.mark.parametrize("kind", ["bf16", "f32"])
@pytest.mark.parametrize("qk,out", TYPES)
@pytest.mark.parametrize("power", [24, 31, 34, 60, 100])
def test_shared_scores_far_past_their_steps(rt, d, kind, qk, out, power):
    """Scores of 2^24 to 2^100, whose steps pass 2^7 from 2^31 on: the largest one alone weighs, and the row is
    its value, but for an f32 output's two roundings (the weight is a power of two, its inverse one too)."""
    rng = np.random.default_rng(power)
    n = 90
    for first in (0, 48):
        k = floats(rng, (n, 1, d), "bf16")
        k[:, :, 0] = rng.permutation(n)[:, None] + 1 - n // 2
        k[:, :, 0] = ref.bf16_value(ref.bf16_bits(k[:, :, 0] * np.float32(2.0 ** (power // 2))))
        v = floats(rng, (n, 1, d), "bf16")
        q = np.zeros((3, 4, d), np.float32)
        q[:, :, 0] = np.float32(2.0 ** (power - power // 2)) * 1.25
        want = v[k[:, 0, 0].argmax(), 0].astype(np.float64)
        for y in shared_and_paged(rt, q, qk, k, v, kind, out, 1.0, first):
            check(y, np.broadcast_to(want, y.shape), np.broadcast_to(4 * STEP["f32"] * np.abs(want), y.shape))


# ---- values --------------------------------------------------------------------------------

@pytest.mark.parametrize("d", [64, 128, 256])
@pytest.mark.parametrize("qk,out", TYPES)
def test_shared_values_near_the_largest(rt, d, qk, out):
    """bf16 values of 3e36 at most, under scores that rise and fall by 2^7.8 from tile to tile, in many heads (so that a
    wave has several tiles): finite where the paged call's are, and right."""
    rng = np.random.default_rng(d)
    n, hkv, b = 768, 64, 4
    for first in (0, 384, 768):
        k, v = np.zeros((n, hkv, d), np.float32), 3e36 * (0.5 + 0.5 * rng.random((n, hkv, d)))
        k[:, :, 0] = (5.4 * (np.arange(n) // 32 % 2) - 8 * ((rng.random(n) < 0.85) & (np.arange(n) % 16 > 0)))[:, None]
        k = ref.bf16_value(ref.bf16_bits(k))
        v = ref.bf16_value(ref.bf16_bits(v.astype(np.float32)))
        q = np.zeros((b, hkv, d), np.float32)
        q[:, :, 0] = 1
        y, z = shared_and_paged(rt, q, qk, k, v, "bf16", out, 1.0, first)
        table = np.tile(np.arange(n // 16, dtype=np.int32), (1, 1))
        want, bound = ref.paged_decode(q[:1], lay(k), lay(v), table, [n], 1.0, out_step=STEP[out])
        check(z, *(np.broadcast_to(x, z.shape) for x in (want, bound)))
        check(y, *(np.broadcast_to(x, y.shape) for x in (want, bound + more.p_step("bf16", out) * np.abs(want))))


# ---- the weights behind a bf16 output ------------------------------------------------------

@pytest.mark.parametrize("d", [64, 128, 256])
@pytest.mark.parametrize("hq,hkv", [(8, 8), (16, 2), (64, 2)])
@pytest.mark.parametrize("first", [0, 96, 320])
def test_shared_weights_keep_16_bits(rt, d, hq, hkv, first):
    """Behind a bf16 output too the weights over bf16 rows are held to 2^-16, as the paged call holds them: rows that few
    keys decide are off by the output's rounding alone."""
    rng = np.random.default_rng(d + first)
    n, b = 320 + 40, 6
    q, k, v = floats(rng, (b, hq, d), "bf16", std=4), floats(rng, (n, hkv, d), "bf16"), floats(rng, (n, hkv, d), "bf16")
    y, _ = shared_and_paged(rt, q, "bf16", k, v, "bf16", "bf16", None, first)
    table = np.tile(np.arange(-(-n // 16), dtype=np.int32), (b, 1))
    check(y, *ref.paged_decode(q, lay(k), lay(v), table, [n] * b, p_step=ref.SPLIT + more.MORE, out_step=ref.BF16))


# ---- biases ---------------------------------------------------------------------------------

@pytest.mark.parametrize("vocab", [3001, 20000])
def test_more_biases_than_a_workgroup_keeps(rt, vocab):
    """511 to 2000 entries of a row, words with entries on both sides of the 512th: the last one counts."""
    rng = np.random.default_rng(vocab)
    counts = [511, 512, 513, 600, 1024, 2000]
    offsets = np.concatenate([[0], np.cumsum(counts)]).astype(I32)
    words = rng.integers(0, vocab, offsets[-1]).astype(I32)
    for b, n in enumerate(counts):
        words[offsets[b] + 3] = words[offsets[b] + n - 1] = 17          # first and last
        words[offsets[b] + 510] = words[offsets[b] + min(512, n - 1)] = 18  # around the border
    z = floats(rng, (len(counts), vocab), "f32", std=4.0)
    o = dict(bias_words=words, bias=(5 * rng.standard_normal(offsets[-1])).astype(np.float32), bias_offsets=offsets)
    check(adjust(rt, z, "f32", **o), *more.adjust(z, STEP["f32"], **o))
    o.update(history(rng, len(counts), vocab, 0, 300))
    check(adjust(rt, z, "f32", **o), *more.adjust(z, STEP["f32"], **o))


@pytest.mark.parametrize("kind", ["f32", "bf16"])
@pytest.mark.parametrize("vocab", [8, 4096, 20000])
def test_in_place_by_pieces(rt, kind, vocab):
    """The logits as the output where rows are whole pieces of 16 bytes: the same bits as into another buffer."""
    rng = np.random.default_rng(vocab)
    z = floats(rng, (3, vocab), kind, std=4.0)
    o = {**history(rng, 3, vocab, 0, 900), **biases(rng, 3, vocab, 50), "mask": masks(rng, 3, vocab, 0.9)}
    y = adjust(rt, z, kind, into="logits", **o)
    check(y, *more.adjust(z, STEP[kind], **o))
    np.testing.assert_array_equal(y, adjust(rt, z, kind, **o))
