"""The paged cache in 8 bits on the GPU: the append's codes and scales, reading pages
back, decode attention over them."""
import numpy as np
import pytest

import serving_more_ref as more
import serving_ref as ref
from test_gpu_serving import check, down, dt, floats, make_pages, rx, up

pytestmark = pytest.mark.gpu


def i32(rt, x):
    return rt.buffer(np.asarray(x, np.int32))


def make_codes(rng, lens, hkv, ps, d, spare=2, entries=None):
    """Pages of codes and scales, the table, and the values that they stand for."""
    kp, vp, table = make_pages(rng, lens, hkv, ps, d, "f32", spare, entries)
    kp[...] *= np.exp(rng.normal(size=kp.shape[:3]))[..., None]  # rows of very different sizes
    vp[...] *= np.exp(rng.normal(size=vp.shape[:3]))[..., None]
    (kc, ks), (vc, vs) = more.encode(kp), more.encode(vp)
    return kc, vc, ks, vs, table


def decode8(rt, q, qk, kc, vc, ks, vs, table, lens, out="f32", scale=None, into=False):
    r = rx()
    bufs = [up(rt, q, qk)] + [rt.buffer(x) for x in (kc, vc, ks, vs, table)] + [i32(rt, lens)]
    if into:
        o = rt.zeros(q.shape, dt(out))
        assert r.grouped_query_attention_paged_q8(rt, *bufs, scale=scale, out=o) is o
    else:
        o = r.grouped_query_attention_paged_q8(rt, *bufs, scale=scale, out_dtype=dt(out))
    return down(o)


def want8(q, kc, vc, ks, vs, table, lens, scale=None, out="f32"):
    return more.decode8(q, kc, vc, ks, vs, table, lens, scale, out)


# ---- the append ------------------------------------------------------------------------

@pytest.mark.parametrize("d", [64, 128, 256, 512, 40, 96, 104, 1, 1000])
@pytest.mark.parametrize("kind", ["f32", "bf16"])
def test_append_codes(rt, d, kind):
    """Codes and scales to the bit, and nothing else in the pages: rows that start inside a page,
    rows behind the table, at negative positions and without a page are left out, so are rows
    outside every sequence."""
    r, rng = rx(), np.random.default_rng(d)
    hkv, ps, counts, starts = 3, 16, [20, 0, 1, 33, 5], [7, 3, 15, 20, -2]
    kc, vc, ks, vs, table = make_codes(rng, [27, 3, 16, 48, 16], hkv, ps, d)
    table[3, 2] = [-1, kc.shape[0]][d % 2]
    offsets = np.cumsum([2] + counts)
    t = offsets[-1] + 3
    k, v = (floats(rng, (t, hkv, d), kind) * np.exp(3 * rng.normal(size=(t, hkv, 1))).astype(np.float32)
            for _ in range(2))
    if kind == "bf16":
        k, v = (ref.bf16_value(ref.bf16_bits(x)) for x in (k, v))
    k[4] = 0                                    # a row of zeros
    v[5, 0, :] = 1e-20                          # below the least scale
    k[6, 1, 0] = np.inf
    v[7, 2, d // 2] = np.nan
    k[8, 0] = np.resize([1, -1, 0.5, 0.25], d) * np.float32(127 / 64)  # quotients halfway between codes
    bufs = [rt.buffer(x) for x in (kc, vc, ks, vs)]
    got = r.paged_kv_append_q8(rt, *bufs, up(rt, k, kind), up(rt, v, kind), rt.buffer(table), i32(rt, starts),
                               i32(rt, offsets))
    assert all(a is b for a, b in zip(got, bufs))
    for x, codes, scales, buf, sbuf in ((k, kc, ks, *bufs[::2]), (v, vc, vs, *bufs[1::2])):
        c, s = more.encode(x)
        np.testing.assert_array_equal(buf.to_numpy(), ref.append(codes, c, table, starts, offsets))
        np.testing.assert_array_equal(sbuf.to_numpy(), ref.append(scales[..., None], s[..., None], table, starts, offsets)[..., 0])


def test_append_is_the_w8_encoders(rt):
    """The codes and scales of quantize_w8 with groups of D, one row for each sequence."""
    r, rng = rx(), np.random.default_rng(0)
    b, hkv, d, ps = 50, 2, 128, 16
    x = floats(rng, (b, hkv, d), "f32", std=3.0)
    kc, vc, ks, vs, table = make_codes(rng, [16] * b, hkv, ps, d)
    bufs = [rt.buffer(a) for a in (kc, vc, ks, vs)]
    starts = rng.integers(0, 16, b).astype(np.int32)
    xb = rt.buffer(x)
    r.paged_kv_append_q8(rt, *bufs, xb, xb, rt.buffer(table), rt.buffer(starts))
    codes, scale = (a.to_numpy() for a in r.quantize_w8(rt, rt.buffer(x.reshape(b * hkv, d)), d))
    for pages, scales in (bufs[::2], bufs[1::2]):
        at = table[np.arange(b), 0]
        np.testing.assert_array_equal(pages.to_numpy()[at, :, starts].reshape(b * hkv, d), codes)
        np.testing.assert_array_equal(scales.to_numpy()[at, :, starts].reshape(b * hkv, 1), scale)


def test_largest_values(rt):
    """Rows near f32's largest value come back finite, within half a step."""
    r = rx()
    x = np.full((1, 1, 64), 3.4e38, np.float32)
    x[0, 0, 1::2] *= np.float32(-0.3)
    pages, scales = [rt.zeros((1, 1, 16, 64), r.DType.U8) for _ in range(2)], [rt.zeros((1, 1, 16), r.DType.F32) for _ in range(2)]
    table, at = i32(rt, [[0]]), i32(rt, [3])
    r.paged_kv_append_q8(rt, *pages, *scales, rt.buffer(x), rt.buffer(-x), table, at)
    back = [rt.zeros((1, 1, 64), r.DType.F32) for _ in range(2)]
    r.paged_kv_read(rt, *pages, table, at, None, *back, *scales)
    s = more.encode(x)[1].astype(np.float64)[0, 0]
    for y, sign in zip(back, (1, -1)):
        y = y.to_numpy().astype(np.float64)
        assert np.isfinite(y).all() and np.abs(y - sign * x.astype(np.float64)).max() <= s * (0.5 + 1e-4)


# ---- reading back -----------------------------------------------------------------------

@pytest.mark.parametrize("d", [64, 128, 256, 40, 100, 520, 3])
@pytest.mark.parametrize("pages", ["q8", "bf16", "f32"])
@pytest.mark.parametrize("back", ["bf16", "f32"])
def test_read(rt, d, pages, back):
    """Every type of pages into every type of rows, to the bit (an 8-bit value rounded to f32, then
    to what the rows hold); 0 where a sequence has no page, rows outside every sequence untouched."""
    r, rng = rx(), np.random.default_rng(d)
    hkv, ps, counts, starts = 2, 16, [30, 0, 1, 40, 6], [3, 0, 31, 30, -3]
    lens = [33, 0, 32, 70, 16]
    if pages == "q8":
        kc, vc, ks, vs, table = make_codes(rng, lens, hkv, ps, d)
        ks[table[0, 1], 1, 3] = np.nan  # a row that stands for NaN
        args, scales = [rt.buffer(kc), rt.buffer(vc)], [rt.buffer(ks), rt.buffer(vs)]
        values = [((c.astype(np.float32) - np.float32(128)) * s[..., None]).astype(np.float32) for c, s in ((kc, ks), (vc, vs))]
    else:
        *values, table = make_pages(rng, lens, hkv, ps, d, pages)
        args, scales = [up(rt, x, pages) for x in values], [None, None]
    table[3, 3] = [-1, 10 ** 6][d % 2]
    offsets = np.cumsum([1] + counts)
    t = int(offsets[-1]) + 2
    outs = [up(rt, np.full((t, hkv, d), 5.0, np.float32), back) for _ in range(2)]
    got = r.paged_kv_read(rt, *args, rt.buffer(table), i32(rt, starts), i32(rt, offsets), *outs,
                          k_scales=scales[0], v_scales=scales[1])
    assert all(a is b for a, b in zip(got, outs))
    for x, y in zip(values, outs):
        want = more.read(x, table, starts, offsets, t)
        outside = np.ones(t, bool)
        outside[offsets[0]:offsets[-1]] = False
        want[outside] = 5.0
        want = want.astype(np.float32)
        if back == "bf16":
            want = np.where(np.isnan(want), np.float32(np.nan), ref.bf16_value(ref.bf16_bits(want)))
        np.testing.assert_array_equal(down(y), want)


def test_read_single_rows(rt):
    """Without offsets: one row of each sequence."""
    r, rng = rx(), np.random.default_rng(2)
    kc, vc, ks, vs, table = make_codes(rng, [20, 1, 33], 2, 16, 128)
    outs = [rt.zeros((3, 2, 128), r.DType.F32) for _ in range(2)]
    r.paged_kv_read(rt, rt.buffer(kc), rt.buffer(vc), rt.buffer(table), i32(rt, [19, 0, 16]), None, *outs,
                    k_scales=rt.buffer(ks), v_scales=rt.buffer(vs))
    for c, s, y in ((kc, ks, outs[0]), (vc, vs, outs[1])):
        want = more.read(more.value(c, s), table, [19, 0, 16], [0, 1, 2, 3], 3).astype(np.float32)
        np.testing.assert_array_equal(y.to_numpy(), want)


# ---- decode attention -------------------------------------------------------------------

@pytest.mark.parametrize("d", [64, 128, 256, 40, 96, 512])
@pytest.mark.parametrize("qk,out", [("bf16", "bf16"), ("f32", "f32"), ("bf16", "f32"), ("f32", "bf16")])
def test_decode8(rt, d, qk, out):
    """Every type and head width, lengths 0, 1, around page and tile borders, long ones."""
    rng = np.random.default_rng(d)
    lens = [0, 1, 15, 16, 17, 33, 64, 200, 531]
    q = floats(rng, (len(lens), 4, d), qk)
    pages = make_codes(rng, lens, 2, 16, d)
    y = decode8(rt, q, qk, *pages, lens, out)
    check(y, *want8(q, *pages, lens, out=out))
    assert not y[0].any()


@pytest.mark.parametrize("hq,hkv", [(1, 1), (3, 3), (6, 2), (8, 1), (16, 1), (40, 2), (48, 16)])
def test_decode8_heads(rt, hq, hkv):
    rng = np.random.default_rng(hq)
    lens = [70, 3, 150]
    q = floats(rng, (3, hq, 128), "f32")
    pages = make_codes(rng, lens, hkv, 32, 128)
    check(decode8(rt, q, "f32", *pages, lens, into=True), *want8(q, *pages, lens))


@pytest.mark.parametrize("ps", [1, 5, 16, 24, 48, 100, 256])
@pytest.mark.parametrize("d", [64, 128, 256])
def test_decode8_page_sizes(rt, ps, d):
    """Pages that end inside a tile, pages longer than a sequence, a scale of its own."""
    rng = np.random.default_rng(ps)
    lens = [1, 47, 130, 300]
    q = floats(rng, (4, 4, d), "f32")
    pages = make_codes(rng, lens, 2, ps, d)
    check(decode8(rt, q, "f32", *pages, lens, scale=0.2), *want8(q, *pages, lens, scale=0.2))


@pytest.mark.parametrize("b,high,hq,hkv,d", [(1, 5000, 16, 8, 128), (70, 900, 8, 2, 64), (130, 40, 4, 4, 128), (3, 3000, 32, 2, 256)])
def test_decode8_runs_of_sequences(rt, b, high, hq, hkv, d):
    """Long sequences dealt to many workgroups, more sequences than a wave has lanes, empty ones among them."""
    rng = np.random.default_rng(b)
    lens = rng.integers(0, high, b)
    lens[b // 2] = high
    lens[::7] = np.where(rng.random(lens[::7].size) < .5, 0, lens[::7]) if b > 1 else lens[::7]
    q = floats(rng, (b, hq, d), "f32")
    pages = make_codes(rng, lens, hkv, 16, d)
    check(decode8(rt, q, "f32", *pages, lens), *want8(q, *pages, lens))


@pytest.mark.parametrize("d,ps", [(128, 16), (256, 48), (64, 16), (96, 16), (128, 7)])
def test_decode8_what_is_not_seen(rt, d, ps):
    """Entries outside the pool, lengths past the table and below 0; NaN and infinite scales in every
    position that is not seen; a row that stands for NaN among those that are."""
    rng = np.random.default_rng(1)
    lens = [100, 37, 10 ** 9, -5, 64, 2]
    q = floats(rng, (6, 8, d), "f32")
    kc, vc, ks, vs, table = make_codes(rng, [100, 37, 90, 0, 64, 2], 2, ps, d, entries=-(-100 // ps))
    bad = (-1, -7, kc.shape[0], 2 ** 31 - 1, -2 ** 31)
    table[table < 0] = np.resize(np.array(bad, np.int64), (table < 0).sum()).astype(np.int32)
    table[4, :] = -1                    # a length without a page
    table[0, 1] = kc.shape[0] + 5       # a hole in the middle
    seen = np.zeros((kc.shape[0], ps), bool)
    for b, n in enumerate(lens):
        for j in range(min(max(n, 0), table.shape[1] * ps)):
            if 0 <= table[b, j // ps] < kc.shape[0]:
                seen[table[b, j // ps], j % ps] = True
    for x, fill in ((ks, np.nan), (vs, np.inf)):
        x[np.broadcast_to(~seen[:, None, :], x.shape)] = fill
    y = decode8(rt, q, "f32", kc, vc, ks, vs, table, lens)
    check(y, *want8(q, kc, vc, ks, vs, table, lens))
    assert not y[3].any() and not y[4].any()
    ks[table[5, 1 // ps], 0, 1 % ps] = np.nan
    y = decode8(rt, q, "f32", kc, vc, ks, vs, table, lens)
    assert np.isnan(y[5, :4]).all() and np.isfinite(y[5, 4:]).all() and np.isfinite(y[:5]).all()


@pytest.mark.parametrize("d", [64, 128, 256, 80])
def test_decode8_scales_far_apart(rt, d):
    """Rows of 1e-12 beside rows of 1e12, scores up to 1e4: the largest weigh alone."""
    rng = np.random.default_rng(d)
    lens = [100, 40]
    q = floats(rng, (2, 4, d), "f32")
    kc, vc, ks, vs, table = make_codes(rng, lens, 2, 16, d)
    vs *= np.float32(10) ** rng.integers(-12, 13, vs.shape).astype(np.float32)
    ks *= np.float32(10) ** rng.integers(-3, 3, ks.shape).astype(np.float32)
    check(decode8(rt, q, "f32", kc, vc, ks, vs, table, lens), *want8(q, kc, vc, ks, vs, table, lens))


@pytest.mark.parametrize("kind", ["bf16", "f32"])
def test_append_codes_at_the_middle(rt, kind):
    """Every quotient near the middle between two codes: values (k + 1/2) s and the ones beside them, for
    scales of every mantissa length (all ones among them) and rows whose largest is an odd multiple."""
    r, rng = rx(), np.random.default_rng(9)
    t, hkv, d = 400, 2, 128
    amax = (1 + rng.random((t, hkv, 1))).astype(np.float32) * np.float32(2) ** rng.integers(-30, 100, (t, hkv, 1)).astype(np.float32)
    amax[:8] = np.nextafter(np.float32(2), np.float32(0)) * np.float32(127) * np.float32(2) ** np.arange(8, dtype=np.float32)[:, None, None]
    if kind == "bf16":
        amax = ref.bf16_value(ref.bf16_bits(amax))
    s = more.encode(amax)[1][..., None]
    half = (rng.integers(-126, 126, (t, hkv, d)) + 0.5) * s.astype(np.float64)
    x = half.astype(np.float32)
    if kind == "bf16":
        x = ref.bf16_value(ref.bf16_bits(x))
    else:
        for _ in range(2):
            x = np.where(rng.random(x.shape) < 0.3, np.nextafter(x, np.float32(np.inf)), x)
            x = np.where(rng.random(x.shape) < 0.3, np.nextafter(x, np.float32(-np.inf)), x)
    x[..., :1] = amax
    x = np.clip(x, -amax, amax)
    pages, scales = [rt.zeros((t, hkv, 16, d), r.DType.U8) for _ in range(2)], [rt.zeros((t, hkv, 16), r.DType.F32) for _ in range(2)]
    r.paged_kv_append_q8(rt, *pages, *scales, up(rt, x, kind), up(rt, -x, kind), i32(rt, np.arange(t)[:, None]), i32(rt, np.zeros(t)))
    for sign, p, q in ((1, *[pages[0], scales[0]]), (-1, *[pages[1], scales[1]])):
        c, want = more.encode(sign * x)
        np.testing.assert_array_equal(q.to_numpy()[:, :, 0], want)
        np.testing.assert_array_equal(p.to_numpy()[:, :, 0], c)
