"""Attention of one new token per sequence behind shared prefixes, on the GPU."""
import numpy as np
import pytest

import serving_more_ref as more
import serving_ref as ref
from test_gpu_serving import check, down, dt, floats, make_pages, rx, up

pytestmark = pytest.mark.gpu


def i32(rt, x):
    return rt.buffer(np.asarray(x, np.int32))


def make(rng, prefix_lens, lens, hkv, ps, d, kind):
    """One pool for prefixes and sequences: (values of K, of V, codes and scales or None,
    prefixes, table)."""
    both = [max(0, n) for n in list(prefix_lens) + list(lens)]
    kp, vp, ids = make_pages(rng, both, hkv, ps, d, "f32" if kind == "q8" else kind)
    n = len(prefix_lens)
    codes = None
    if kind == "q8":
        codes = [*more.encode(kp), *more.encode(vp)]
        kp, vp = more.value(*codes[:2]), more.value(*codes[2:])
    width = [max([1] + [-(-x // ps) for x in part]) for part in (both[:n], both[n:])]
    return kp, vp, codes, ids[:n, :width[0]].copy(), ids[n:, :width[1]].copy()


def call(rt, q, qk, kp, vp, codes, kind, prefixes, prefix_lens, groups, table, lens, out="f32", scale=None, into=False):
    r = rx()
    pages = [rt.buffer(codes[0]), rt.buffer(codes[2])] if codes else [up(rt, kp, kind), up(rt, vp, kind)]
    scales = dict(k_scales=rt.buffer(codes[1]), v_scales=rt.buffer(codes[3])) if codes else {}
    args = [up(rt, q, qk), *pages, i32(rt, prefixes), i32(rt, prefix_lens), i32(rt, groups), i32(rt, table), i32(rt, lens)]
    if into:
        o = rt.zeros(q.shape, dt(out))
        assert r.grouped_query_attention_shared(rt, *args, scale=scale, out=o, **scales) is o
    else:
        o = r.grouped_query_attention_shared(rt, *args, scale=scale, out_dtype=dt(out), **scales)
    return down(o)


def run(rt, rng, prefix_lens, groups, lens, hq, hkv, d, kind, qk="f32", out="f32", ps=16, scale=None, into=False):
    kp, vp, codes, prefixes, table = make(rng, prefix_lens, lens, hkv, ps, d, kind)
    q = floats(rng, (len(lens), hq, d), qk)
    y = call(rt, q, qk, kp, vp, codes, kind, prefixes, prefix_lens, groups, table, lens, out, scale, into)
    check(y, *more.shared(q, kp, vp, prefixes, prefix_lens, groups, table, lens, scale, out, codes and codes[3]))
    return y


@pytest.mark.parametrize("d", [64, 128, 256, 40, 512])
@pytest.mark.parametrize("kind", ["bf16", "q8", "f32"])
@pytest.mark.parametrize("qk,out", [("bf16", "bf16"), ("f32", "f32"), ("bf16", "f32"), ("f32", "bf16")])
def test_shared(rt, d, kind, qk, out):
    """Every type and head width; prefixes and lengths 0, 1, around page and tile borders; a
    sequence in no group, a group without sequences."""
    rng = np.random.default_rng(d)
    lens = [0, 1, 15, 16, 17, 40, 0, 3, 0]
    y = run(rt, rng, [100, 7, 0, 16, 333], [0, 3, 3, 5, 6, 8], lens, 4, 2, d, kind, qk, out)
    assert not y[8].any() and y[0].any() and y[6].any()


@pytest.mark.parametrize("hq,hkv", [(1, 1), (3, 3), (6, 2), (8, 1), (16, 1), (40, 2), (24, 8)])
@pytest.mark.parametrize("kind", ["bf16", "q8", "f32"])
def test_shared_heads(rt, hq, hkv, kind):
    rng = np.random.default_rng(hq)
    lens = rng.integers(0, 40, 9)
    run(rt, rng, [130, 65], [0, 6, 9], lens, hq, hkv, 128, kind, into=True)


@pytest.mark.parametrize("ps", [1, 5, 16, 24, 48, 100, 256])
@pytest.mark.parametrize("kind", ["bf16", "q8", "f32"])
def test_shared_page_sizes(rt, ps, kind):
    rng = np.random.default_rng(ps)
    run(rt, rng, [300, 47], [0, 2, 5], [1, 47, 130, 300, 2], 4, 2, 64, kind, ps=ps, scale=0.2)


@pytest.mark.parametrize("b,n,prefix,high,hq,hkv,d,kind", [
    (1, 1, 3000, 5, 16, 8, 128, "bf16"), (70, 1, 500, 90, 8, 2, 128, "bf16"), (200, 3, 200, 10, 4, 4, 64, "q8"),
    (33, 2, 700, 50, 8, 1, 256, "bf16"), (130, 130, 40, 9, 4, 2, 128, "bf16"), (40, 1, 2000, 3, 32, 2, 128, "q8"),
    (37, 1, 300, 30, 16, 2, 256, "q8"), (20, 1, 400, 30, 16, 2, 128, "f32"), (64, 1, 64, 1, 64, 8, 64, "bf16")])
def test_shared_runs(rt, b, n, prefix, high, hq, hkv, d, kind):
    """Groups of more rows than a tile, long prefixes dealt to many workgroups, many groups."""
    rng = np.random.default_rng(b + n)
    lens = rng.integers(0, high, b)
    prefix_lens = rng.integers(max(1, prefix // 4), prefix + 1, n)
    groups = np.sort(np.concatenate([[0, b], rng.integers(0, b + 1, n - 1)])) if n < 100 else np.arange(n + 1)
    run(rt, rng, prefix_lens, groups, lens, hq, hkv, d, kind, "bf16", "f32")


def test_groups_outside_the_batch(rt):
    """Offsets of groups below 0 and past the batch: what lies in it counts."""
    rng = np.random.default_rng(5)
    run(rt, rng, [50, 60, 70], [-9, 2, 4, 2 ** 31 - 1], [3, 4, 5, 6, 7, 8], 4, 2, 128, "bf16")
    run(rt, rng, [50, 60], [2, 4, 5], [3, 0, 5, 6, 0, 8], 4, 2, 128, "q8")


@pytest.mark.parametrize("d,kind,ps", [(128, "bf16", 16), (64, "f32", 16), (256, "bf16", 48), (128, "q8", 16), (96, "bf16", 16)])
def test_shared_what_is_not_seen(rt, d, kind, ps):
    """Entries outside the pool and lengths past the tables, in prefixes and behind them; NaN in every
    position that is not seen; a prefix without a page."""
    rng = np.random.default_rng(1)
    prefix_lens, lens, groups = [100, 10 ** 9, 64, -3], [37, 2, 10 ** 9, -5, 20, 0], [0, 2, 4, 5, 6]
    kp, vp, codes, prefixes, table = make(rng, [100, 90, 64, 0], [37, 2, 40, 0, 20, 0], 2, ps, d, kind)
    bad = (-1, -7, kp.shape[0], 2 ** 31 - 1, -2 ** 31)
    for t in (prefixes, table):
        t[t < 0] = np.resize(np.array(bad, np.int64), (t < 0).sum()).astype(np.int32)
    prefixes[0, 1], prefixes[2, :] = kp.shape[0] + 5, -1
    seen = np.zeros((kp.shape[0], ps), bool)
    for t, ns in ((prefixes, prefix_lens), (table, lens)):
        for b, n in enumerate(ns):
            for j in range(min(max(n, 0), t.shape[1] * ps)):
                if 0 <= t[b, j // ps] < kp.shape[0]:
                    seen[t[b, j // ps], j % ps] = True
    if codes:
        for s in (codes[1], codes[3]):
            s[np.broadcast_to(~seen[:, None, :], s.shape)] = np.nan
    for x, fill in ((kp, np.nan), (vp, np.inf)):
        x[np.broadcast_to(~seen[:, None, :, None], x.shape)] = fill
    q = floats(rng, (6, 8, d), "f32")
    y = call(rt, q, "f32", kp, vp, codes, kind, prefixes, prefix_lens, groups, table, lens)
    check(y, *more.shared(q, kp, vp, prefixes, prefix_lens, groups, table, lens, vs=codes and codes[3]))
    assert not y[5].any()


@pytest.mark.parametrize("kind", ["bf16", "q8", "f32"])
def test_shared_large_scores(rt, kind):
    """Scores of hundreds whose maximum moves from the prefix to a sequence's own keys and back."""
    rng = np.random.default_rng(3)
    kp, vp, codes, prefixes, table = make(rng, [200], [30, 30, 1], 2, 16, 128, kind)
    q = floats(rng, (3, 8, 128), "f32") * 20
    y = call(rt, q, "f32", kp, vp, codes, kind, prefixes, [200], [0, 3], table, [30, 30, 1])
    check(y, *more.shared(q, kp, vp, prefixes, [200], [0, 3], table, [30, 30, 1], vs=codes and codes[3]))


def test_infinite_values_of_a_prefix(rt):
    """An infinite value and a NaN key that a prefix holds reach its own group alone."""
    rng = np.random.default_rng(4)
    kp, vp, codes, prefixes, table = make(rng, [90, 90], [9] * 6, 2, 16, 128, "bf16")
    vp[prefixes[0, 2], 1, 3, 7] = np.inf
    q = floats(rng, (6, 4, 128), "f32")
    args = (prefixes, [90, 90], [0, 3, 6], table, [9] * 6)
    y = call(rt, q, "f32", kp, vp, codes, "bf16", *args)
    assert np.isposinf(y[:3, 2:, 7]).all() and np.isfinite(np.delete(y[:3], 7, axis=2)).all() and np.isfinite(y[3:]).all()
    kp[prefixes[1, 0], 0, 2, 5] = np.nan
    y = call(rt, q, "f32", kp, vp, codes, "bf16", *args)
    assert np.isnan(y[3:, :2]).all() and np.isfinite(y[3:, 2:]).all() and np.isfinite(y[:3, :2]).all()


def test_shared_is_paged_over_whole_tables(rt):
    """Page tables that begin with the prefix's pages: the paged call's rows, within both bounds."""
    r, rng = rx(), np.random.default_rng(6)
    lens = [5, 60, 33]
    kp, vp, codes, prefixes, table = make(rng, [96], lens, 2, 16, 128, "bf16")
    q = floats(rng, (3, 8, 128), "f32")
    y = call(rt, q, "f32", kp, vp, None, "bf16", prefixes, [96], [0, 3], table, lens)
    whole = np.concatenate([np.repeat(prefixes, 3, axis=0), table], axis=1)
    z = down(r.grouped_query_attention_paged(rt, up(rt, q, "f32"), up(rt, kp, "bf16"), up(rt, vp, "bf16"), i32(rt, whole),
                                             i32(rt, [96 + n for n in lens])))
    _, bound = more.shared(q, kp, vp, prefixes, [96], [0, 3], table, lens)
    assert (np.abs(y - z) <= 2 * bound).all()
