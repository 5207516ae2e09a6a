"""The serving operators on the GPU against their 64-bit forms: paged append and
decode attention, packed prompts, sampling."""
import numpy as np
import pytest

import serving_ref as ref

pytestmark = pytest.mark.gpu


def rx():
    import rxla_amd
    return rxla_amd


def floats(rng, shape, kind, std=1.0):
    """Values of the type (bf16: rounded), and what is uploaded for them."""
    x = (rng.standard_normal(shape) * std).astype(np.float32)
    return ref.bf16_value(ref.bf16_bits(x)) if kind == "bf16" else x


def up(rt, x, kind):
    r = rx()
    return rt.buffer(ref.bf16_bits(x), r.DType.BF16) if kind == "bf16" else rt.buffer(x, r.DType.F32)


def down(buf):
    r = rx()
    y = buf.to_numpy()
    return ref.bf16_value(y) if buf.dtype == r.DType.BF16 else y


def dt(kind):
    r = rx()
    return r.DType.BF16 if kind == "bf16" else r.DType.F32


def check(y, want, bound):
    y = np.asarray(y, np.float64)
    assert np.array_equal(np.isfinite(y), np.isfinite(want))
    off = np.abs(y - want) - bound
    assert not (off > 0).any(), (float(np.nanmax(off)), np.argwhere(off > 0)[:4].tolist(),
                                 float(np.nanmax(np.abs(y - want))))


def make_pages(rng, lens, hkv, ps, d, kind, spare=2, entries=None):
    need = [-(-max(0, n) // ps) for n in lens]
    entries = max(need + [1]) if entries is None else entries
    order = rng.permutation(sum(need) + spare).astype(np.int32)
    table, at = np.full((len(lens), entries), -1, np.int32), 0
    for b, n in enumerate(need):
        table[b, :n] = order[at:at + n]
        at += n
    kp, vp = (floats(rng, (sum(need) + spare, hkv, ps, d), kind) for _ in range(2))
    return kp, vp, table


def decode(rt, q, qk, kp, vp, pk, table, lens, out="f32", scale=None, into=False):
    r = rx()
    bufs = [up(rt, q, qk), up(rt, kp, pk), up(rt, vp, pk), rt.buffer(table),
            rt.buffer(np.asarray(lens, np.int32))]
    if into:
        o = rt.zeros(q.shape, dt(out))
        assert r.grouped_query_attention_paged(rt, *bufs, scale=scale, out=o) is o
    else:
        o = r.grouped_query_attention_paged(rt, *bufs, scale=scale, out_dtype=dt(out))
    return down(o)


STEP = {"f32": ref.F32, "bf16": ref.BF16}


@pytest.mark.parametrize("d", [64, 128, 256, 40, 96, 512])
@pytest.mark.parametrize("pk,qk,out", [("bf16", "bf16", "bf16"), ("bf16", "f32", "f32"),
                                       ("f32", "f32", "f32"), ("f32", "bf16", "bf16")])
def test_paged_decode(rt, d, pk, qk, out):
    """Every type and head width, lengths 0, 1, around page and tile borders, long ones."""
    rng = np.random.default_rng(d)
    lens = [0, 1, 15, 16, 17, 33, 64, 200, 531]
    q = floats(rng, (len(lens), 4, d), qk)
    kp, vp, table = make_pages(rng, lens, 2, 16, d, pk)
    y = decode(rt, q, qk, kp, vp, pk, table, lens, out)
    want, bound = ref.paged_decode(q, kp, vp, table, lens, out_step=STEP[out])
    check(y, want, bound)
    assert not y[0].any()


@pytest.mark.parametrize("hq,hkv", [(1, 1), (3, 3), (6, 2), (8, 1), (16, 1), (40, 2), (48, 16)])
@pytest.mark.parametrize("pk", ["bf16", "f32"])
def test_paged_decode_heads(rt, hq, hkv, pk):
    rng = np.random.default_rng(hq)
    lens = [70, 3, 150]
    q = floats(rng, (3, hq, 128), "f32")
    kp, vp, table = make_pages(rng, lens, hkv, 32, 128, pk)
    y = decode(rt, q, "f32", kp, vp, pk, table, lens, into=True)
    check(y, *ref.paged_decode(q, kp, vp, table, lens))


@pytest.mark.parametrize("ps", [1, 5, 16, 24, 48, 100, 256])
@pytest.mark.parametrize("d,pk", [(128, "bf16"), (64, "bf16"), (256, "f32")])
def test_paged_decode_page_sizes(rt, ps, d, pk):
    """Pages that end inside a tile, pages longer than a sequence, a scale of its own."""
    rng = np.random.default_rng(ps)
    lens = [1, 47, 130, 300]
    q = floats(rng, (4, 4, d), "f32")
    kp, vp, table = make_pages(rng, lens, 2, ps, d, pk)
    y = decode(rt, q, "f32", kp, vp, pk, table, lens, scale=0.2)
    check(y, *ref.paged_decode(q, kp, vp, table, lens, scale=0.2))


@pytest.mark.parametrize("d,pk,ps", [(128, "bf16", 16), (256, "f32", 48), (64, "f32", 16),
                                     (96, "bf16", 16), (128, "bf16", 7)])
def test_paged_decode_what_is_not_seen(rt, d, pk, ps):
    """Entries outside the pool, lengths past the table and below 0; NaN and infinities in
    every position that is not seen, and an infinite value in the last one that is."""
    rng = np.random.default_rng(1)
    lens = [100, 37, 10 ** 9, -5, 64, 2]
    q = floats(rng, (6, 8, d), "f32")
    kp, vp, table = make_pages(rng, [100, 37, 90, 0, 64, 2], 2, ps, d, pk, entries=-(-100 // ps))
    bad = (-1, -7, kp.shape[0], 2 ** 31 - 1, -2 ** 31)
    table[table < 0] = np.resize(np.array(bad, np.int64), (table < 0).sum()).astype(np.int32)
    table[4, :] = -1                    # a length without a page
    table[0, 1] = kp.shape[0] + 5       # a hole in the middle
    seen = np.zeros(kp.shape[:1] + (ps,), bool)
    for b, n in enumerate(lens):
        for j in range(min(max(n, 0), table.shape[1] * ps)):
            if 0 <= table[b, j // ps] < kp.shape[0]:
                seen[table[b, j // ps], j % ps] = True
    for x, fill in ((kp, np.nan), (vp, np.inf)):
        x[np.broadcast_to(~seen[:, None, :, None], x.shape)] = fill
    y = decode(rt, q, "f32", kp, vp, pk, table, lens)
    check(y, *ref.paged_decode(q, kp, vp, table, lens))
    assert not y[3].any() and not y[4].any()
    vp[table[5, 1 // ps], :, 1 % ps, 3] = np.inf
    y = decode(rt, q, "f32", kp, vp, pk, table, lens)
    assert np.isposinf(y[5, :, 3]).all() and np.isfinite(np.delete(y[5], 3, axis=1)).all()


@pytest.mark.parametrize("d,pk", [(128, "bf16"), (256, "f32"), (80, "bf16")])
def test_paged_decode_large_scores(rt, d, pk):
    """Scores that grow along the sequence (the running maximum moves at every tile) and ones
    too far apart for all but the largest to count."""
    rng = np.random.default_rng(2)
    lens = [400, 400]
    q = floats(rng, (2, 4, d), "f32")
    kp, vp, table = make_pages(rng, lens, 1, 16, d, pk)
    for j in range(400):
        kp[table[0, j // 16], :, j % 16] *= np.float32(1 + j / 64)
        kp[table[1, j // 16], :, j % 16] *= np.float32(40 if j == 123 else 1)
    if pk == "bf16":
        kp = ref.bf16_value(ref.bf16_bits(kp))
    y = decode(rt, q, "f32", kp, vp, pk, table, lens)
    check(y, *ref.paged_decode(q, kp, vp, table, lens))


@pytest.mark.parametrize("pk,qk,d,hq,hkv", [("bf16", "bf16", 128, 8, 2), ("f32", "f32", 64, 4, 4),
                                            ("bf16", "f32", 72, 4, 2)])
def test_paged_decode_long_and_ragged(rt, pk, qk, d, hq, hkv):
    """One long sequence over many workgroups beside short and empty ones; twice the same bits."""
    rng = np.random.default_rng(3)
    lens = [5000, 0, 1, 700, 0, 64, 2049, 16]
    q = floats(rng, (len(lens), hq, d), qk)
    kp, vp, table = make_pages(rng, lens, hkv, 32, d, pk)
    y = decode(rt, q, qk, kp, vp, pk, table, lens)
    check(y, *ref.paged_decode(q, kp, vp, table, lens))
    assert np.array_equal(y, decode(rt, q, qk, kp, vp, pk, table, lens))


@pytest.mark.parametrize("pk,d,hq,hkv", [("bf16", 128, 16, 1), ("bf16", 256, 16, 1), ("f32", 64, 3, 1),
                                         ("bf16", 64, 34, 2)])
def test_paged_decode_pieces(rt, pk, d, hq, hkv):
    """So many keys that waves take several tiles each, some of them the end of one sequence and
    the beginning of another; up to 17 query heads to a kv head."""
    rng = np.random.default_rng(d)
    lens = rng.integers(1500, 2600, 64)
    lens[10:20] = rng.integers(0, 40, 10)
    q = floats(rng, (64, hq, d), "f32")
    kp, vp, table = make_pages(rng, lens, hkv, 16, d, pk)
    y = decode(rt, q, "f32", kp, vp, pk, table, lens)
    check(y, *ref.paged_decode(q, kp, vp, table, lens))


@pytest.mark.parametrize("batch", [63, 64, 65, 130, 700])
def test_paged_decode_many_sequences(rt, batch):
    rng = np.random.default_rng(batch)
    lens = rng.integers(0, 60, batch)
    lens[rng.integers(0, batch, batch // 4)] = 0
    q = floats(rng, (batch, 2, 64), "f32")
    kp, vp, table = make_pages(rng, lens, 1, 16, 64, "bf16")
    y = decode(rt, q, "f32", kp, vp, "bf16", table, lens)
    check(y, *ref.paged_decode(q, kp, vp, table, lens))


def test_paged_decode_pool_past_32_bits(rt):
    """Pages whose byte offsets (and element offsets) pass 2^32: the last pages of a 9 GB pool."""
    torch = pytest.importorskip("torch")
    r, rng = rx(), np.random.default_rng(4)
    pages, hkv, ps, d = 9 * 2 ** 30 // (8 * 64 * 128 * 2), 8, 64, 128
    kp = torch.zeros(pages, hkv, ps, d, dtype=torch.bfloat16, device="cuda")
    vp = torch.zeros_like(kp)
    table = np.array([[pages - 1, 0, pages - 2]], np.int32)
    k, v = (floats(rng, (150, hkv, d), "bf16") for _ in range(2))
    q = floats(rng, (1, 8, d), "f32")
    torch.cuda.synchronize()
    kb, vb, tb = rt.wrap_tensor(kp), rt.wrap_tensor(vp), rt.buffer(table)
    r.paged_kv_append(rt, kb, vb, up(rt, k, "bf16"), up(rt, v, "bf16"), tb,
                      rt.buffer(np.zeros(1, np.int32)), rt.buffer(np.array([0, 150], np.int32)))
    y = down(r.grouped_query_attention_paged(rt, up(rt, q, "f32"), kb, vb, tb,
                                             rt.buffer(np.array([150], np.int32))))
    small = [np.zeros((3, hkv, ps, d), np.float32) for _ in range(2)]
    for pool, new in zip(small, (k, v)):
        for j in range(150):
            pool[j // ps, :, j % ps] = new[j]
    check(y, *ref.paged_decode(q, *small, np.array([[0, 1, 2]]), [150]))


# ---- append ---------------------------------------------------------------------

@pytest.mark.parametrize("pk,nk", [("bf16", "bf16"), ("bf16", "f32"), ("f32", "f32"), ("f32", "bf16")])
@pytest.mark.parametrize("hkv,d,ps", [(2, 64, 16), (1, 128, 7), (3, 36, 48), (2, 9, 1)])
def test_paged_append(rt, pk, nk, hkv, d, ps):
    """Ragged rows at ragged starts; rows before the first and behind the last sequence, positions
    below 0, behind the table and without a page are left out; everything else stays."""
    r, rng = rx(), np.random.default_rng(d)
    counts, starts = [5, 0, 33, 1, 20, 4], [0, 9, 14, 3, -3, 10 ** 6]
    offsets = np.concatenate([[2], 2 + np.cumsum(counts)]).astype(np.int32)
    t = int(offsets[-1]) + 6
    kp, vp, table = make_pages(rng, [60] * 6, hkv, ps, d, pk)
    table[2, min(20 // ps, table.shape[1] - 1)] = kp.shape[0]
    table[3, 0] = -2
    k, v = (floats(rng, (t, hkv, d), nk) for _ in range(2))
    kb, vb = up(rt, kp, pk), up(rt, vp, pk)
    r.paged_kv_append(rt, kb, vb, up(rt, k, nk), up(rt, v, nk), rt.buffer(table),
                      rt.buffer(np.array(starts, np.int32)), rt.buffer(offsets))
    for buf, pool, new in ((kb, kp, k), (vb, vp, v)):
        if pk == "bf16":
            new = ref.bf16_value(ref.bf16_bits(new))
        assert np.array_equal(down(buf), ref.append(pool, new, table, starts, offsets))


@pytest.mark.parametrize("batch", [1, 64, 65, 300, 5000])
def test_paged_append_of_many_sequences(rt, batch):
    """The sequence of a row among many, empty ones included; and the one-row form."""
    r, rng = rx(), np.random.default_rng(batch)
    counts = rng.integers(0, 3, batch)
    offsets = np.concatenate([[0], np.cumsum(counts)]).astype(np.int32)
    starts = rng.integers(0, 14, batch).astype(np.int32)
    kp, vp, table = make_pages(rng, [16] * batch, 1, 16, 8, "f32")
    for off, t in ((offsets, int(offsets[-1])), (None, batch)):
        k, v = (floats(rng, (t, 1, 8), "f32") for _ in range(2))
        kb, vb = up(rt, kp, "f32"), up(rt, vp, "f32")
        r.paged_kv_append(rt, kb, vb, up(rt, k, "f32"), up(rt, v, "f32"), rt.buffer(table),
                          rt.buffer(starts), None if off is None else rt.buffer(off))
        rows = np.arange(batch + 1) if off is None else off
        assert np.array_equal(down(kb), ref.append(kp, k, table, starts, rows))
        assert np.array_equal(down(vb), ref.append(vp, v, table, starts, rows))


# ---- packed prompts ---------------------------------------------------------------

def packed(rt, q, qk, k, v, offsets, out="f32", scale=None, into=None, copies=1):
    """copies: of all heads beside each other, which have to come out alike (with many of them there are
    workgroups enough without sharing a row's keys among waves)."""
    if copies > 1:
        wide = [np.tile(x, (1, copies, 1)) for x in (q, k, v)] + [None if into is None else np.tile(into, (1, copies, 1))]
        y = packed(rt, wide[0], qk, wide[1], wide[2], offsets, out, scale, wide[3])
        y = y.reshape(q.shape[0], copies, q.shape[1], q.shape[2])
        assert all(np.array_equal(y[:, 0], y[:, i], equal_nan=True) for i in range(copies))
        return y[:, 0]
    r = rx()
    bufs = [up(rt, q, qk), up(rt, k, "bf16"), up(rt, v, "bf16"),
            rt.buffer(np.asarray(offsets, np.int32))]
    if into is None:
        return down(r.grouped_query_attention_packed(rt, *bufs, scale=scale, out_dtype=dt(out)))
    o = up(rt, into, out)
    assert r.grouped_query_attention_packed(rt, *bufs, scale=scale, out=o) is o
    return down(o)


def prompts(rng, counts, hq, hkv, d, qk, first=0, tail=0):
    offsets = np.concatenate([[first], first + np.cumsum(counts)]).astype(int)
    t = int(offsets[-1]) + tail
    return (floats(rng, (t, hq, d), qk), floats(rng, (t, hkv, d), "bf16"),
            floats(rng, (t, hkv, d), "bf16"), offsets)


# a BF16 output takes its weights rounded to bf16, an F32 one split in two
P_STEP = {"f32": ref.SPLIT, "bf16": ref.BF16}


@pytest.mark.parametrize("d", [64, 128, 256, 40, 96, 512])
@pytest.mark.parametrize("qk,out", [("bf16", "bf16"), ("f32", "f32"), ("f32", "bf16"), ("bf16", "f32")])
def test_packed_prefill(rt, d, qk, out):
    """Lengths 0, 1 and around the tiles' borders; rows outside every sequence are 0."""
    rng = np.random.default_rng(d)
    q, k, v, offsets = prompts(rng, [1, 0, 16, 17, 63, 64, 65, 0, 130], 4, 2, d, qk, first=3, tail=5)
    y = packed(rt, q, qk, k, v, offsets, out)
    want, bound = ref.packed_prefill(q, k, v, offsets, p_step=P_STEP[out], out_step=STEP[out])
    outside = np.isnan(want).all(axis=(1, 2))
    assert outside.sum() == 8 and not y[outside].any()
    check(y[~outside], want[~outside], bound[~outside])


@pytest.mark.parametrize("d", [64, 128, 256])
@pytest.mark.parametrize("qk,out", [("bf16", "bf16"), ("f32", "f32"), ("f32", "bf16"), ("bf16", "f32")])
@pytest.mark.parametrize("hq,hkv", [(64, 16), (96, 48), (60, 60), (168, 14)])
def test_packed_prefill_of_many_heads(rt, d, qk, out, hq, hkv):
    """The same where there are workgroups enough without sharing a row's keys among waves."""
    rng = np.random.default_rng(d + hq)
    q, k, v, offsets = prompts(rng, [1, 0, 16, 17, 33, 64, 65, 0, 130, 200], hq, hkv, d, qk, first=3, tail=5)
    y = packed(rt, q, qk, k, v, offsets, out)
    g = hq // hkv
    for h in (0, hkv // 2, hkv - 1):
        mine = slice(h * g, (h + 1) * g)
        want, bound = ref.packed_prefill(q[:, mine], k[:, h:h + 1], v[:, h:h + 1], offsets, p_step=P_STEP[out],
                                         out_step=STEP[out])
        outside = np.isnan(want).all(axis=(1, 2))
        assert outside.sum() == 8 and not y[outside].any()
        check(y[~outside][:, mine], want[~outside], bound[~outside])


@pytest.mark.parametrize("hq,hkv", [(1, 1), (3, 3), (6, 2), (8, 1), (16, 1), (20, 2), (12, 4)])
def test_packed_prefill_heads(rt, hq, hkv):
    rng = np.random.default_rng(hq)
    q, k, v, offsets = prompts(rng, [40, 100, 7], hq, hkv, 128, "bf16")
    y = packed(rt, q, "bf16", k, v, offsets, "bf16", scale=0.11)
    check(y, *ref.packed_prefill(q, k, v, offsets, scale=0.11, p_step=ref.BF16, out_step=ref.BF16))


@pytest.mark.parametrize("copies", [1, 90])
@pytest.mark.parametrize("d,qk,out", [(128, "bf16", "bf16"), (128, "f32", "f32"), (64, "bf16", "bf16"),
                                      (256, "f32", "f32"), (72, "f32", "f32")])
def test_packed_prefill_into_leaves_other_rows(rt, d, qk, out, copies):
    """_into writes its sequences' rows and no other; NaN in rows of other sequences stay there."""
    rng = np.random.default_rng(9)
    q, k, v, offsets = prompts(rng, [33, 90], 4, 2, d, qk, first=4, tail=70)
    q[:4], k[:4], v[:4] = np.nan, np.nan, np.nan
    q[offsets[-1]:], k[offsets[-1]:], v[offsets[-1]:] = np.nan, np.inf, np.nan
    k[4:37], v[4:37] = np.nan, np.inf  # the first sequence must not reach the second
    old = floats(rng, q.shape, out)
    y = packed(rt, q, qk, k, v, offsets, out, into=old, copies=copies)
    assert np.array_equal(y[:4], old[:4]) and np.array_equal(y[offsets[-1]:], old[offsets[-1]:])
    want, bound = ref.packed_prefill(q, k, v, [37, 127], p_step=P_STEP[out], out_step=STEP[out])
    check(y[37:127], want[37:127], bound[37:127])
    # a value that is infinite in a sequence's last row reaches that row alone
    v[offsets[-1] - 1, :, 5] = np.inf
    y = packed(rt, q, qk, k, v, offsets, out, copies=copies)
    assert np.isfinite(y[37:126]).all() and np.isposinf(y[126, :, 5]).all()
    assert np.isfinite(np.delete(y[126], 5, axis=1)).all()


@pytest.mark.parametrize("copies", [1, 40])
@pytest.mark.parametrize("hq,hkv,d,qk,out,counts", [
    (8, 2, 128, "bf16", "bf16", [1500, 3, 777, 128]), (2, 2, 128, "f32", "f32", [1000, 129]),
    (8, 1, 64, "bf16", "bf16", [1025]), (4, 1, 256, "f32", "f32", [700, 1])])
def test_packed_prefill_long(rt, hq, hkv, d, qk, out, counts, copies):
    rng = np.random.default_rng(len(counts))
    q, k, v, offsets = prompts(rng, counts, hq, hkv, d, qk)
    y = packed(rt, q, qk, k, v, offsets, out, copies=copies)
    rows = set(rng.integers(0, offsets[-1], 60).tolist()) | {0, int(offsets[-1]) - 1, counts[0] - 1}
    want, bound = ref.packed_prefill(q, k, v, offsets, p_step=P_STEP[out], out_step=STEP[out], rows=rows)
    at = sorted(rows)
    check(y[at], want[at], bound[at])
    assert np.isfinite(y).all()
    assert np.array_equal(y, packed(rt, q, qk, k, v, offsets, out, copies=copies))


@pytest.mark.parametrize("batch", [63, 64, 65, 500])
def test_packed_prefill_many_sequences(rt, batch):
    rng = np.random.default_rng(batch)
    counts = rng.integers(0, 6, batch)
    counts[batch // 2] = 80
    q, k, v, offsets = prompts(rng, counts, 2, 1, 64, "bf16", tail=3)
    y = packed(rt, q, "bf16", k, v, offsets, "bf16")
    want, bound = ref.packed_prefill(q, k, v, offsets, p_step=ref.BF16, out_step=ref.BF16)
    check(y[:offsets[-1]], want[:offsets[-1]], bound[:offsets[-1]])
    assert not y[offsets[-1]:].any()


def test_packed_prefill_offsets_out_of_range(rt):
    """Offsets below 0 and past T are clamped; no sequence at all is no work."""
    rng = np.random.default_rng(5)
    q, k, v, _ = prompts(rng, [50], 2, 1, 128, "f32")
    y = packed(rt, q, "f32", k, v, [-7, 20, 2 ** 31 - 1])
    check(y, *ref.packed_prefill(q, k, v, [0, 20, 50]))
    assert not packed(rt, q, "f32", k, v, [0]).any()
    assert not packed(rt, q, "f32", k, v, [0, 0]).any()
    assert packed(rt, q[:0], "f32", k[:0], v[:0], [0, 0]).size == 0


@pytest.mark.parametrize("copies", [1, 60])
@pytest.mark.parametrize("d,qk,out", [(64, "bf16", "bf16"), (128, "bf16", "bf16"), (256, "bf16", "bf16"), (64, "f32", "f32"),
                                      (128, "f32", "f32"), (256, "f32", "f32"), (128, "f32", "bf16"), (256, "bf16", "f32")])
@pytest.mark.parametrize("hq,hkv", [(2, 2), (4, 2), (4, 1)])
def test_packed_prefill_infinite_values(rt, d, qk, out, hq, hkv, copies):
    """Infinite values of a key: in the rows that see it, and in no row of the same workgroup, wave or
    step that does not."""
    rng = np.random.default_rng(d)
    q, k, v, offsets = prompts(rng, [300, 40], hq, hkv, d, qk)
    v[133, :, 7], v[250, 0, 9] = np.inf, -np.inf
    y = packed(rt, q, qk, k, v, offsets, out, copies=copies)
    rows = {0, 31, 32, 100, 127, 128, 130, 132, 133, 140, 249, 250, 299, 300, 339}
    want, bound = ref.packed_prefill(q, k, v, offsets, p_step=P_STEP[out], out_step=STEP[out], rows=rows)
    at = sorted(rows)
    far = np.isinf(want[at])
    assert np.array_equal(y[at][far], want[at][far])
    check(np.where(far, 0, y[at]), np.where(far, 0, want[at]), np.where(far, 0, bound[at]))
    seen = np.zeros(y.shape, bool)
    seen[133:300, :, 7], seen[250:300, :hq // hkv, 9] = True, True
    assert np.isinf(y[seen]).all() and np.isfinite(y[~seen]).all()


@pytest.mark.parametrize("copies", [1, 60])
@pytest.mark.parametrize("d,qk,out", [(128, "bf16", "bf16"), (128, "f32", "f32"), (64, "f32", "f32"),
                                      (256, "f32", "f32")])
def test_packed_prefill_large_scores(rt, d, qk, out, copies):
    rng = np.random.default_rng(6)
    q, k, v, offsets = prompts(rng, [300, 200], 2, 1, d, qk)
    k[:300] *= (1 + np.arange(300, dtype=np.float32) / 40)[:, None, None]
    k[400] *= 30
    k = ref.bf16_value(ref.bf16_bits(k))
    y = packed(rt, q, qk, k, v, offsets, out, copies=copies)
    check(y, *ref.packed_prefill(q, k, v, offsets, p_step=P_STEP[out], out_step=STEP[out]))


# ---- sampling ---------------------------------------------------------------------

def sample(rt, z, u, kind="f32", t=None, k=None, p=None, m=None, into=False):
    r = rx()
    f = lambda x, d=np.float32: None if x is None else rt.buffer(np.asarray(x, d))  # noqa: E731
    args = (rt, up(rt, z, kind), f(u), f(t), f(k, np.int32), f(p), f(m))
    if into:
        o = rt.zeros((z.shape[0],), r.DType.I32)
        assert r.sample(*args, out=o) is o
        return o.to_numpy()
    return r.sample(*args).to_numpy()


def pick(x, i):
    return None if x is None else np.asarray(x, np.float32 if np.asarray(x).dtype.kind == "f" else np.int32)[i]


def check_sample(rt, z, u, kind="f32", **f):
    got = sample(rt, z, u, kind, **f)
    want = [ref.sample(z[i], np.float32(u[i]), *(pick(f.get(n), i) for n in "tkpm")) for i in range(len(u))]
    assert got.tolist() == want


@pytest.mark.parametrize("v", [1, 2, 63, 1000, 4097, 50000, 248320])
@pytest.mark.parametrize("kind", ["f32", "bf16"])
def test_sample(rt, v, kind):
    """Settings alone and together, over vocabularies from one word on; bf16 logits tie often."""
    rng = np.random.default_rng(v)
    b = 12
    z = floats(rng, (b, v), kind, std=3.0)
    u = rng.random(b).astype(np.float32)
    t = rng.uniform(0.3, 1.5, b).astype(np.float32)
    k = rng.integers(1, min(v, 60) + 1, b)
    p, m = rng.uniform(0.05, 0.99, b).astype(np.float32), rng.uniform(0.005, 0.3, b).astype(np.float32)
    for f in ({}, dict(t=t), dict(k=k), dict(p=p), dict(m=m), dict(t=t, k=k, p=p, m=m), dict(t=t, p=p, m=m)):
        check_sample(rt, z, u, kind, **f)


@pytest.mark.parametrize("v", [5, 1030, 151936])
def test_sample_settings_that_are_off(rt, v):
    """Values that switch a filter off or leave one word, random numbers at and past their ends."""
    rng = np.random.default_rng(v)
    vals = dict(t=[1, 0, -1, np.nan, 1e-6, 1e-40, 1e30, np.inf, 1, 1, 1, 1, 1, 1, 1, 1],
                k=[0, 0, 0, 0, 0, 0, 0, 0, 1, -4, v, v + 9, 2 ** 31 - 1, 3, 3, 0],
                p=[1, 1, 1, 1, 1, 1, 1, 1, 1, 0, -1, 2, np.nan, 1e-9, 0.9, 1],
                m=[0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, np.nan, -1, 0, 5, 1])
    u = np.array([0, .5, .5, .5, .999, .5, .5, .25, .99, .99, .99, 1, 7, -1, np.nan, .9], np.float32)
    z = floats(rng, (16, v), "f32", std=2.0)
    check_sample(rt, z, u, **vals)


@pytest.mark.parametrize("v", [7, 2050, 100003])
def test_sample_ties_and_special_values(rt, v):
    """Rows of equal logits, of two values, of zeros of both signs, with words at -inf, all at -inf,
    with infinities and with NaNs."""
    rng = np.random.default_rng(v)
    rows = [np.zeros(v), np.where(rng.random(v) < .5, 1.0, 1.5), np.where(rng.random(v) < .5, 0.0, -0.0),
            np.where(rng.random(v) < .7, -np.inf, rng.standard_normal(v)), np.full(v, -np.inf),
            np.where(rng.random(v) < .3, np.inf, 1.0), np.where(rng.random(v) < .3, np.nan, 1.0),
            np.full(v, 3e38), np.linspace(-3e38, 3e38, v), np.full(v, 1e-42)]
    rows[3][v // 2] = 0.5
    rows[5][v // 3] = rows[6][v // 3] = np.inf
    rows[6][v // 2] = np.nan
    z = np.array(rows, np.float32)
    n = len(rows)
    for u in (0.0, 0.3, 0.5, 0.97):
        us = np.full(n, u, np.float32)
        check_sample(rt, z, us)
        check_sample(rt, z, us, k=[min(v, 5)] * n, p=[0.6] * n)
        check_sample(rt, z, us, p=[0.5] * n, m=[0.5] * n, t=[0.7] * n)


@pytest.mark.parametrize("v,b", [(1 << 20, 3), (1 << 20, 130), (200000, 100), (40000, 3)])
def test_sample_crowded_borders(rt, v, b):
    """Borders and tokens among words of nearly the same weight, thousands of them at a time, and
    far down the row; rows that one, two and more workgroups share."""
    rng = np.random.default_rng(v + b)
    crowd = (0.01 * rng.standard_normal(v)).astype(np.float32)
    crowd[v // 5] = 12
    even = rng.standard_normal(v).astype(np.float32)
    kinds = [crowd, even, ref.bf16_value(ref.bf16_bits(even)), (3 * even).astype(np.float32)]
    z = np.stack([kinds[i % 4] for i in range(min(b, 12))])
    sets = [dict(k=[0]), dict(k=[0], p=[.99]), dict(k=[1000]), dict(k=[9000]), dict(k=[v - 1]), dict(k=[200], p=[.95]),
            dict(m=[.2]), dict(m=[.02], p=[.999]), dict(k=[5000], p=[.9], m=[.05])]
    u = rng.random(b).astype(np.float32)
    for f in sets:
        n = min(b, 12)
        want = [ref.sample(z[i], u[i], *(pick(f.get(x), 0) for x in "tkpm")) for i in range(n)]
        rows = np.arange(b) % n
        got = sample(rt, z[rows], u[rows], **{x: np.repeat(np.asarray(y), b) for x, y in f.items()})
        assert got.tolist() == [want[i] for i in rows], f


@pytest.mark.parametrize("b", [1, 3, 64, 300])
def test_sample_batches(rt, b):
    """Rows of a batch are independent; the same inputs give the same tokens, into a buffer too."""
    rng = np.random.default_rng(b)
    z = floats(rng, (b, 3001), "bf16", std=2.0)
    u = rng.random(b).astype(np.float32)
    f = dict(t=rng.choice([0.0, 0.7, 1.0], b).astype(np.float32), k=rng.choice([0, 1, 40], b),
             p=rng.choice([1.0, 0.9], b).astype(np.float32))
    check_sample(rt, z, u, **f)
    assert sample(rt, z, u, **f).tolist() == sample(rt, z, u, into=True, **f).tolist()


def test_sample_frequencies(rt):
    """Many random numbers over one row of words give each word's probability: counts of an even
    grid of numbers differ from V p by less than one at each end of a word's interval."""
    v, n = 50, 4096
    z = floats(np.random.default_rng(8), (1, v), "f32")
    u = ((np.arange(n) + 0.5) / n).astype(np.float32)
    got = sample(rt, np.repeat(z, n, axis=0), u)
    p = np.exp(z[0].astype(np.float64))
    p /= p.sum()
    assert (np.abs(np.bincount(got, minlength=v) - n * p) < 2).all()


def test_sample_of_zero_temperature_is_argmax(rt):
    r, rng = rx(), np.random.default_rng(7)
    z = floats(rng, (9, 5000), "bf16")
    z[4, 77] = np.nan
    got = sample(rt, z, np.full(9, 0.9, np.float32), t=np.zeros(9, np.float32))
    assert got.tolist() == r.argmax(rt, rt.buffer(z), 1).to_numpy().tolist()
