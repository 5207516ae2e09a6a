"""The serving operators as a serving loop uses them: together, captured into graphs, on other
streams, from two threads, over tensors of any alignment and of sizes past 32 bits."""
import threading

import numpy as np
import pytest

import serving_ref as ref
from test_gpu_serving import check, down, dt, floats, make_pages, prompts, rx, up

pytestmark = pytest.mark.gpu


def i32(rt, x):
    return rt.buffer(np.asarray(x, np.int32))


# ---- refusals, through the package ---------------------------------------------------

def test_refusals_raise_and_leave_the_runtime_usable(rt):
    r, rng = rx(), np.random.default_rng(0)
    q, k, v, offsets = prompts(rng, [3, 4], 4, 2, 64, "f32")
    qb, kb, vb, ob = up(rt, q, "f32"), up(rt, k, "bf16"), up(rt, v, "bf16"), i32(rt, offsets)
    kp, vp, table = make_pages(rng, [40, 9], 2, 16, 64, "bf16")
    kpb, vpb, tb, lens = up(rt, kp, "bf16"), up(rt, vp, "bf16"), i32(rt, table), i32(rt, [40, 9])
    q1, z, u = up(rt, q[:2], "f32"), up(rt, q[0], "f32"), rt.buffer(np.zeros(4, np.float32))
    out = rt.zeros((2, 4, 64), r.DType.F32)
    for bad in (lambda: r.grouped_query_attention_packed(rt, qb, kb, up(rt, v[:6], "bf16"), ob),
                lambda: r.grouped_query_attention_packed(rt, qb, kb, vb, ob, scale=float("nan")),
                lambda: r.grouped_query_attention_packed(rt, qb, kb, vb, ob, out=out),
                lambda: r.grouped_query_attention_packed(rt, qb, kb, vb, ob, out=qb),
                lambda: r.grouped_query_attention_paged(rt, q1, kpb, vpb, tb, i32(rt, [1])),
                lambda: r.grouped_query_attention_paged(rt, q1, kpb, up(rt, vp, "f32"), tb, lens),
                lambda: r.grouped_query_attention_paged(rt, q1, kpb, vpb, tb, lens, out_dtype=r.DType.I32),
                lambda: r.grouped_query_attention_paged(rt, q1, kpb, vpb, tb, lens, out=q1),
                lambda: r.paged_kv_append(rt, kpb, kpb, kb, vb, tb, lens, i32(rt, [0, 3, 7])),
                lambda: r.paged_kv_append(rt, kpb, vpb, kb, vb, tb, lens),
                lambda: r.sample(rt, z, rt.buffer(np.zeros(3, np.float32))),
                lambda: r.sample(rt, z, u, top_k=u),
                lambda: r.sample(rt, z, u, out=rt.zeros((4,), r.DType.F32))):
        with pytest.raises(r.Error) as e:
            bad()
        assert e.value.code == r.Status.INVALID_ARGUMENT
    check(down(r.grouped_query_attention_packed(rt, qb, kb, vb, ob, out_dtype=r.DType.F32)),
          *ref.packed_prefill(q, k, v, offsets))


# ---- together ------------------------------------------------------------------------

@pytest.mark.parametrize("hq,hkv,d,kind,ps", [(8, 2, 128, "bf16", 16), (4, 4, 64, "bf16", 64), (6, 1, 256, "f32", 48),
                                              (4, 2, 40, "bf16", 5)])
def test_a_serving_loop(rt, hq, hkv, d, kind, ps):
    """Prompts of different lengths into the pages and through packed attention, then steps that
    append a row, attend over the pages and sample a token whose embedding is the next query:
    every attention within its bound of the 64-bit form over the rows written so far, every token
    that of the 64-bit form of the logits it came from, and the pages' contents the contiguous
    cache's, over which the framework's contiguous decode attention gives the same rows within
    both bounds."""
    r, rng = rx(), np.random.default_rng(d + hq)
    counts, steps, vocab = [37, 1, 100, 16], 6, 500
    b = len(counts)
    q, k, v, offsets = prompts(rng, counts, hq, hkv, d, "f32")
    lens = np.array(counts)
    kp, vp, table = make_pages(rng, lens + steps, hkv, ps, d, kind)
    pools = [up(rt, kp, kind), up(rt, vp, kind)]
    tb = i32(rt, table)
    kb, vb = up(rt, k, "bf16"), up(rt, v, "bf16")
    r.paged_kv_append(rt, *pools, kb, vb, tb, i32(rt, [0] * b), i32(rt, offsets))
    y = down(r.grouped_query_attention_packed(rt, up(rt, q, "f32"), kb, vb, i32(rt, offsets), out_dtype=r.DType.F32))
    check(y, *ref.packed_prefill(q, k, v, offsets))
    keys = [[x[offsets[i]:offsets[i + 1]] for i in range(b)] for x in (k, v)]
    head = floats(rng, (hq * d, vocab), "f32") / np.float32(np.sqrt(d))
    embed = [floats(rng, (vocab, h, d), "f32") for h in (hq, hkv, hkv)]
    x = y[offsets[1:] - 1]
    lmax = int(lens.max()) + steps
    for step in range(steps):
        logits = (x.reshape(b, -1) @ head).astype(np.float32)
        u = rng.random(b).astype(np.float32)
        tokens = r.sample(rt, up(rt, logits, "f32"), rt.buffer(u), rt.buffer(np.full(b, 0.8, np.float32)),
                          i32(rt, [40] * b), rt.buffer(np.full(b, 0.95, np.float32))).to_numpy()
        f32 = np.float32
        assert tokens.tolist() == [ref.sample(logits[i], u[i], f32(.8), 40, f32(.95)) for i in range(b)]
        qs, ks, vs = (e[tokens] for e in embed)
        r.paged_kv_append(rt, *pools, up(rt, ks, "f32"), up(rt, vs, "f32"), tb, i32(rt, lens))
        for pool, new in zip(keys, (ks, vs)):
            for i in range(b):
                row = new[i] if kind == "f32" else ref.bf16_value(ref.bf16_bits(new[i]))
                pool[i] = np.concatenate([pool[i], row[None]])
        lens = lens + 1
        x = down(r.grouped_query_attention_paged(rt, up(rt, qs, "f32"), *pools, tb, i32(rt, lens), out_dtype=r.DType.F32))
        pages = [down(p) for p in pools]
        want, bound = ref.paged_decode(qs, *pages, table, lens)
        check(x, want, bound)
        planes = [np.zeros((b, hkv, lmax, d), np.float32) for _ in range(2)]
        for plane, pool in zip(planes, keys):
            for i in range(b):
                plane[i, :, :lens[i]] = pool[i].transpose(1, 0, 2)
        for i in range(b):
            for h in range(hkv):
                for page, plane in zip(pages, planes):
                    assert np.array_equal(ref.paged_keys(page, table[i], lens[i], h), plane[i, h, :lens[i]])
        z = down(r.grouped_query_attention(rt, up(rt, qs, "f32"), up(rt, planes[0], kind), up(rt, planes[1], kind),
                                           i32(rt, lens)))
        loose = max(float(np.abs(want).max()) * 1e-4, 1e-6)  # (its own tests': 1e-4 of the largest)
        assert np.abs(x - z).max() <= loose + bound.max()


def test_sequences_that_share_pages(rt):
    """One prompt's pages read by several sequences that go on differently."""
    r, rng = rx(), np.random.default_rng(3)
    hkv, ps, d = 2, 16, 128
    kp, vp, _ = make_pages(rng, [16 * 12], hkv, ps, d, "bf16")
    table = np.array([[0, 1, 2, 3, 4], [0, 1, 2, 5, 6], [0, 1, 2, 0, 1], [7, 7, 7, 7, 7]], np.int32)
    lens = [70, 80, 79, 33]
    q = floats(rng, (4, 8, d), "f32")
    y = down(r.grouped_query_attention_paged(rt, up(rt, q, "f32"), up(rt, kp, "bf16"), up(rt, vp, "bf16"), i32(rt, table),
                                             i32(rt, lens), out_dtype=r.DType.F32))
    check(y, *ref.paged_decode(q, kp, vp, table, lens))


# ---- alignment -------------------------------------------------------------------------

@pytest.mark.parametrize("which", ["q", "k", "v", "out"])
@pytest.mark.parametrize("elements", [1, 3])
def test_operands_at_odd_addresses(rt, which, elements):
    """Tensors that begin an element or more past a 16-byte boundary."""
    torch = pytest.importorskip("torch")
    r, rng = rx(), np.random.default_rng(elements)

    def dev(x, name):
        t = torch.from_numpy(np.ascontiguousarray(x))
        t = t.to(torch.bfloat16 if name in "kv" else torch.float32).cuda()
        if name != which:
            return t
        whole = torch.zeros(t.numel() + 16, dtype=t.dtype, device="cuda")
        part = whole[elements:elements + t.numel()].view(t.shape)
        part.copy_(t)
        return part

    q, k, v, offsets = prompts(rng, [70, 5], 4, 2, 64, "f32", first=1, tail=2)
    kp, vp, table = make_pages(rng, [50, 20], 2, 16, 64, "bf16")
    seen = [dev(q, "q"), dev(k, "k"), dev(v, "v"), dev(np.full(q.shape, 5.0, np.float32), "out"), dev(q[:2], "q"), dev(kp, "k"),
            dev(vp, "v"), dev(np.zeros((2, 4, 64), np.float32), "out")]
    logits = dev(floats(rng, (3, 999), "f32"), "q")
    torch.cuda.synchronize()
    b = [rt.wrap_tensor(t) for t in seen]
    r.grouped_query_attention_packed(rt, b[0], b[1], b[2], i32(rt, offsets), out=b[3])
    want, bound = ref.packed_prefill(q, k, v, offsets)
    y, outside = down(b[3]), np.isnan(want).all(axis=(1, 2))
    assert (y[outside] == 5).all() and outside.sum() == 3
    check(y[~outside], want[~outside], bound[~outside])
    r.grouped_query_attention_paged(rt, b[4], b[5], b[6], i32(rt, table), i32(rt, [50, 20]), out=b[7])
    check(down(b[7]), *ref.paged_decode(q[:2], kp, vp, table, [50, 20]))
    r.paged_kv_append(rt, b[5], b[6], b[1], b[2], i32(rt, table), i32(rt, [10, 3]), i32(rt, [0, 30, 40]))
    assert np.array_equal(down(b[5]), ref.append(kp, k, table, [10, 3], [0, 30, 40]))
    assert np.array_equal(down(b[6]), ref.append(vp, v, table, [10, 3], [0, 30, 40]))
    u = rng.random(3).astype(np.float32)
    got = r.sample(rt, rt.wrap_tensor(logits), rt.buffer(u), None, i32(rt, [0, 50, 900])).to_numpy()
    z = logits.cpu().numpy()
    assert got.tolist() == [ref.sample(z[i], u[i], k=n) for i, n in enumerate((0, 50, 900))]


# ---- graphs, streams, threads ------------------------------------------------------------

def cases(own, rng):
    """name: (a call into buffers of its own, its output buffers)."""
    r = rx()
    q, k, v, offsets = prompts(rng, [300, 1, 77], 8, 2, 128, "f32")
    kp, vp, table = make_pages(rng, [900, 40, 333], 2, 16, 128, "bf16")
    pools = [up(own, kp, "bf16"), up(own, vp, "bf16")]
    qb, kb, vb, ob, tb = up(own, q, "f32"), up(own, k, "bf16"), up(own, v, "bf16"), i32(own, offsets), i32(own, table)
    q1, lens = up(own, q[:3], "f32"), i32(own, [900, 40, 333])
    new = [up(own, x[:3], "bf16") for x in (k, v)]
    z, z1 = up(own, floats(rng, (5, 30000), "f32"), "f32"), up(own, floats(rng, (3, 151936), "bf16"), "bf16")
    f = lambda *x: own.buffer(np.array(x, np.float32))  # noqa: E731
    y1, y2 = own.zeros(q.shape, r.DType.BF16), own.zeros((3, 8, 128), r.DType.F32)
    t1, t2 = own.zeros((5,), r.DType.I32), own.zeros((3,), r.DType.I32)
    s1 = (f(.1, .5, .9, .2, .7), f(1, .8, 0, 1.2, 1), i32(own, [0, 50, 9, 1000, 0]), f(1, .9, 1, .95, .5))
    s2 = (f(.3, .6, .99), None, i32(own, [0, 300, 20]), f(.97, .9, 1))
    starts = i32(own, [899, 39, 332])
    return {
        "prefill": (lambda: r.grouped_query_attention_packed(own, qb, kb, vb, ob, out=y1), [y1]),
        "append and decode": (lambda: (r.paged_kv_append(own, *pools, *new, tb, starts),
                                       r.grouped_query_attention_paged(own, q1, *pools, tb, lens, out=y2)), [y2, *pools]),
        "sample": (lambda: r.sample(own, z, *s1, out=t1), [t1]),
        "sample, shared rows": (lambda: r.sample(own, z1, *s2, out=t2), [t2]),
    }


def clear(buffers):
    for b in buffers:
        x = b.to_numpy()
        if x.ndim != 4:
            b.copy_from(np.full(x.shape, 7, x.dtype))


@pytest.mark.parametrize("name", ["prefill", "append and decode", "sample", "sample, shared rows", "all"])
def test_captured_calls_replay(rt, name):
    """A captured call gives the eager call's bits at every replay, with eager calls between the
    replays and beside them."""
    import torch
    own = rx().Runtime(0)
    got = cases(own, np.random.default_rng(1))
    others = cases(own, np.random.default_rng(2))
    names = list(got) if name == "all" else [name]
    call = lambda: [got[n][0]() for n in names]  # noqa: E731
    outs = [b for n in names for b in got[n][1]]
    call()
    eager = [b.to_numpy() for b in outs]
    stream = torch.cuda.Stream()
    own.synchronize()
    own.set_stream(stream.cuda_stream)
    call()
    own.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=stream, capture_error_mode="thread_local"):
        call()
    own.set_stream(None)  # eager calls on a stream of their own from here on
    for c, _ in others.values():
        c()
    want = {n: [b.to_numpy() for b in bufs] for n, (_, bufs) in others.items()}
    for i in range(4):
        clear(outs)
        torch.cuda.synchronize()
        with torch.cuda.stream(stream):
            graph.replay()
            graph.replay()
        for c, _ in others.values():  # beside the replays
            c()
        torch.cuda.synchronize()
        for b, e in zip(outs, eager):
            np.testing.assert_array_equal(b.to_numpy(), e)
        for n, (_, bufs) in others.items():
            for b, e in zip(bufs, want[n]):
                np.testing.assert_array_equal(b.to_numpy(), e)


def test_calls_that_allocate_can_be_captured(rt):
    """The forms that make their output: the captured call writes the buffer it returned."""
    import torch
    r, own, rng = rx(), rx().Runtime(0), np.random.default_rng(5)
    q, k, v, offsets = prompts(rng, [60, 9], 4, 4, 64, "bf16", first=2, tail=3)
    qb, kb, vb, ob = up(own, q, "bf16"), up(own, k, "bf16"), up(own, v, "bf16"), i32(own, offsets)
    z, u = up(own, floats(rng, (2, 5000), "f32"), "f32"), own.buffer(np.array([.2, .8], np.float32))

    def call():
        return r.grouped_query_attention_packed(own, qb, kb, vb, ob, out_dtype=r.DType.BF16), r.sample(own, z, u)
    eager = [b.to_numpy() for b in call()]  # (their blocks go back to the runtime: the capture takes them)
    stream = torch.cuda.Stream()
    own.synchronize()
    own.set_stream(stream.cuda_stream)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=stream, capture_error_mode="thread_local"):
        outs = call()
    for _ in range(3):
        clear(outs)
        torch.cuda.synchronize()
        with torch.cuda.stream(stream):
            graph.replay()
        torch.cuda.synchronize()
        for b, e in zip(outs, eager):
            np.testing.assert_array_equal(b.to_numpy(), e)
    own.set_stream(None)


def test_a_stream_of_the_callers(rt):
    """Calls go to the stream that the runtime was given: behind what is already on it."""
    import torch
    r, own, rng = rx(), rx().Runtime(0), np.random.default_rng(6)
    kp, vp, table = make_pages(rng, [600, 31], 2, 16, 128, "bf16")
    bufs = [up(own, kp, "bf16"), up(own, vp, "bf16"), i32(own, table), i32(own, [600, 31])]
    host = torch.from_numpy(floats(rng, (2, 8, 128), "f32")).pin_memory()
    q = torch.zeros(2, 8, 128, device="cuda")
    out = torch.zeros(2, 8, 128, device="cuda")
    busy = torch.randn(4096, 4096, device="cuda")
    torch.cuda.synchronize()
    own.synchronize()
    stream = torch.cuda.Stream()
    own.set_stream(stream.cuda_stream)
    with torch.cuda.stream(stream):
        for _ in range(20):
            busy = busy @ busy * 1e-3
        q.copy_(host, non_blocking=True)
        r.grouped_query_attention_paged(own, own.wrap_tensor(q), *bufs, out=own.wrap_tensor(out))
        y = out.clone()
    stream.synchronize()
    own.set_stream(None)
    check(y.cpu().numpy(), *ref.paged_decode(host.numpy(), kp, vp, table, [600, 31]))


def test_two_threads_and_two_runtimes(rt):
    """Two threads, on one runtime and each on its own, call at once and get what one gets."""
    for runtimes in ([rx().Runtime(0)] * 2, [rx().Runtime(0), rx().Runtime(0)]):
        work = [cases(own, np.random.default_rng(8 + i)) for i, own in enumerate(runtimes)]
        want = []
        for w in work:
            for c, _ in w.values():
                c()
            want.append({n: [b.to_numpy() for b in bufs] for n, (_, bufs) in w.items()})
        wrong = []

        def run(i):
            try:
                for _ in range(20):
                    for n, (c, bufs) in work[i].items():
                        c()
                        for b, e in zip(bufs[:1], want[i][n]):
                            if not np.array_equal(b.to_numpy(), e):
                                wrong.append((i, n))
            except Exception as e:  # noqa: BLE001
                wrong.append((i, e))
        threads = [threading.Thread(target=run, args=(i,)) for i in range(2)]
        for t in threads:
            t.start()
        for t in threads:
            t.join(60)
        assert not wrong and not any(t.is_alive() for t in threads)


# ---- sizes past 32 bits --------------------------------------------------------------------

def test_packed_rows_past_32_bits(rt):
    """The last rows of 70000 of 256 heads of 128: offsets of elements past 2^31, of bytes past 2^32."""
    torch = pytest.importorskip("torch")
    r, rng = rx(), np.random.default_rng(9)
    t, hq, hkv, d, n = 70000, 256, 64, 128, 70
    q, k, v = (torch.zeros(t, h, d, dtype=torch.bfloat16, device="cuda") for h in (hq, hkv, hkv))
    out = torch.full((t, hq, d), 3.0, dtype=torch.bfloat16, device="cuda")
    vals = [floats(rng, (n, h, d), "bf16") for h in (hq, hkv, hkv)]
    for x, y in zip((q, k, v), vals):
        x[t - n:].copy_(torch.from_numpy(y))
    torch.cuda.synchronize()
    r.grouped_query_attention_packed(rt, *(rt.wrap_tensor(x) for x in (q, k, v)), i32(rt, [t - n, t - n + 50, t]),
                                     out=rt.wrap_tensor(out))
    rt.synchronize()
    want, bound = ref.packed_prefill(*(x[:, :4 if x.shape[1] == hq else 1] for x in vals), [0, 50, n], p_step=ref.BF16,
                                     out_step=ref.BF16)
    got = out[t - n:, :4].float().cpu().numpy()
    check(got, want, bound)
    last = [x[:, -4:] if x.shape[1] == hq else x[:, -1:] for x in vals]
    check(out[t - n:, -4:].float().cpu().numpy(), *ref.packed_prefill(*last, [0, 50, n], p_step=ref.BF16, out_step=ref.BF16))
    assert bool((out[:t - n] == 3.0).all())


@pytest.mark.parametrize("b,v", [(300, 1 << 24), (70, 1 << 24)])
def test_sample_words_past_32_bits(rt, b, v):
    """Rows of 2^24 words, the longest there are: all alike, and a single one that counts, so that the
    token is known."""
    torch = pytest.importorskip("torch")
    r, rng = rx(), np.random.default_rng(10)
    z = torch.zeros(b, v, dtype=torch.bfloat16, device="cuda")
    at = rng.integers(0, v, b)
    at[-1] = v - 1
    one = (np.arange(b) % 2 == 0) | (np.arange(b) == b - 1)
    for i in np.flatnonzero(one):
        z[i, at[i]] = 60.0  # the others weigh e^-60 V together, nothing beside u = 0.5
    torch.cuda.synchronize()
    u = np.full(b, 0.5, np.float32)
    k = np.where(np.arange(b) % 4 == 1, 1000, 0)
    got = r.sample(rt, rt.wrap_tensor(z), rt.buffer(u), None, i32(rt, k)).to_numpy()
    # of n equal words the first whose running mass exceeds n / 2
    want = [at[i] if one[i] else 500 if k[i] else v // 2 for i in range(b)]
    assert got.tolist() == want


# ---- nothing there -----------------------------------------------------------------------------

@pytest.mark.parametrize("pages,entries", [(0, 3), (4, 0), (0, 0)])
def test_no_pages(rt, pages, entries):
    """A pool without pages, a table without entries: rows see no key, and new rows have no place."""
    r = rx()
    kp, vp = (rt.zeros((pages, 2, 16, 64), r.DType.BF16) for _ in range(2))
    table = rt.zeros((3, entries), r.DType.I32)
    q = rt.buffer(np.ones((3, 4, 64), np.float32))
    y = r.grouped_query_attention_paged(rt, q, kp, vp, table, i32(rt, [5, 0, 70]))
    assert not down(y).any()
    new = rt.buffer(np.ones((3, 2, 64), np.float32))
    r.paged_kv_append(rt, kp, vp, new, new, table, i32(rt, [0, 5, 47]))
    assert not kp.to_numpy().any() and not vp.to_numpy().any()


def test_extreme_positions_and_lengths(rt):
    """Lengths, starts and offsets at the ends of their type."""
    r, rng = rx(), np.random.default_rng(12)
    top = 2 ** 31 - 1
    kp, vp, table = make_pages(rng, [48, 48, 48], 2, 16, 128, "bf16")
    q = floats(rng, (3, 4, 128), "f32")
    pools = [up(rt, kp, "bf16"), up(rt, vp, "bf16")]
    y = down(r.grouped_query_attention_paged(rt, up(rt, q, "f32"), *pools, i32(rt, table), i32(rt, [top, -2 ** 31, 48]),
                                             out_dtype=r.DType.F32))
    check(y, *ref.paged_decode(q, kp, vp, table, [48, 0, 48]))
    new = [floats(rng, (3, 2, 128), "bf16") for _ in range(2)]
    r.paged_kv_append(rt, *pools, *(up(rt, x, "bf16") for x in new), i32(rt, table), i32(rt, [top, -2 ** 31, 47]))
    for pool, old, x in zip(pools, (kp, vp), new):
        assert np.array_equal(down(pool), ref.append(old, x, table, [top, -5, 47], [0, 1, 2, 3]))
    q, k, v, _ = prompts(rng, [30], 4, 2, 128, "f32")
    y = down(r.grouped_query_attention_packed(rt, up(rt, q, "f32"), up(rt, k, "bf16"), up(rt, v, "bf16"),
                                              i32(rt, [-2 ** 31, 9, top]), out_dtype=r.DType.F32))
    check(y, *ref.packed_prefill(q, k, v, [0, 9, 30]))
