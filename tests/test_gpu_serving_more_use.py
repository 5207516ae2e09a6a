"""The operators over 8-bit pages and shared prefixes and the logits' adjustments as a serving
loop uses them: together, captured into graphs, on other streams, from two threads, over tensors
of any alignment and of sizes past 32 bits."""
import threading

import numpy as np
import pytest

import serving_more_ref as more
import serving_ref as ref
from test_gpu_cache8 import make_codes
from test_gpu_logits import adjust, biases, history, masks
from test_gpu_serving import check, down, floats, make_pages, prompts, rx, up
from test_gpu_serving_use import clear, i32
from test_gpu_shared import make, run

pytestmark = pytest.mark.gpu


# ---- refusals, through the package ---------------------------------------------------

def test_refusals_raise_and_leave_the_runtime_usable(rt):
    r, rng = rx(), np.random.default_rng(0)
    kc, vc, ks, vs, table = make_codes(rng, [40, 9], 2, 16, 64)
    pages = [rt.buffer(x) for x in (kc, vc)]
    scales = [rt.buffer(x) for x in (ks, vs)]
    tb, lens = i32(rt, table), i32(rt, [40, 9])
    q = floats(rng, (2, 4, 64), "f32")
    qb, new, two = up(rt, q, "f32"), up(rt, floats(rng, (2, 2, 64), "f32"), "f32"), i32(rt, [0, 1, 2])
    plain = [up(rt, floats(rng, kc.shape, "f32"), "bf16") for _ in range(2)]
    prefix = (i32(rt, [[0]]), i32(rt, [16]), i32(rt, [0, 2]))
    z = up(rt, floats(rng, (2, 100), "f32"), "f32")
    keep = [x.to_numpy() for x in (*pages, *scales)]
    for bad in (lambda: r.paged_kv_append_q8(rt, *pages, *scales, new, up(rt, floats(rng, (2, 2, 32), "f32"), "f32"), tb, lens),
                lambda: r.paged_kv_append_q8(rt, *pages, scales[0], scales[0], new, new, tb, lens),
                lambda: r.paged_kv_append_q8(rt, *plain, *scales, new, new, tb, lens),
                lambda: r.paged_kv_append_q8(rt, *pages, *scales, new, new, tb, i32(rt, [1])),
                lambda: r.paged_kv_read(rt, *pages, tb, lens, two, new, new, k_scales=scales[0], v_scales=scales[1]),
                lambda: r.paged_kv_read(rt, *pages, tb, lens, two, new, up(rt, q[:, :2], "f32")),
                lambda: r.paged_kv_read(rt, *plain, tb, lens, two, new, up(rt, q[:, :2], "f32"), k_scales=scales[0], v_scales=scales[1]),
                lambda: r.grouped_query_attention_paged_q8(rt, qb, *plain, *scales, tb, lens),
                lambda: r.grouped_query_attention_paged_q8(rt, qb, *pages, *scales, tb, lens, scale=float("inf")),
                lambda: r.grouped_query_attention_paged_q8(rt, qb, *pages, *scales, tb, lens, out=qb),
                lambda: r.grouped_query_attention_shared(rt, qb, *pages, *prefix, tb, lens),
                lambda: r.grouped_query_attention_shared(rt, qb, *pages, *prefix, tb, lens, k_scales=scales[0]),
                lambda: r.grouped_query_attention_shared(rt, qb, *plain, *prefix[:2], i32(rt, [0]), tb, lens),
                lambda: r.grouped_query_attention_shared(rt, qb, *plain, *prefix, tb, lens, out_dtype=r.DType.I32),
                lambda: r.adjust_logits(rt, z, repetition=scales[0]),
                lambda: r.adjust_logits(rt, z, tokens=two),
                lambda: r.adjust_logits(rt, z, mask=two),
                lambda: r.adjust_logits(rt, z, out=qb),
                lambda: r.adjust_logits(rt, qb)):
        with pytest.raises(r.Error) as e:
            bad()
        assert e.value.code == r.Status.INVALID_ARGUMENT
    for x, was in zip((*pages, *scales), keep):
        assert np.array_equal(x.to_numpy(), was)
    check(down(r.grouped_query_attention_paged_q8(rt, qb, *pages, *scales, tb, lens)), *more.decode8(q, kc, vc, ks, vs, table, [40, 9]))


# ---- together ------------------------------------------------------------------------

@pytest.mark.parametrize("hq,hkv,d,ps", [(8, 2, 128, 16), (4, 4, 64, 64), (6, 1, 256, 48), (4, 2, 40, 5)])
@pytest.mark.parametrize("kind", ["q8", "bf16"])
def test_a_serving_loop(rt, hq, hkv, d, ps, kind):
    """Two system prompts into pages of their own, read back for the packed attention over them;
    then users behind them, step by step: a row appended, attention over the prefix and their own
    rows, the same over whole tables by paged decode, penalties and a mask by what they said, a token
    whose embedding is the next query. Every attention within its bound of the 64-bit form over
    the pages as they stand, every row of logits within that of the adjustments, every token that of
    the 64-bit form of its logits."""
    r, rng = rx(), np.random.default_rng(d + hq)
    plens, groups, steps, vocab = [3 * ps, 5 * ps], [0, 3, 5], 7, 501
    b = groups[-1]
    kp, vp, ids = make_pages(rng, plens + [steps + 1] * b, hkv, ps, d, "bf16")
    prefixes, table = ids[:2].copy(), ids[2:, :-(-(steps + 1) // ps)].copy()
    pb, tb, gb, lb = i32(rt, prefixes), i32(rt, table), i32(rt, groups), i32(rt, plens)
    shape = kp.shape
    if kind == "q8":
        pools = [rt.buffer(np.full(shape, 9, np.uint8)) for _ in range(2)] + [rt.buffer(np.full(shape[:3], np.nan, np.float32)) for _ in range(2)]
    else:
        pools = [up(rt, np.full(shape, np.nan, np.float32), "bf16") for _ in range(2)]
    scales = dict(k_scales=pools[2], v_scales=pools[3]) if kind == "q8" else {}

    def append(k, v, tables, starts, offsets=None):
        f = r.paged_kv_append_q8 if kind == "q8" else r.paged_kv_append
        f(rt, *pools, up(rt, k, "f32"), up(rt, v, "f32"), tables, starts, *([] if offsets is None else [offsets]))

    def held():  # what the pages hold, and V's scales
        x = [down(p) for p in pools]
        if kind == "bf16":
            return x[0], x[1], None
        zero = [np.nan_to_num(s) for s in x[2:]]
        return more.value(x[0], zero[0]), more.value(x[1], zero[1]), zero[1]

    q, k, v, offsets = prompts(rng, plens, hq, hkv, d, "f32")
    append(k, v, pb, i32(rt, [0, 0]), i32(rt, offsets))
    back = [rt.zeros(k.shape, r.DType.BF16) for _ in range(2)]
    r.paged_kv_read(rt, *pools[:2], pb, i32(rt, [0, 0]), i32(rt, offsets), *back, **scales)
    rows = [down(x) for x in back]
    for got, page in zip(rows, held()):
        want = more.read(page, prefixes, [0, 0], offsets, len(k))
        assert (np.abs(got - want) <= (ref.BF16 + ref.F32) * np.abs(want)).all()
    y = down(r.grouped_query_attention_packed(rt, up(rt, q, "f32"), *back, i32(rt, offsets), out_dtype=r.DType.F32))
    check(y, *ref.packed_prefill(q, *rows, offsets))

    x = y[[offsets[1] - 1] * 3 + [offsets[2] - 1] * 2]
    head = floats(rng, (hq * d, vocab), "f32") / np.float32(np.sqrt(d))
    embed = [floats(rng, (vocab, h, d), "f32") for h in (hq, hkv, hkv)]
    said = [[] for _ in range(b)]
    f32 = np.float32
    allowed = masks(rng, 2, vocab, 0.7)
    mask_rows = np.array([0, -1, 1, 1, 2], np.int32)
    for step in range(steps):
        logits = (x.reshape(b, -1) @ head).astype(f32)
        settings = dict(tokens=np.array(sum(said, []), np.int32), offsets=np.cumsum([0] + [len(s) for s in said]).astype(np.int32),
                        repetition=np.full(b, 1.2, f32), frequency=np.full(b, 0.3, f32), presence=np.full(b, 0.1, f32),
                        **biases(rng, b, vocab, 4), mask=allowed, mask_rows=mask_rows)
        zb = up(rt, logits, "f32")
        r.adjust_logits(rt, zb, out=zb, **{n: rt.buffer(s) for n, s in settings.items()})
        z = down(zb)
        check(z, *more.adjust(logits, 0, **settings))
        u = rng.random(b).astype(f32)
        tokens = r.sample(rt, zb, rt.buffer(u), rt.buffer(np.full(b, 0.8, f32)), i32(rt, [40] * b),
                          rt.buffer(np.full(b, 0.95, f32))).to_numpy()
        assert tokens.tolist() == [ref.sample(z[i], u[i], f32(.8), 40, f32(.95)) for i in range(b)]
        for i, t in enumerate(tokens.tolist()):
            said[i].append(t)
            if mask_rows[i] in (0, 1):
                assert allowed[mask_rows[i]].view(np.uint32)[t // 32] >> (t % 32) & 1
        qs, ks, vs = (e[tokens] for e in embed)
        append(ks, vs, tb, i32(rt, [step] * b))
        lens = [step + 1] * b
        x = down(r.grouped_query_attention_shared(rt, up(rt, qs, "f32"), *pools[:2], pb, lb, gb, tb, i32(rt, lens),
                                                  out_dtype=r.DType.F32, **scales))
        kv, vv, vscale = held()
        want, bound = more.shared(qs, kv, vv, prefixes, plens, groups, table, lens, vs=vscale)
        check(x, want, bound)
        whole = np.concatenate([prefixes[[0] * 3 + [1] * 2], table], axis=1)
        for i in range(3):  # (3 ps positions of the first group: its pages, then its own)
            whole[i, 3:3 + table.shape[1]] = table[i]
        paged = r.grouped_query_attention_paged_q8 if kind == "q8" else r.grouped_query_attention_paged
        z = down(paged(rt, up(rt, qs, "f32"), *pools, i32(rt, whole), i32(rt, [plens[0]] * 3 + [plens[1]] * 2 + np.array(lens)),
                       out_dtype=r.DType.F32))
        assert (np.abs(x - z) <= 2 * bound).all()


# ---- alignment -------------------------------------------------------------------------

@pytest.mark.parametrize("which", ["q", "k", "v", "pages", "out"])
@pytest.mark.parametrize("elements", [1, 3])
def test_operands_at_odd_addresses(rt, which, elements):
    """Tensors that begin an element or more past a 16-byte boundary."""
    torch = pytest.importorskip("torch")
    r, rng = rx(), np.random.default_rng(elements)
    alive = []

    def dev(x, name):
        t = torch.from_numpy(np.ascontiguousarray(x)).cuda()
        if name == which:
            whole = torch.zeros(t.numel() + 16, dtype=t.dtype, device="cuda")
            part = whole[elements:elements + t.numel()].view(t.shape)
            part.copy_(t)
            t = part
        alive.append(t)
        torch.cuda.synchronize()
        return rt.wrap_tensor(t)

    kc, vc, ks, vs, table = make_codes(rng, [50, 20], 2, 16, 64)
    pages, scales = [dev(x, "pages") for x in (kc, vc)], [dev(x, "pages") for x in (ks, vs)]
    tb, lens = i32(rt, table), [40, 13]
    k, v = (floats(rng, (17, 2, 64), "f32") for _ in range(2))
    r.paged_kv_append_q8(rt, *pages, *scales, dev(k, "k"), dev(v, "v"), tb, i32(rt, [30, 6]), i32(rt, [0, 10, 17]))
    for x, codes, s, old in zip((k, v), pages, scales, ((kc, ks), (vc, vs))):
        c, n = more.encode(x)
        want = ref.append(old[0], c, table, [30, 6], [0, 10, 17])
        assert np.array_equal(codes.to_numpy(), want)
        assert np.array_equal(s.to_numpy(), ref.append(old[1][..., None], n[..., None], table, [30, 6], [0, 10, 17])[..., 0])
    now = [x.to_numpy() for x in (*pages, *scales)]
    back = [dev(np.full((17, 2, 64), 5, np.float32), n) for n in ("k", "v")]
    r.paged_kv_read(rt, *pages, tb, i32(rt, [30, 6]), i32(rt, [1, 10, 16]), *back, k_scales=scales[0], v_scales=scales[1])
    for got, c, s in zip(back, now[:2], now[2:]):
        want = more.read(more.value(c, s), table, [30, 6], [1, 10, 16], 17)
        got = got.to_numpy()
        assert (got[[0, 16]] == 5).all() and (np.abs(got - want)[1:16] <= ref.F32 * np.abs(want)[1:16]).all()
    q = floats(rng, (2, 4, 64), "f32")
    qb, out = dev(q, "q"), dev(np.full(q.shape, 5, np.float32), "out")
    r.grouped_query_attention_paged_q8(rt, qb, *pages, *scales, tb, i32(rt, lens), out=out)
    check(out.to_numpy(), *more.decode8(q, now[0], now[1], now[2], now[3], table, lens))
    r.grouped_query_attention_shared(rt, qb, *pages, i32(rt, table[:1]), i32(rt, [33]), i32(rt, [0, 2]), tb, i32(rt, lens), out=out,
                                     k_scales=scales[0], v_scales=scales[1])
    values = [more.value(c, s) for c, s in zip(now[:2], now[2:])]
    check(out.to_numpy(), *more.shared(q, *values, table[:1], [33], [0, 2], table, lens, vs=now[3]))
    z = floats(rng, (3, 1000), "f32")
    zb, zo, some = dev(z, "q"), dev(z, "out"), {**history(rng, 3, 1000, 5, 50), **biases(rng, 3, 1000, 9)}
    r.adjust_logits(rt, zb, out=zo, **{n: rt.buffer(x) for n, x in some.items()})
    check(zo.to_numpy(), *more.adjust(z, 0, **some))


# ---- graphs, streams, threads ------------------------------------------------------------

def cases(own, rng):
    """name: (a call into buffers of its own, its output buffers)."""
    r = rx()
    plens, lens, groups = [700, 90], [40, 1, 333, 80, 5], [0, 3, 4]
    q = up(own, floats(rng, (5, 8, 128), "f32"), "f32")
    ints = {n: i32(own, x) for n, x in (("plens", plens), ("lens", lens), ("groups", groups), ("starts", [39, 0, 332, 79, 4]))}
    new = [up(own, floats(rng, (5, 2, 128), "f32"), "f32") for _ in range(2)]
    _, _, codes, prefixes, table = make(rng, plens, lens, 2, 16, 128, "q8")
    q8 = [own.buffer(x) for x in (codes[0], codes[2], codes[1], codes[3])]
    pb, tb = i32(own, prefixes), i32(own, table)
    kp, vp, _, prefixes, table = make(rng, plens, lens, 2, 16, 128, "bf16")
    bf = [up(own, kp, "bf16"), up(own, vp, "bf16")]
    pb2, tb2 = i32(own, prefixes), i32(own, table)
    y1, y2, y3 = (own.zeros((5, 8, 128), t) for t in (r.DType.F32, r.DType.BF16, r.DType.BF16))
    back = [own.zeros((5, 2, 128), r.DType.BF16) for _ in range(2)]
    z = up(own, floats(rng, (3, 40000), "bf16"), "bf16")
    z1 = own.zeros((3, 40000), r.DType.F32)
    some = {n: own.buffer(x) for n, x in {**history(rng, 3, 40000, 50, 900), **biases(rng, 3, 40000, 90), "mask": masks(rng, 3, 40000)}.items()}
    return {
        "append, read and decode": (lambda: (r.paged_kv_append_q8(own, *q8, *new, tb, ints["starts"]),
                                             r.paged_kv_read(own, *q8[:2], tb, ints["starts"], None, *back, k_scales=q8[2], v_scales=q8[3]),
                                             r.grouped_query_attention_paged_q8(own, q, *q8, tb, ints["lens"], out=y1)), [y1, *back, *q8[:2]]),
        "shared, 8 bits": (lambda: r.grouped_query_attention_shared(own, q, *q8[:2], pb, ints["plens"], ints["groups"], tb, ints["lens"],
                                                                    out=y2, k_scales=q8[2], v_scales=q8[3]), [y2]),
        "shared": (lambda: r.grouped_query_attention_shared(own, q, *bf, pb2, ints["plens"], ints["groups"], tb2, ints["lens"], out=y3), [y3]),
        "logits": (lambda: r.adjust_logits(own, z, out=z1, **some), [z1]),
    }


@pytest.mark.parametrize("name", ["append, read and decode", "shared, 8 bits", "shared", "logits", "all"])
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
    kc, vc, ks, vs, table = make_codes(rng, [200, 33], 2, 16, 128)
    q8, tb, lens = [own.buffer(x) for x in (kc, vc, ks, vs)], i32(own, table), i32(own, [200, 33])
    q, z = up(own, floats(rng, (2, 8, 128), "bf16"), "bf16"), up(own, floats(rng, (2, 9000), "f32"), "f32")
    prefix = [i32(own, x) for x in (table[:1], [77], [0, 2])]
    some = {n: own.buffer(x) for n, x in history(rng, 2, 9000, 50, 100).items()}

    def call():
        return (r.grouped_query_attention_paged_q8(own, q, *q8, tb, lens),
                r.grouped_query_attention_shared(own, q, *q8[:2], *prefix, tb, lens, k_scales=q8[2], v_scales=q8[3]),
                r.adjust_logits(own, z, **some))
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
    kc, vc, ks, vs, table = make_codes(rng, [600, 31], 2, 16, 128)
    bufs = [own.buffer(x) for x in (kc, vc, ks, vs, table)]
    starts, lens, prefix = i32(own, [599, 30]), i32(own, [600, 31]), [i32(own, x) for x in (table[:1], [77], [0, 2])]
    host = [torch.from_numpy(floats(rng, (2, h, 128), "f32")).pin_memory() for h in (8, 2, 2)]
    q, k, v = (torch.zeros(x.shape, device="cuda") for x in host)
    y1, y2 = (torch.zeros(2, 8, 128, device="cuda") for _ in range(2))
    busy = torch.randn(4096, 4096, device="cuda")
    torch.cuda.synchronize()
    own.synchronize()
    stream = torch.cuda.Stream()
    own.set_stream(stream.cuda_stream)
    with torch.cuda.stream(stream):
        for _ in range(20):
            busy = busy @ busy * 1e-3
        for x, h in zip((q, k, v), host):
            x.copy_(h, non_blocking=True)
        r.paged_kv_append_q8(own, *bufs[:4], own.wrap_tensor(k), own.wrap_tensor(v), bufs[4], starts)
        r.grouped_query_attention_paged_q8(own, own.wrap_tensor(q), *bufs, lens, out=own.wrap_tensor(y1))
        r.grouped_query_attention_shared(own, own.wrap_tensor(q), *bufs[:2], *prefix, bufs[4], lens, out=own.wrap_tensor(y2),
                                         k_scales=bufs[2], v_scales=bufs[3])
        got = [y1.clone(), y2.clone()]
        r.adjust_logits(own, own.wrap_tensor(y1.view(2, 1024)), out=own.wrap_tensor(y1.view(2, 1024)))
        same = y1.clone()
    stream.synchronize()
    own.set_stream(None)
    assert torch.equal(same, got[0])
    now = []
    for x, old in zip(host[1:], ((kc, ks), (vc, vs))):
        c, s = more.encode(x.numpy())
        now.append(ref.append(old[0], c, table, [599, 30], [0, 1, 2]))
        now.append(ref.append(old[1][..., None], s[..., None], table, [599, 30], [0, 1, 2])[..., 0])
    kc, ks, vc, vs = now
    check(got[0].cpu().numpy(), *more.decode8(host[0].numpy(), kc, vc, ks, vs, table, [600, 31]))
    check(got[1].cpu().numpy(), *more.shared(host[0].numpy(), more.value(kc, ks), more.value(vc, vs), table[:1], [77], [0, 2], table,
                                             [600, 31], vs=vs))


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

        def several(i):
            try:
                for _ in range(20):
                    for n, (c, bufs) in work[i].items():
                        c()
                        for b, e in zip(bufs[:1], want[i][n]):
                            if not np.array_equal(b.to_numpy(), e):
                                wrong.append((i, n))
            except Exception as e:  # noqa: BLE001
                wrong.append((i, e))
        threads = [threading.Thread(target=several, args=(i,)) for i in range(2)]
        for t in threads:
            t.start()
        for t in threads:
            t.join(60)
        assert not wrong and not any(t.is_alive() for t in threads)


# ---- batches of many rows, prefixes of few positions ----------------------------------------

@pytest.mark.parametrize("hq,hkv,d,kind,qk", [(64, 8, 256, "bf16", "f32"), (64, 8, 256, "q8", "bf16"), (128, 2, 128, "f32", "bf16")])
def test_shared_batches_past_one_launch(rt, hq, hkv, d, kind, qk):
    """More rows than the records of one launch: groups that end inside a launch's part of the batch,
    one over all of them, sequences in none."""
    rng = np.random.default_rng(hq)
    b = 70
    lens = rng.integers(0, 20, b)
    run(rt, rng, [40, 25], [0, 33, 68], lens, hq, hkv, d, kind, qk, "f32")
    run(rt, rng, [70], [1, b], lens, hq, hkv, d, kind, qk, "bf16")


@pytest.mark.parametrize("kind", ["bf16", "q8", "f32"])
@pytest.mark.parametrize("hq,hkv,d", [(64, 8, 128), (8, 8, 64), (16, 1, 256)])
def test_short_prefixes_of_many_rows(rt, hq, hkv, d, kind):
    """Prefixes of less than a tile before many rows: many blocks of one tile each."""
    rng = np.random.default_rng(d)
    lens = rng.integers(0, 4, 90)
    run(rt, rng, [3, 1, 15], [0, 40, 41, 90], lens, hq, hkv, d, kind, "bf16", "f32")
    run(rt, rng, [2], [0, 90], np.zeros(90, int), hq, hkv, d, kind)


@pytest.mark.parametrize("kind,hq,hkv,d", [("bf16", 40, 1, 64), ("q8", 8, 4, 128), ("f32", 4, 4, 64), ("bf16", 6, 2, 256)])
def test_prefixes_of_very_different_lengths(rt, kind, hq, hkv, d):
    """More than 64 groups, of which two have long prefixes, cut into pieces, one of them the last; and
    two, one of them with a sequence less than there are workgroups."""
    rng = np.random.default_rng(d + hq)
    b = 75
    prefix_lens = rng.integers(0, 70, b)
    prefix_lens[[7, 74]] = 2500, 3001
    run(rt, rng, prefix_lens, np.arange(b + 1), rng.integers(0, 30, b), hq, hkv, d, kind, "bf16", "f32")
    run(rt, rng, [2500, 17], [0, 3, 45], np.zeros(45, int), hq, hkv, d, kind, "bf16", "f32")
    run(rt, rng, [40, 1999], [0, 30, 60], rng.integers(0, 200, 60), hq, hkv, d, kind, "bf16", "f32")


# ---- sizes past 32 bits --------------------------------------------------------------------

def test_8_bit_pools_past_32_bits(rt):
    """The last of 70000 pages of 64 KiB: offsets of bytes past 2^32."""
    torch = pytest.importorskip("torch")
    r, rng = rx(), np.random.default_rng(9)
    p, hkv, ps, d, n = 70000, 8, 64, 128, 6
    pools = [torch.full((p, hkv, ps, d), 128, dtype=torch.uint8, device="cuda") for _ in range(2)]
    scales = [torch.full((p, hkv, ps), float("nan"), device="cuda") for _ in range(2)]
    torch.cuda.synchronize()
    wrapped = [rt.wrap_tensor(x) for x in (*pools, *scales)]
    table = np.array([[p - 1, p - 3], [p - 2, p - 4], [p - 5, p - 6]], np.int32)
    small = (table - (p - n)).astype(np.int32)  # in the last n pages by themselves
    counts = [100, 128, 70]
    offsets = np.cumsum([0] + counts)
    k, v = (floats(rng, (offsets[-1], hkv, d), "f32") for _ in range(2))
    r.paged_kv_append_q8(rt, *wrapped, up(rt, k, "f32"), up(rt, v, "f32"), i32(rt, table), i32(rt, [0] * 3), i32(rt, offsets))
    rt.synchronize()
    now = [x[p - n:].cpu().numpy() for x in (*pools, *scales)]
    for x, c, s in ((k, now[0], now[2]), (v, now[1], now[3])):
        codes, want = more.encode(x)
        assert np.array_equal(c, ref.append(np.full(c.shape, 128, np.uint8), codes, small, [0] * 3, offsets))
        assert np.array_equal(s, ref.append(np.full(s.shape + (1,), np.nan, np.float32), want[..., None], small, [0] * 3, offsets)[..., 0],
                              equal_nan=True)
    assert all(bool((x[:p - n] == 128).all()) for x in pools) and all(bool(x[:p - n].isnan().all()) for x in scales)
    back = [rt.zeros(k.shape, r.DType.F32) for _ in range(2)]
    r.paged_kv_read(rt, *wrapped[:2], i32(rt, table), i32(rt, [0] * 3), i32(rt, offsets), *back, k_scales=wrapped[2], v_scales=wrapped[3])
    clean = [np.nan_to_num(s) for s in now[2:]]
    values = [more.value(c, s) for c, s in zip(now[:2], clean)]
    for got, x in zip(back, values):
        want = more.read(x, small, [0] * 3, offsets, len(k))
        assert (np.abs(got.to_numpy() - want) <= ref.F32 * np.abs(want)).all()
    q = floats(rng, (3, 16, d), "f32")
    y = r.grouped_query_attention_paged_q8(rt, up(rt, q, "f32"), *wrapped, i32(rt, table), i32(rt, counts))
    check(down(y), *more.decode8(q, now[0], now[1], *clean, small, counts))
    y = r.grouped_query_attention_shared(rt, up(rt, q[:2], "f32"), *wrapped[:2], i32(rt, table[2:]), i32(rt, [70]), i32(rt, [0, 2]),
                                         i32(rt, table[:2]), i32(rt, counts[:2]), k_scales=wrapped[2], v_scales=wrapped[3])
    check(down(y), *more.shared(q[:2], *values, small[2:], [70], [0, 2], small[:2], counts[:2], vs=clean[1]))


def test_shared_pools_past_32_bits(rt):
    """bf16 pages whose bytes and elements lie past 2^32 and 2^31."""
    torch = pytest.importorskip("torch")
    r, rng = rx(), np.random.default_rng(10)
    p, hkv, ps, d, n = 70000, 4, 64, 128, 6
    kp, vp = (floats(rng, (n, hkv, ps, d), "bf16") for _ in range(2))
    pools = [torch.full((p, hkv, ps, d), float("nan"), dtype=torch.bfloat16, device="cuda") for _ in range(2)]
    for x, y in zip(pools, (kp, vp)):
        x[p - n:].copy_(torch.from_numpy(y))
    torch.cuda.synchronize()
    wrapped = [rt.wrap_tensor(x) for x in pools]
    prefixes, table = np.array([[0, 5]], np.int32), np.array([[1, 2], [4, 3]], np.int32)
    q = floats(rng, (2, 8, d), "f32")
    y = r.grouped_query_attention_shared(rt, up(rt, q, "f32"), *wrapped, i32(rt, prefixes + (p - n)), i32(rt, [110]), i32(rt, [0, 2]),
                                         i32(rt, table + (p - n)), i32(rt, [128, 65]))
    check(down(y), *more.shared(q, kp, vp, prefixes, [110], [0, 2], table, [128, 65]))
    back = [rt.zeros((193, hkv, d), r.DType.BF16) for _ in range(2)]
    r.paged_kv_read(rt, *wrapped, i32(rt, table + (p - n)), i32(rt, [0, 0]), i32(rt, [0, 128, 193]), *back)
    for got, x in zip(back, (kp, vp)):
        assert np.array_equal(down(got), more.read(x, table, [0, 0], [0, 128, 193], 193))


def test_logits_past_32_bits(rt):
    """Rows of 2^24 words, the longest there are, in place: bytes past 2^32, the last row's last word."""
    torch = pytest.importorskip("torch")
    r, b, v = rx(), 140, 1 << 24
    z = torch.ones(b, v, dtype=torch.bfloat16, device="cuda")
    torch.cuda.synchronize()
    rows = np.repeat(np.arange(b), 2)
    words = np.stack([np.full(b, v - 1), (np.arange(b) * 119_123) % (v - 1)], 1).astype(np.int32)
    off = (2 * np.arange(b + 1)).astype(np.int32)
    zb = rt.wrap_tensor(z)
    r.adjust_logits(rt, zb, out=zb, tokens=rt.buffer(words.reshape(-1)), offsets=rt.buffer(off), presence=rt.buffer(np.full(b, 3, np.float32)),
                    bias_words=rt.buffer(words.reshape(-1)), bias=rt.buffer(np.tile([0.5, 0.25], b).astype(np.float32)), bias_offsets=rt.buffer(off))
    rt.synchronize()
    at = (torch.from_numpy(rows).cuda(), torch.from_numpy(words.reshape(-1).astype(np.int64)).cuda())
    assert z[at].tolist() == [-1.5, -1.75] * b
    z[at] = 1
    assert bool((z == 1).all())


# ---- nothing there -----------------------------------------------------------------------------

@pytest.mark.parametrize("pages,entries", [(0, 3), (4, 0), (0, 0)])
def test_no_pages(rt, pages, entries):
    """A pool without pages, tables without entries: rows see no key, new rows have no place, and what
    is read back is 0."""
    r = rx()
    kp, vp = (rt.zeros((pages, 2, 16, 64), r.DType.U8) for _ in range(2))
    ks, vs = (rt.zeros((pages, 2, 16), r.DType.F32) for _ in range(2))
    table = rt.zeros((3, entries), r.DType.I32)
    q, new = rt.buffer(np.ones((3, 4, 64), np.float32)), rt.buffer(np.ones((3, 2, 64), np.float32))
    assert not down(r.grouped_query_attention_paged_q8(rt, q, kp, vp, ks, vs, table, i32(rt, [5, 0, 70]))).any()
    assert not down(r.grouped_query_attention_shared(rt, q, kp, vp, rt.zeros((2, entries), r.DType.I32), i32(rt, [9, 700]), i32(rt, [0, 1, 3]),
                                                     table, i32(rt, [5, 0, 70]), k_scales=ks, v_scales=vs)).any()
    r.paged_kv_append_q8(rt, kp, vp, ks, vs, new, new, table, i32(rt, [0, 5, 47] if not pages or not entries else [48, 48, 48]))
    assert not kp.to_numpy().any() and not vs.to_numpy().any()
    if not pages or not entries:
        back = [rt.buffer(np.full((3, 2, 64), 4, np.float32)) for _ in range(2)]
        r.paged_kv_read(rt, kp, vp, table, i32(rt, [0, 5, 47]), None, *back, k_scales=ks, v_scales=vs)
        assert not any(x.to_numpy().any() for x in back)


@pytest.mark.parametrize("kind", ["bf16", "q8", "f32"])
def test_no_groups_and_no_prefix_pages(rt, kind):
    """No group at all, prefixes without table entries, groups without sequences: plain decode."""
    rng = np.random.default_rng(2)
    run(rt, rng, [], [0], [40, 3, 0], 4, 2, 64, kind)
    run(rt, rng, [0, 0], [0, 1, 3], [40, 3, 0], 4, 2, 64, kind)
    run(rt, rng, [50, 60], [0, 0, 0], [40, 3, 0], 4, 2, 64, kind)
    r = rx()
    kp, vp, codes, _, table = make(rng, [], [40, 3], 2, 16, 64, kind)
    q = floats(rng, (2, 4, 64), "f32")
    pages = [rt.buffer(codes[0]), rt.buffer(codes[2])] if codes else [up(rt, kp, kind), up(rt, vp, kind)]
    scales = dict(k_scales=rt.buffer(codes[1]), v_scales=rt.buffer(codes[3])) if codes else {}
    y = r.grouped_query_attention_shared(rt, up(rt, q, "f32"), *pages, rt.zeros((1, 0), r.DType.I32), i32(rt, [9]), i32(rt, [0, 2]),
                                         i32(rt, table), i32(rt, [40, 3]), out_dtype=r.DType.F32, **scales)
    check(down(y), *more.shared(q, kp, vp, np.zeros((1, 0), np.int32), [9], [0, 2], table, [40, 3], vs=codes and codes[3]))


def test_extreme_positions_and_lengths(rt):
    """Lengths, starts and offsets at the ends of their type."""
    r, rng = rx(), np.random.default_rng(12)
    top, low = 2 ** 31 - 1, -2 ** 31
    kc, vc, ks, vs, table = make_codes(rng, [48, 48, 48], 2, 16, 128)
    q = floats(rng, (3, 4, 128), "f32")
    bufs = [rt.buffer(x) for x in (kc, vc, ks, vs)]
    y = down(r.grouped_query_attention_paged_q8(rt, up(rt, q, "f32"), *bufs, i32(rt, table), i32(rt, [top, low, 48])))
    check(y, *more.decode8(q, kc, vc, ks, vs, table, [48, 0, 48]))
    y = down(r.grouped_query_attention_shared(rt, up(rt, q, "f32"), *bufs[:2], i32(rt, table[1:]), i32(rt, [top, low]), i32(rt, [low, 2, top]),
                                              i32(rt, table), i32(rt, [low, top, 1]), k_scales=bufs[2], v_scales=bufs[3]))
    values = more.value(kc, ks), more.value(vc, vs)
    check(y, *more.shared(q, *values, table[1:], [48, 0], [0, 2, 3], table, [0, 48, 1], vs=vs))
    new = [floats(rng, (3, 2, 128), "f32") for _ in range(2)]
    r.paged_kv_append_q8(rt, *bufs, *(up(rt, x, "f32") for x in new), i32(rt, table), i32(rt, [top, low, 47]))
    for x, codes, s, old in zip(new, bufs[:2], bufs[2:], ((kc, ks), (vc, vs))):
        c, n = more.encode(x)
        assert np.array_equal(codes.to_numpy(), ref.append(old[0], c, table, [top, -5, 47], [0, 1, 2, 3]))
        assert np.array_equal(s.to_numpy(), ref.append(old[1][..., None], n[..., None], table, [top, -5, 47], [0, 1, 2, 3])[..., 0])
    back = [rt.buffer(np.full((5, 2, 128), 4, np.float32)) for _ in range(2)]
    r.paged_kv_read(rt, *bufs[:2], i32(rt, table), i32(rt, [low, 47, top]), i32(rt, [low, 2, 4, top]), *back, k_scales=bufs[2],
                    v_scales=bufs[3])
    for got, c, s in zip(back, bufs[:2], bufs[2:]):
        x = more.value(c.to_numpy(), s.to_numpy())
        got = got.to_numpy()
        # sequence 0 begins at -2^31 and its rows at -2^31: row i holds position i; 1 at 47; 2 past every position
        want = np.zeros((5, 2, 128))
        want[0], want[1], want[2] = x[table[0, 0], :, 0], x[table[0, 0], :, 1], x[table[1, 2], :, 15]
        assert (np.abs(got - want) <= ref.F32 * np.abs(want)).all()
    z, words = floats(rng, (2, 64), "f32"), np.array([3, low, top, 63, 64, -1, 3], np.int32)
    some = dict(tokens=words, offsets=np.array([low, 4, top], np.int32), prompts=np.array([low, 1], np.int32),
                presence=np.ones(2, np.float32), frequency=np.ones(2, np.float32))
    check(adjust(rt, z, "f32", **some), *more.adjust(z, 0, tokens=words, offsets=[0, 4, 7], prompts=[0, 1], presence=some["presence"],
                                                     frequency=some["frequency"]))
    some = dict(tokens=words, offsets=np.array([0, 4, 7], np.int32), prompts=np.array([top, 1], np.int32), presence=np.ones(2, np.float32))
    check(adjust(rt, z, "f32", **some), *more.adjust(z, 0, **some))
