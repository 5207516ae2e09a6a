"""The serving operators' host code on the CPU: what they refuse, with which status and
before anything is launched, and the launches that they plan."""
import ctypes as c
import os
import random
import subprocess

import pytest

HERE = os.path.dirname(os.path.abspath(__file__))
U8, I32, BF16, F32 = 1, 2, 4, 5  # of include/rxw8.h
OK, INVALID, UNIMPLEMENTED = 0, 3, 12
ITEM = {F32: 4, I32: 4, BF16: 2, U8: 1}


@pytest.fixture(scope="module")
def lib(tmp_path_factory):
    so = str(tmp_path_factory.mktemp("serving") / "serving_host.so")
    subprocess.run(["g++", "-std=c++17", "-O1", "-fPIC", "-shared", "-Wl,-Bsymbolic", "-D__HIP_PLATFORM_AMD__", "-I/opt/rocm/include",
                    "-I", os.path.join(HERE, "..", "include"), os.path.join(HERE, "serving_host.cpp"), "-o", so],
                   check=True)
    lib = c.CDLL(so)
    for name in ("host_runtime", "host_buffer"):
        getattr(lib, name).restype = c.c_void_p
    for name in ("host_message", "host_launch"):
        getattr(lib, name).restype = c.c_char_p
    lib.host_runtime.argtypes = [c.c_int, c.c_size_t]
    lib.host_buffer.argtypes = [c.c_void_p, c.c_int, c.c_int, c.c_void_p, c.c_size_t, c.c_int64]
    p, f, i = c.c_void_p, c.c_float, c.c_int
    lib.rxw8_paged_kv_append.argtypes = [p] * 8
    lib.rxw8_gqa_decode_paged.argtypes = [p] * 6 + [f, i, p]
    lib.rxw8_gqa_decode_paged_into.argtypes = [p] * 6 + [f, p]
    lib.rxw8_gqa_prefill_packed.argtypes = [p] * 5 + [f, i, p]
    lib.rxw8_gqa_prefill_packed_into.argtypes = [p] * 5 + [f, p]
    lib.rxw8_sample.argtypes = lib.rxw8_sample_into.argtypes = [p] * 8
    return lib


class Host:
    def __init__(self, lib, cus=256, lds=160 << 10):
        self.lib, self.rt, self.at = lib, lib.host_runtime(cus, lds), 1 << 30
        lib.host_launches(1)

    def buf(self, dtype, *dims, at=None, rt=None):
        n = ITEM[dtype]
        for d in dims:
            n *= d
        if at is None:
            at, self.at = self.at, self.at + ((n + 255) & ~255) + 256
        return self.lib.host_buffer(rt or self.rt, dtype, len(dims), (c.c_int64 * 8)(*dims), at, n)

    def launches(self):
        n = self.lib.host_launches(0)
        got = []
        for i in range(n):
            g, t, l = c.c_uint(), c.c_uint(), c.c_uint()
            name = self.lib.host_launch(i, c.byref(g), c.byref(t), c.byref(l)).decode()
            got.append((name, g.value, t.value, l.value))
        self.lib.host_launches(1)
        return got


# name: the arguments of a call that is right, as (dtype, dims), and the entry points' own ends
def shapes(op):
    return {
        "append": dict(k_pages=(BF16, 9, 2, 16, 64), v_pages=(BF16, 9, 2, 16, 64), k=(F32, 7, 2, 64), v=(F32, 7, 2, 64),
                       table=(I32, 3, 4), starts=(I32, 3), offsets=(I32, 4)),
        "decode": dict(q=(F32, 3, 8, 64), k_pages=(BF16, 9, 2, 16, 64), v_pages=(BF16, 9, 2, 16, 64), table=(I32, 3, 4),
                       lens=(I32, 3), scale=0.125, out=(F32, 3, 8, 64)),
        "prefill": dict(q=(F32, 7, 8, 64), k=(BF16, 7, 2, 64), v=(BF16, 7, 2, 64), offsets=(I32, 4), scale=0.125,
                        out=(BF16, 7, 8, 64)),
        "sample": dict(logits=(BF16, 5, 100), uniform=(F32, 5), temperature=(F32, 5), top_k=(I32, 5), top_p=(F32, 5),
                       min_p=(F32, 5), out=(I32, 5)),
    }[op]


ENTRY = {"append": "rxw8_paged_kv_append", "decode": "rxw8_gqa_decode_paged", "prefill": "rxw8_gqa_prefill_packed",
         "sample": "rxw8_sample"}


def call(host, op, into=True, rt=True, **change):
    """The status of a call whose arguments are those of shapes(op) but for `change` (a tuple: another
    shape; None: NULL; an int: that buffer)."""
    args = {**shapes(op), **change}
    out_dtype = args.pop("out_dtype", F32)
    if not into:
        args.pop("out", None)
    bufs = [host.buf(*x) if isinstance(x, tuple) else x for x in args.values()]
    lib, name = host.lib, ENTRY[op]
    if op == "append":
        return getattr(lib, name)(host.rt if rt else None, *bufs)
    if into:
        return getattr(lib, name + "_into")(host.rt if rt else None, *bufs)
    out = c.c_void_p(0)
    ends = [c.byref(out)] if op == "sample" else [out_dtype, c.byref(out)]
    rc = getattr(lib, name)(host.rt if rt else None, *bufs, *ends)
    assert (rc == OK) == bool(out.value)
    return rc


@pytest.mark.parametrize("op,into", [(op, into) for op in ENTRY for into in (True, False) if op != "append" or into])
def test_right_calls_launch(lib, op, into):
    host = Host(lib)
    assert call(host, op, into) == OK and host.launches()
    if op == "append":
        assert call(host, op, offsets=None, k=(F32, 3, 2, 64), v=(F32, 3, 2, 64)) == OK
    if op == "sample":
        assert call(host, op, into, temperature=None, top_k=None, top_p=None, min_p=None) == OK
    # no rows: nothing to launch
    host.launches()
    none = {"append": dict(k=(F32, 0, 2, 64), v=(F32, 0, 2, 64)),
            "decode": dict(q=(F32, 0, 8, 64), table=(I32, 0, 4), lens=(I32, 0), out=(F32, 0, 8, 64)),
            "prefill": dict(q=(F32, 0, 8, 64), k=(BF16, 0, 2, 64), v=(BF16, 0, 2, 64), out=(BF16, 0, 8, 64)),
            "sample": dict(logits=(F32, 0, 100), out=(I32, 0), **{x: (F32, 0) for x in ("uniform", "temperature", "top_p", "min_p")},
                           top_k=(I32, 0))}[op]
    if not into:
        none.pop("out", None)
    assert call(host, op, into, **none) == OK and not host.launches()


REFUSED = {
    "append": [
        dict(k_pages=(BF16, 9, 2, 16, 32)), dict(v_pages=(F32, 9, 2, 16, 64)), dict(v_pages=(BF16, 8, 2, 16, 64)),
        dict(k_pages=(BF16, 18, 16, 64), v_pages=(BF16, 18, 16, 64)), dict(k=(F32, 7, 2, 32), v=(F32, 7, 2, 32)),
        dict(k=(F32, 7, 4, 64), v=(F32, 7, 4, 64)), dict(v=(BF16, 7, 2, 64)), dict(v=(F32, 6, 2, 64)), dict(k=(F32, 7, 128)),
        dict(k=(I32, 7, 2, 64), v=(I32, 7, 2, 64)), dict(table=(F32, 3, 4)), dict(table=(I32, 12)), dict(table=(I32, 4, 4)),
        dict(starts=(I32, 2)), dict(starts=(F32, 3)), dict(starts=(I32, 3, 1)), dict(offsets=(I32, 3)), dict(offsets=(F32, 4)),
        dict(offsets=None), dict(k_pages=(BF16, 9, 0, 16, 64), v_pages=(BF16, 9, 0, 16, 64), k=(F32, 7, 0, 64), v=(F32, 7, 0, 64)),
        dict(k_pages=(BF16, 9, 2, 0, 64), v_pages=(BF16, 9, 2, 0, 64))],
    "decode": [
        dict(q=(F32, 3, 7, 64), out=(F32, 3, 7, 64)), dict(q=(F32, 3, 0, 64), out=(F32, 3, 0, 64)), dict(q=(I32, 3, 8, 64)),
        dict(q=(F32, 3, 512)), dict(q=(F32, 4, 8, 64)), dict(q=(F32, 3, 8, 128), out=(F32, 3, 8, 128)), dict(table=(I32, 4, 4)),
        dict(table=(U8, 3, 4)), dict(lens=(I32, 4)), dict(lens=(F32, 3)), dict(lens=(I32, 3, 1)), dict(out=(F32, 3, 8, 32)),
        dict(out=(I32, 3, 8, 64)), dict(out=(F32, 24, 64)), dict(scale=float("nan")), dict(scale=float("inf")),
        dict(k_pages=(F32, 9, 2, 16, 64)), dict(v_pages=(BF16, 9, 2, 32, 64))],
    "prefill": [
        dict(q=(F32, 8, 8, 64)), dict(q=(F32, 7, 9, 64), out=(F32, 7, 9, 64)), dict(q=(F32, 7, 8, 32), out=(F32, 7, 8, 32)),
        dict(k=(F32, 7, 2, 64), v=(F32, 7, 2, 64)), dict(v=(BF16, 7, 4, 64)), dict(k=(BF16, 7, 0, 64), v=(BF16, 7, 0, 64)),
        dict(q=(F32, 7, 0, 64), out=(F32, 7, 0, 64)), dict(offsets=(F32, 4)), dict(offsets=(I32, 2, 2)), dict(offsets=(I32, 0)),
        dict(out=(BF16, 7, 8, 32)), dict(out=(I32, 7, 8, 64)), dict(out=(BF16, 6, 8, 64)), dict(scale=float("-inf")),
        dict(q=(F32, 7, 8, 0), k=(BF16, 7, 2, 0), v=(BF16, 7, 2, 0), out=(F32, 7, 8, 0))],
    "sample": [
        dict(logits=(F32, 500)), dict(logits=(I32, 5, 100)), dict(logits=(F32, 5, 0)), dict(uniform=(F32, 4)), dict(uniform=(BF16, 5)),
        dict(temperature=(F32, 1)), dict(temperature=(F32, 5, 1)), dict(top_k=(F32, 5)), dict(top_p=(I32, 5)), dict(min_p=(F32, 6)),
        dict(out=(F32, 5)), dict(out=(I32, 6)), dict(out=(I32, 5, 1)), dict(uniform=None), dict(logits=None)],
}


@pytest.mark.parametrize("op", ENTRY)
def test_wrong_arguments_are_refused(lib, op):
    host = Host(lib)
    for change in REFUSED[op]:
        change = dict(change)
        assert call(host, op, **change) == INVALID, change
        if op != "append" and set(change) != {"out"}:
            change.pop("out", None)
            assert call(host, op, into=False, **change) == INVALID, change
        assert lib.host_message() and not host.launches(), change


@pytest.mark.parametrize("op", ENTRY)
def test_null_arguments_are_refused(lib, op):
    host = Host(lib)
    optional = {"append": {"offsets"}, "sample": {"temperature", "top_k", "top_p", "min_p"}}.get(op, set())
    for name in shapes(op):
        if name not in optional | {"scale"}:
            assert call(host, op, **{name: None}) == INVALID, name
            assert name == "out" or op == "append" or call(host, op, into=False, **{name: None}) == INVALID, name
    assert call(host, op, rt=False) == INVALID
    if op in ("decode", "prefill"):
        assert call(host, op, into=False, out_dtype=I32) == INVALID
    assert not host.launches()


@pytest.mark.parametrize("op", ENTRY)
def test_buffers_of_another_runtime_and_shared_memory_are_refused(lib, op):
    host, other = Host(lib), Host(lib)
    written = {"append": ["k_pages", "v_pages"]}.get(op, ["out"])
    for name, x in shapes(op).items():
        if not isinstance(x, tuple):
            continue
        assert call(host, op, **{name: host.buf(*x, rt=other.rt)}) == INVALID, name
        assert name == "out" or op == "append" or call(host, op, into=False, **{name: host.buf(*x, rt=other.rt)}) == INVALID
        for w in written:
            if w == name:
                continue
            whole = shapes(op)[w]
            size = ITEM[whole[0]]
            for d in whole[1:]:
                size *= d
            at = 1 << 45
            assert call(host, op, **{w: host.buf(*whole, at=at), name: host.buf(*x, at=at + size - 4)}) == INVALID, (w, name)
            assert not host.launches()
            assert call(host, op, **{w: host.buf(*whole, at=at), name: host.buf(*x, at=at + size)}) == OK, (w, name)
            host.launches()
    assert call(host, op) == OK
    if op == "append":  # what is only read may share memory
        kv = host.buf(F32, 7, 2, 64)
        assert call(host, op, k=kv, v=kv) == OK
        pages = host.buf(BF16, 9, 2, 16, 64)
        assert call(host, op, k_pages=pages, v_pages=pages) == INVALID


def test_sizes_past_the_kernels_are_refused(lib):
    host = Host(lib)
    for change in (dict(q=(F32, 3, 8, 513), k_pages=(BF16, 9, 2, 16, 513), v_pages=(BF16, 9, 2, 16, 513), out=(F32, 3, 8, 513)),
                   dict(table=(I32, 3, 1 << 27)), dict(k_pages=(BF16, 9, 2, 1 << 29, 64), v_pages=(BF16, 9, 2, 1 << 29, 64)),
                   dict(k_pages=(BF16, 9, 2, 1 << 31, 64), v_pages=(BF16, 9, 2, 1 << 31, 64)),
                   dict(q=(F32, 1 << 21, 8, 64), table=(I32, 1 << 21, 4), lens=(I32, 1 << 21), out=(F32, 1 << 21, 8, 64))):
        assert call(host, "decode", **change) == UNIMPLEMENTED, change
    for change in (dict(q=(F32, 7, 8, 576), k=(BF16, 7, 2, 576), v=(BF16, 7, 2, 576), out=(F32, 7, 8, 576)),
                   dict(q=(F32, 1 << 23, 8, 64), k=(BF16, 1 << 23, 2, 64), v=(BF16, 1 << 23, 2, 64), out=(F32, 1 << 23, 8, 64))):
        assert call(host, "prefill", **change) == UNIMPLEMENTED, change
    assert call(host, "append", table=(I32, 3, 1 << 28)) == UNIMPLEMENTED
    assert call(host, "append", k=(F32, 1 << 25, 2, 64), v=(F32, 1 << 25, 2, 64)) == UNIMPLEMENTED
    assert call(host, "sample", logits=(BF16, 5, (1 << 24) + 1)) == UNIMPLEMENTED
    b = 1 << 22
    assert call(host, "sample", logits=(BF16, b, 2), uniform=(F32, b), temperature=None, top_k=None, top_p=None, min_p=None,
                out=(I32, b)) == UNIMPLEMENTED
    assert not host.launches()
    assert call(host, "sample", logits=(BF16, 5, 1 << 24)) == OK


def test_decode_plans(lib):
    """Launches of random shapes: known kernels, threads within a launch's, LDS within the device's, and
    counters and records within the runtime's block, that of captured calls for a captured call."""
    host, rng, seen = Host(lib), random.Random(1), set()
    for _ in range(4000):
        d, es = rng.choice([8, 64, 128, 200, 256, 512]), rng.choice([BF16, F32])
        hkv, g = rng.choice([1, 2, 3, 8, 64, 300, 4097]), rng.choice([1, 2, 4, 5, 8, 16, 17, 40])
        b, ps, m, p = rng.choice([1, 2, 37, 700]), rng.choice([1, 16, 40, 64, 1024]), rng.choice([0, 1, 30, 2000]), rng.choice([0, 1, 50])
        captured = rng.random() < 0.5
        odd = rng.choice([0, 0, 0, 2, 8])
        lib.host_capturing(int(captured))
        q = host.buf(F32, b, hkv * g, d, at=(1 << 44) + odd * (rng.random() < 0.5))
        pages = [host.buf(es, p, hkv, ps, d, at=(x << 46) + odd) for x in (1, 2)]
        rc = call(host, "decode", q=q, k_pages=pages[0], v_pages=pages[1], table=(I32, b, m), lens=(I32, b),
                  out=host.buf(F32, b, hkv * g, d, at=1 << 50))
        assert rc == (OK if b * hkv * g < 1 << 24 else UNIMPLEMENTED)
        if rc:
            continue
        (name, grid, threads, lds), = host.launches()
        seen.add(name)
        assert grid * threads < 1 << 32 and lds <= 160 << 10
        if odd or d not in (64, 128, 256) or ps % 16 or not p:
            assert name == "rxw8_paged_decode_any" and grid == b * hkv * g
        if name == "rxw8_paged_decode_any":
            continue
        assert name == "rxw8_paged_decode_%s_d%d" % ("f32" if es == F32 else "bf16", d) and threads == 512
        got = (c.c_int64 * 4)()
        lib.host_decode(got)
        units, waves, counters, part = got
        heads = hkv * -(-g // 16)
        assert grid == heads * units and 1 <= units <= 256 and 1 <= waves <= 8
        block = (2 if captured else 1) << 40
        assert counters == block and part == block + (64 << 10) and 4 * grid <= 64 << 10
        record = -(-min(g, 16) * (d + 4) * 4 // 1024) * 1024  # (one workgroup to a head leaves no records)
        assert units == 1 or 2 * grid * record <= 16 << 20
    lib.host_capturing(0)
    assert len(seen) == 7


def test_prefill_plans(lib):
    host, rng, seen = Host(lib), random.Random(2), set()
    for _ in range(4000):
        d, qt, ot = rng.choice([8, 64, 128, 200, 256, 512]), rng.choice([BF16, F32]), rng.choice([BF16, F32])
        hkv, g = rng.choice([1, 2, 3, 8, 64]), rng.choice([1, 2, 3, 4, 6, 8, 12])
        t, b, odd = rng.choice([1, 2, 31, 700, 50000]), rng.choice([0, 1, 5, 900]), rng.choice([0, 0, 0, 2, 8])
        args = dict(q=host.buf(qt, t, hkv * g, d, at=1 << 44), k=host.buf(BF16, t, hkv, d, at=(1 << 45) + odd),
                    v=(BF16, t, hkv, d), offsets=(I32, b + 1))
        into = rng.random() < 0.5
        if into:
            args["out"] = host.buf(ot, t, hkv * g, d, at=1 << 50)
        assert call(host, "prefill", into=into, **(args if into else dict(args, out_dtype=ot))) == OK
        got = host.launches()
        seen.add(got[-1][0])
        for name, grid, threads, lds in got:
            assert grid * threads < 1 << 32 and lds <= 160 << 10
        matrix = d in (64, 128, 256) and not odd
        assert [x[0] for x in got[:-1]] == (["rxw8_packed_fill"] if matrix and not into else [])
        name = got[-1][0]
        if not matrix:
            assert name == "rxw8_packed_prefill_any" and got[-1][1] == (t * hkv * g + 3) // 4
            continue
        kind = "f32" if qt == F32 else "bf16_f32" if ot == F32 else "bf16"
        heads = 4 if g % 4 == 0 else 2 if g % 2 == 0 else 1
        rows = (64 if kind == "bf16" and d == 64 else 32) * (4 // heads)
        grid = (-(-t // rows) + b) * hkv * g // heads
        mean = t / max(b, 1)
        rounds = min(0.4 + mean / 800, 1.05) if kind == "bf16" and d > 64 else min(0.75 + mean / 512, 2)
        few = (t / 32 + b / 2) * hkv * g <= rounds * (1 if d == 256 else 2) * 256
        assert name == "rxw8_packed_%s_%s_d%d" % ("quarters" if few else "prefill", kind, d)
        assert got[-1][1] == ((-(-t // 32) + b) * hkv * g if few else grid)
    assert len(seen) == 19


def test_append_plans(lib):
    host, rng = Host(lib), random.Random(3)
    for _ in range(1000):
        t, hkv, d = rng.choice([1, 7, 5000]), rng.choice([1, 3, 8, 64]), rng.choice([1, 8, 12, 64, 128, 1000])
        odd, nk, pk = rng.choice([0, 0, 4, 8]), rng.choice([BF16, F32]), rng.choice([BF16, F32])
        assert call(host, "append", k=(nk, t, hkv, d), v=host.buf(nk, t, hkv, d, at=(1 << 45) + odd), k_pages=(pk, 9, hkv, 16, d),
                    v_pages=(pk, 9, hkv, 16, d)) == OK
        (name, grid, threads, lds), = host.launches()
        any_ = d % 8 != 0 or odd != 0
        waves = t * (hkv if any_ else -(-hkv * d // 8 // 128))
        assert name == "rxw8_paged_append" + ("_any" if any_ else "") and threads == 256 and grid == -(-waves // 4)


def test_sample_plans(lib):
    """Workgroups that share rows: their chunks cover the row, and their records and counters lie apart
    from each other within the runtime's block."""
    host, rng, shared = Host(lib), random.Random(4), set()
    for _ in range(4000):
        b = rng.choice([1, 2, 31, 32, 33, 64, 100, 128, 129, 300])
        v = rng.choice([1, 2, 1000, 49152, 56173, 56174, 98304, 151936, 248320, 1 << 24])
        captured = rng.random() < 0.5
        lib.host_capturing(int(captured))
        vec = {x: (F32, b) for x in ("uniform", "temperature", "top_p", "min_p")}
        assert call(host, "sample", logits=host.buf(BF16, b, v, at=1 << 47), **vec, top_k=(I32, b), out=(I32, b)) == OK
        launches = host.launches()
        got = (c.c_int64 * 7)()
        lib.host_sample(got)
        s, chunk, shift, extremes, arrivals, listed, bins = got
        assert v << shift <= 1 << 62 and (shift == 51 or v << (shift + 1) > 1 << 62) and shift <= 51
        shared.add(s)
        names = ["rxw8_sample_extremes", "rxw8_sample_draw", "rxw8_sample_words"] if s > 1 else ["rxw8_sample_draw"]
        assert launches == [(n, b * s, 1024, 92 << 10) for n in names]
        assert 1 <= s <= 8 and chunk * (s - 1) < v <= chunk * s and b * s <= max(b, 256)
        if s > 1:
            block = (2 if captured else 1) << 40
            assert arrivals == block and listed == arrivals + 4 * b and listed + 4 * b <= extremes
            assert extremes == block + (64 << 10) and extremes + 16 * b * s <= bins
            assert bins + (12 << 10) * b * s <= block + (64 << 10) + (16 << 20)
    lib.host_capturing(0)
    assert shared == {1, 2, 4, 7, 8}
