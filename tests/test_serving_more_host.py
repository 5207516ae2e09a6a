"""The host code of the operators over 8-bit pages and shared prefixes and of the logits'
adjustments on the CPU: what they refuse, with which status and before anything is launched, and
the launches that they plan."""
import ctypes as c
import os
import random
import subprocess

import pytest

from rxla_amd import _ffi
from test_serving_host import BF16, F32, HERE, I32, INVALID, ITEM, OK, U8, UNIMPLEMENTED, Host

LOGITS = ["tokens", "offsets", "prompts", "repetition", "frequency", "presence", "bias_words", "bias", "bias_offsets",
          "mask", "mask_rows"]


class Options(c.Structure):
    _fields_ = [(x, c.c_void_p) for x in LOGITS]


@pytest.fixture(scope="module")
def lib(tmp_path_factory):
    so = str(tmp_path_factory.mktemp("serving") / "serving_more_host.so")
    subprocess.run(["g++", "-std=c++17", "-O1", "-fPIC", "-shared", "-Wl,-Bsymbolic", "-D__HIP_PLATFORM_AMD__", "-I/opt/rocm/include",
                    "-I", os.path.join(HERE, "..", "include"), os.path.join(HERE, "serving_more_host.cpp"), "-o", so],
                   check=True)
    lib = c.CDLL(so)
    for name in ("host_runtime", "host_buffer"):
        getattr(lib, name).restype = c.c_void_p
    for name in ("host_message", "host_launch"):
        getattr(lib, name).restype = c.c_char_p
    lib.host_runtime.argtypes = [c.c_int, c.c_size_t]
    lib.host_buffer.argtypes = [c.c_void_p, c.c_int, c.c_int, c.c_void_p, c.c_size_t, c.c_int64]
    p, f, i = c.c_void_p, c.c_float, c.c_int
    lib.rxw8_paged_kv_append_q8.argtypes = lib.rxw8_paged_kv_read.argtypes = [p] * 10
    lib.rxw8_gqa_decode_paged_q8.argtypes = [p] * 8 + [f, i, p]
    lib.rxw8_gqa_decode_paged_q8_into.argtypes = [p] * 8 + [f, p]
    lib.rxw8_gqa_decode_shared.argtypes = [p] * 11 + [f, i, p]
    lib.rxw8_gqa_decode_shared_into.argtypes = [p] * 11 + [f, p]
    lib.rxw8_adjust_logits.argtypes = [p, p, p, i, p]
    lib.rxw8_adjust_logits_into.argtypes = [p] * 4
    return lib


PAGES = dict(k_pages=(U8, 9, 2, 16, 64), v_pages=(U8, 9, 2, 16, 64), k_scales=(F32, 9, 2, 16), v_scales=(F32, 9, 2, 16))
PLAIN = dict(k_pages=(BF16, 9, 2, 16, 64), v_pages=(BF16, 9, 2, 16, 64), k_scales=None, v_scales=None)
SHAPES = {
    "append": dict(**PAGES, k=(F32, 7, 2, 64), v=(F32, 7, 2, 64), table=(I32, 3, 4), starts=(I32, 3), offsets=(I32, 4)),
    "read": dict(**PAGES, table=(I32, 3, 4), starts=(I32, 3), offsets=(I32, 4), k=(BF16, 7, 2, 64), v=(BF16, 7, 2, 64)),
    "decode": dict(q=(F32, 3, 8, 64), **PAGES, table=(I32, 3, 4), lens=(I32, 3), scale=0.125, out=(F32, 3, 8, 64)),
    "shared": dict(q=(F32, 3, 8, 64), **PAGES, prefixes=(I32, 2, 5), prefix_lens=(I32, 2), groups=(I32, 3), table=(I32, 3, 4),
                   lens=(I32, 3), scale=0.125, out=(F32, 3, 8, 64)),
    "logits": dict(logits=(BF16, 5, 100), tokens=(I32, 40), offsets=(I32, 6), prompts=(I32, 5), repetition=(F32, 5),
                   frequency=(F32, 5), presence=(F32, 5), bias_words=(I32, 9), bias=(F32, 9), bias_offsets=(I32, 6),
                   mask=(I32, 3, 4), mask_rows=(I32, 5), out=(F32, 5, 100)),
}
ENTRY = {"append": "rxw8_paged_kv_append_q8", "read": "rxw8_paged_kv_read", "decode": "rxw8_gqa_decode_paged_q8",
         "shared": "rxw8_gqa_decode_shared", "logits": "rxw8_adjust_logits"}
WRITTEN = {"append": ["k_pages", "v_pages", "k_scales", "v_scales"], "read": ["k", "v"]}
ALLOCATES = [op for op in SHAPES if op not in WRITTEN]
FORMS = [(op, into) for op in ENTRY for into in (True, False) if into or op in ALLOCATES]


def call(host, op, into=True, rt=True, options=True, **change):
    """The status of a call whose arguments are those of SHAPES[op] but for `change` (a tuple: another
    shape; None: NULL; an int: that buffer)."""
    args = {**SHAPES[op], **change}
    out_dtype = args.pop("out_dtype", F32)
    if not into:
        args.pop("out", None)
    bufs = {n: host.buf(*x) if isinstance(x, tuple) else x for n, x in args.items()}
    if op == "logits":
        o = Options(**{n: bufs.pop(n) for n in LOGITS})
        bufs = {"logits": bufs["logits"], "options": c.byref(o) if options else None, **({"out": bufs["out"]} if into else {})}
    fn = getattr(host.lib, ENTRY[op] + ("_into" if into and op in ALLOCATES else ""))
    if into:
        return fn(host.rt if rt else None, *bufs.values())
    out = c.c_void_p(0)
    rc = fn(host.rt if rt else None, *bufs.values(), out_dtype, c.byref(out))
    assert (rc == OK) == bool(out.value)
    return rc


def test_the_packages_options_are_the_headers():
    assert [n for n, _ in _ffi.LogitsOptions._fields_] == LOGITS


NONE = {"append": dict(k=(F32, 0, 2, 64), v=(F32, 0, 2, 64)), "read": dict(k=(F32, 0, 2, 64), v=(F32, 0, 2, 64)),
        "decode": dict(q=(F32, 0, 8, 64), table=(I32, 0, 4), lens=(I32, 0), out=(F32, 0, 8, 64)),
        "shared": dict(q=(F32, 0, 8, 64), table=(I32, 0, 4), lens=(I32, 0), out=(F32, 0, 8, 64)),
        "logits": dict(logits=(F32, 0, 100), offsets=(I32, 1), prompts=(I32, 0), repetition=(F32, 0), frequency=(F32, 0),
                       presence=(F32, 0), bias_offsets=(I32, 1), mask_rows=(I32, 0), out=(F32, 0, 100))}


@pytest.mark.parametrize("op,into", FORMS)
def test_right_calls_launch(lib, op, into):
    host = Host(lib)
    assert call(host, op, into) == OK and host.launches()
    if op in WRITTEN:
        assert call(host, op, offsets=None, k=(F32, 3, 2, 64), v=(F32, 3, 2, 64)) == OK
    if op in ("read", "shared"):
        for kind in (BF16, F32):
            plain = {**PLAIN, "k_pages": (kind, 9, 2, 16, 64), "v_pages": (kind, 9, 2, 16, 64)}
            assert call(host, op, into, **plain) == OK and host.launches()
    if op == "shared":  # no groups, prefixes without pages
        assert call(host, op, into, prefixes=(I32, 0, 5), prefix_lens=(I32, 0), groups=(I32, 1)) == OK and host.launches()
        assert call(host, op, into, prefixes=(I32, 2, 0)) == OK and host.launches()
    if op == "logits":
        off = dict.fromkeys(LOGITS)
        assert call(host, op, into, **off) == OK and host.launches()
        on = dict(tokens=SHAPES[op]["tokens"], offsets=SHAPES[op]["offsets"])
        assert call(host, op, into, **{**off, **on}) == OK
        assert call(host, op, into, **{**off, **{x: SHAPES[op][x] for x in ("bias_words", "bias", "bias_offsets")}}) == OK
        assert call(host, op, into, **{**off, "mask": (I32, 5, 4)}) == OK
        assert call(host, op, into, **{**off, "mask": (I32, 0, 4), "mask_rows": (I32, 5)}) == OK
    # no rows: nothing to launch
    host.launches()
    assert call(host, op, into, **NONE[op]) == OK and not host.launches()


BAD_PAGES = [
    dict(k_pages=(U8, 9, 2, 16, 32)), dict(v_pages=(BF16, 9, 2, 16, 64)), dict(v_pages=(U8, 8, 2, 16, 64)),
    dict(k_pages=(U8, 18, 16, 64), v_pages=(U8, 18, 16, 64)), dict(PLAIN, k_scales=PAGES["k_scales"], v_scales=PAGES["v_scales"]),
    dict(k_scales=None), dict(v_scales=None), dict(k_scales=(F32, 9, 2, 8)), dict(v_scales=(BF16, 9, 2, 16)),
    dict(k_scales=(F32, 8, 2, 16), v_scales=(F32, 8, 2, 16)), dict(k_scales=(F32, 18, 16), v_scales=(F32, 18, 16)),
    dict(k_scales=(F32, 9, 2, 16, 1), v_scales=(F32, 9, 2, 16, 1)), dict(k_scales=None, v_scales=None),
    dict(k_pages=(I32, 9, 2, 16, 64), v_pages=(I32, 9, 2, 16, 64), k_scales=None, v_scales=None)]
BAD_ROWS = [
    dict(k=(F32, 7, 2, 32), v=(F32, 7, 2, 32)), dict(k=(F32, 7, 4, 64), v=(F32, 7, 4, 64)), dict(k=(F32, 7, 2, 64), v=(BF16, 7, 2, 64)),
    dict(k=(F32, 7, 2, 64), v=(F32, 6, 2, 64)), dict(k=(F32, 7, 128), v=(F32, 7, 128)), dict(k=(I32, 7, 2, 64), v=(I32, 7, 2, 64)),
    dict(table=(F32, 3, 4)), dict(table=(I32, 12)), dict(table=(I32, 4, 4)), dict(starts=(I32, 2)), dict(starts=(F32, 3)),
    dict(starts=(I32, 3, 1)), dict(offsets=(I32, 3)), dict(offsets=(F32, 4)), dict(offsets=None)]
BAD_DECODE = [
    dict(q=(F32, 3, 7, 64), out=(F32, 3, 7, 64)), dict(q=(F32, 3, 0, 64), out=(F32, 3, 0, 64)), dict(q=(I32, 3, 8, 64)),
    dict(q=(F32, 3, 512)), dict(q=(F32, 4, 8, 64)), dict(q=(F32, 3, 8, 128), out=(F32, 3, 8, 128)), dict(table=(I32, 4, 4)),
    dict(table=(U8, 3, 4)), dict(lens=(I32, 4)), dict(lens=(F32, 3)), dict(lens=(I32, 3, 1)), dict(out=(F32, 3, 8, 32)),
    dict(out=(I32, 3, 8, 64)), dict(out=(F32, 24, 64)), dict(scale=float("nan")), dict(scale=float("inf")), dict(scale=2.4e38)]
REFUSED = {
    "append": BAD_PAGES + BAD_ROWS, "read": BAD_PAGES + BAD_ROWS, "decode": BAD_PAGES + BAD_DECODE,
    "shared": BAD_PAGES + BAD_DECODE + [
        dict(prefixes=(F32, 2, 5)), dict(prefixes=(I32, 10)), dict(prefix_lens=(I32, 3)), dict(prefix_lens=(F32, 2)),
        dict(groups=(I32, 2)), dict(groups=(F32, 3)), dict(groups=(I32, 3, 1)), dict(prefixes=(I32, 3, 5))],
    "logits": [
        dict(logits=(F32, 500)), dict(logits=(I32, 5, 100)), dict(logits=(F32, 5, 0), out=(F32, 5, 0)), dict(logits=(BF16, 6, 100)),
        dict(tokens=None), dict(offsets=None), dict(tokens=None, offsets=None), dict(tokens=(F32, 40)), dict(tokens=(I32, 4, 10)),
        dict(offsets=(I32, 5)), dict(offsets=(F32, 6)), dict(prompts=(I32, 6)), dict(prompts=(F32, 5)), dict(repetition=(F32, 4)),
        dict(frequency=(BF16, 5)), dict(presence=(F32, 5, 1)), dict(bias_words=None), dict(bias=None), dict(bias_offsets=None),
        dict(bias_words=(I32, 8)), dict(bias=(BF16, 9)), dict(bias=(F32, 3, 3)), dict(bias_offsets=(I32, 5)), dict(mask=None),
        dict(mask=(F32, 3, 4)), dict(mask=(I32, 3, 3)), dict(mask=(I32, 12)), dict(mask_rows=None), dict(mask_rows=(I32, 4)),
        dict(mask_rows=(F32, 5)), dict(out=(F32, 5, 99)), dict(out=(I32, 5, 100)), dict(out=(F32, 500))],
}


@pytest.mark.parametrize("op", ENTRY)
def test_wrong_arguments_are_refused(lib, op):
    host = Host(lib)
    for change in REFUSED[op]:
        change = dict(change)
        assert call(host, op, **change) == INVALID, change
        if op in ALLOCATES and set(change) != {"out"}:
            change.pop("out", None)
            assert call(host, op, into=False, **change) == INVALID, change
        assert lib.host_message() and not host.launches(), change


@pytest.mark.parametrize("op", ENTRY)
def test_null_arguments_are_refused(lib, op):
    host = Host(lib)
    optional = set(LOGITS) if op == "logits" else {"offsets"} if op in WRITTEN else set()
    for name in SHAPES[op]:
        if name not in optional | {"scale"}:
            assert call(host, op, **{name: None}) == INVALID, name
            assert name == "out" or op in WRITTEN or call(host, op, into=False, **{name: None}) == INVALID, name
    assert call(host, op, rt=False) == INVALID
    if op in ALLOCATES:
        assert call(host, op, into=False, rt=False) == INVALID
        assert call(host, op, into=False, out_dtype=I32) == INVALID
    if op == "logits":
        assert call(host, op, options=False) == INVALID and call(host, op, into=False, options=False) == INVALID
    assert not host.launches()


@pytest.mark.parametrize("op", ENTRY)
def test_buffers_of_another_runtime_and_shared_memory_are_refused(lib, op):
    host, other = Host(lib), Host(lib)
    for name, x in SHAPES[op].items():
        if not isinstance(x, tuple):
            continue
        assert call(host, op, **{name: host.buf(*x, rt=other.rt)}) == INVALID, name
        assert name == "out" or op in WRITTEN or call(host, op, into=False, **{name: host.buf(*x, rt=other.rt)}) == INVALID
        for w in WRITTEN.get(op, ["out"]):
            if w == name:
                continue
            whole = SHAPES[op][w]
            size = ITEM[whole[0]]
            for d in whole[1:]:
                size *= d
            at = 1 << 45
            assert call(host, op, **{w: host.buf(*whole, at=at), name: host.buf(*x, at=at + size - 4)}) == INVALID, (w, name)
            assert not host.launches()
            assert call(host, op, **{w: host.buf(*whole, at=at), name: host.buf(*x, at=at + size)}) == OK, (w, name)
            host.launches()
    assert call(host, op) == OK
    if op in WRITTEN:
        for a, b in (("k_pages", "v_pages"), ("k_scales", "v_scales")) if op == "append" else (("k", "v"),):
            one = host.buf(*SHAPES[op][a])
            assert call(host, op, **{a: one, b: one}) == INVALID
    if op != "logits":  # what is only read may share memory
        a, b = ("k", "v") if op == "append" else ("k_pages", "v_pages")
        one = host.buf(*SHAPES[op][a])
        assert call(host, op, **{a: one, b: one}) == OK


def test_logits_in_place(lib):
    """The logits may be the output, of one type and address; not a part of them, nor of another type."""
    host = Host(lib)
    x = host.buf(BF16, 5, 100, at=1 << 45)
    assert call(host, "logits", logits=x, out=x) == OK
    assert call(host, "logits", logits=x, out=host.buf(BF16, 5, 100, at=1 << 45)) == OK
    host.launches()
    assert call(host, "logits", logits=x, out=host.buf(F32, 5, 100, at=1 << 45)) == INVALID
    assert call(host, "logits", logits=x, out=host.buf(BF16, 5, 100, at=(1 << 45) + 200)) == INVALID
    assert call(host, "logits", logits=x, out=host.buf(BF16, 5, 100, at=1 << 45, rt=Host(lib).rt)) == INVALID
    assert call(host, "logits", logits=x, out=x, mask=host.buf(I32, 3, 4, at=(1 << 45) + 4)) == INVALID
    assert not host.launches()


def test_sizes_past_the_kernels_are_refused(lib):
    host = Host(lib)

    def pages(p, hkv, ps, d):
        return dict(k_pages=(U8, p, hkv, ps, d), v_pages=(U8, p, hkv, ps, d), k_scales=(F32, p, hkv, ps), v_scales=(F32, p, hkv, ps))

    for op in ("decode", "shared"):
        b = 1 << 21
        for change in (dict(q=(F32, 3, 8, 513), **pages(9, 2, 16, 513), out=(F32, 3, 8, 513)), dict(table=(I32, 3, 1 << 27)),
                       pages(9, 2, 1 << 29, 64), pages(9, 2, 1 << 31, 64),
                       dict(q=(F32, b, 8, 64), table=(I32, b, 4), lens=(I32, b), out=(F32, b, 8, 64))):
            assert call(host, op, **change) == UNIMPLEMENTED, change
    assert call(host, "shared", prefixes=(I32, 2, 1 << 27)) == UNIMPLEMENTED
    for op in WRITTEN:
        assert call(host, op, table=(I32, 3, 1 << 28)) == UNIMPLEMENTED
        assert call(host, op, k=(F32, 1 << 25, 2, 64), v=(F32, 1 << 25, 2, 64)) == UNIMPLEMENTED
    assert call(host, "logits", logits=(BF16, 5, (1 << 24) + 1), mask=(I32, 3, (1 << 19) + 1), out=(F32, 5, (1 << 24) + 1)) == UNIMPLEMENTED
    assert call(host, "logits", tokens=(I32, 1 << 31)) == UNIMPLEMENTED
    assert call(host, "logits", bias=(F32, 1 << 31), bias_words=(I32, 1 << 31)) == UNIMPLEMENTED
    b = 1 << 23
    assert call(host, "logits", logits=(BF16, b, 2), **dict.fromkeys(LOGITS), out=(F32, b, 2)) == UNIMPLEMENTED
    assert not host.launches()
    assert call(host, "logits", logits=(BF16, 5, 1 << 24), mask=(I32, 3, 1 << 19), out=(F32, 5, 1 << 24)) == OK


KEYS = {(U8, 64): 64, (U8, 128): 64, (U8, 256): 32, (F32, 64): 16, (F32, 128): 16, (F32, 256): 16, (BF16, 64): 32,
        (BF16, 128): 32, (BF16, 256): 16}  # of a prefix's tile


def test_shared_plans(lib):
    """Launches of random shapes: known kernels in pairs that cover the batch, threads and LDS within the
    device's; plan, counters and records apart from each other within the runtime's block, that of
    captured calls for a captured call."""
    host, rng, seen, several = Host(lib), random.Random(5), set(), 0
    for _ in range(3000):
        d, kind, qt, ot = rng.choice([8, 64, 128, 256, 256, 512]), rng.choice([U8, BF16, F32]), rng.choice([BF16, F32]), rng.choice([BF16, F32])
        hkv, g = rng.choice([1, 2, 3, 8, 64, 300, 4097]), rng.choice([1, 2, 4, 5, 8, 16, 17, 40])
        b, ps, m = rng.choice([1, 2, 37, 700]), rng.choice([1, 16, 40, 64, 1024]), rng.choice([0, 1, 30, 2000])
        p, n, mp = rng.choice([0, 1, 50, 50]), rng.choice([0, 1, 3, 100]), rng.choice([0, 1, 9, 2000])
        captured, odd = rng.random() < 0.5, rng.choice([0, 0, 0, 0, 4, 8])
        lib.host_capturing(int(captured))
        hq, qa, oa, ta, la = hkv * g, (1 << 44) + odd * (rng.random() < 0.5), 1 << 50, 1 << 43, 1 << 42
        pages = {x: host.buf(kind, p, hkv, ps, d, at=((i + 1) << 46) + odd) for i, x in enumerate(("k_pages", "v_pages"))}
        scales = {x: (F32, p, hkv, ps) if kind == U8 else None for x in ("k_scales", "v_scales")}
        rc = call(host, "shared", q=host.buf(qt, b, hq, d, at=qa), **pages, **scales, prefixes=(I32, n, mp), prefix_lens=(I32, n),
                  groups=(I32, n + 1), table=host.buf(I32, b, m, at=ta), lens=host.buf(I32, b, at=la), out=host.buf(ot, b, hq, d, at=oa))
        assert rc == (OK if b * hq < 1 << 24 else UNIMPLEMENTED)
        if rc:
            continue
        got = host.launches()
        seen.add(got[0][0])
        if got[0][0] == "rxw8_shared_any":
            assert got == [("rxw8_shared_any", b * hq, 256, 0)]
            continue
        assert not odd and d in (64, 128, 256) and ps % 16 == 0 and p and n and mp
        high = "_high" if kind != F32 and F32 in (qt, ot) else ""
        name = "rxw8_shared_%s%s_d%d" % ({U8: "q8", F32: "f32", BF16: "bf16"}[kind], high, d)
        heads, rec, first, done = hkv * -(-g // 16), (d + 4) * 4, None, 0
        several += len(got) > 2
        for i in range(0, len(got), 2):
            x = (c.c_int64 * 16)()
            lib.host_shared(i, x)
            b0, nb, units, waves, columns, keys, counters, plan, part, parts, own, whole, q, out, table, lens = x
            assert got[i][:3] == (name, heads * units, 512) and got[i + 1] == ("rxw8_shared_join", -(-nb * hq // 4), 256, 0)
            assert 0 < got[i][3] <= (160 << 10) - 1024 and 1 <= units <= 256 and 1 <= waves <= 8
            assert b0 == done and nb > 0 and 4 * heads * units <= 64 << 10
            assert columns in (16, 32, 64) and keys == KEYS[kind, d]
            done += nb
            block = (2 if captured else 1) << 40
            assert counters == block and plan == block + (64 << 10) and part == plan + 1024
            record = -(-min(g, 16) * rec // 1024) * 1024
            assert parts == part + 2 * heads * units * record
            assert own >= parts + 2 * heads * units * columns * rec and whole >= own + nb * hq * rec
            assert whole + nb * hq * rec <= block + (64 << 10) + (16 << 20)
            size, osize = ITEM[qt] * hq * d, ITEM[ot] * hq * d
            assert (q, out, table, lens) == (qa + b0 * size, oa + b0 * osize, ta + 4 * b0 * m, la + 4 * b0)
            first = first or tuple(x)
            assert tuple(x)[2:12] == first[2:12]
        assert done == b
    lib.host_capturing(0)
    assert len(seen) == 16 and several > 20


def test_decode_plans(lib):
    host, rng, seen = Host(lib), random.Random(6), set()
    for _ in range(2000):
        d, qt, ot = rng.choice([8, 64, 128, 256, 512]), rng.choice([BF16, F32]), rng.choice([BF16, F32])
        hkv, g = rng.choice([1, 2, 3, 8, 64, 300, 4097]), rng.choice([1, 2, 4, 5, 8, 16, 17, 40])
        b, ps, m, p = rng.choice([1, 2, 37, 700]), rng.choice([1, 16, 40, 64, 1024]), rng.choice([0, 1, 30, 2000]), rng.choice([0, 1, 50])
        captured, odd = rng.random() < 0.5, rng.choice([0, 0, 0, 1, 8])
        lib.host_capturing(int(captured))
        pages = {x: host.buf(U8, p, hkv, ps, d, at=((i + 1) << 46) + odd) for i, x in enumerate(("k_pages", "v_pages"))}
        rc = call(host, "decode", q=(qt, b, hkv * g, d), **pages, k_scales=(F32, p, hkv, ps), v_scales=(F32, p, hkv, ps),
                  table=(I32, b, m), lens=(I32, b), out=(ot, b, hkv * g, d))
        assert rc == (OK if b * hkv * g < 1 << 24 else UNIMPLEMENTED)
        if rc:
            continue
        (name, grid, threads, lds), = host.launches()
        seen.add(name)
        if name == "rxw8_q8_decode_any":
            assert grid == b * hkv * g and threads == 256 and not lds
            continue
        assert not odd and d in (64, 128, 256) and ps % 16 == 0 and p
        assert name == "rxw8_q8_decode%s_d%d" % ("_high" if F32 in (qt, ot) else "", d) and threads == 512
        x = (c.c_int64 * 4)()
        lib.host_decode(0, x)
        units, waves, counters, part = x
        assert grid == hkv * -(-g // 16) * units and 1 <= units <= 256 and 1 <= waves <= 8 and 0 < lds <= (160 << 10) - 1024
        block = (2 if captured else 1) << 40
        assert counters == block and part == block + (64 << 10) and 4 * grid <= 64 << 10
        record = -(-min(g, 16) * (d + 4) * 4 // 1024) * 1024
        assert units == 1 or 2 * grid * record <= 16 << 20
    lib.host_capturing(0)
    assert len(seen) == 7


@pytest.mark.parametrize("op", WRITTEN)
def test_row_plans(lib, op):
    host, rng, seen = Host(lib), random.Random(7), set()
    for _ in range(1000):
        t, hkv, d = rng.choice([1, 7, 5000]), rng.choice([1, 3, 8, 64]), rng.choice([1, 8, 12, 64, 128, 512, 1000])
        odd, kt = rng.choice([0, 0, 4, 8]), rng.choice([BF16, F32])
        args = dict(k_pages=(U8, 9, hkv, 16, d), v_pages=(U8, 9, hkv, 16, d), k_scales=(F32, 9, hkv, 16), v_scales=(F32, 9, hkv, 16))
        assert call(host, op, **args, k=(kt, t, hkv, d), v=host.buf(kt, t, hkv, d, at=(1 << 45) + odd)) == OK
        (name, grid, threads, lds), = host.launches()
        any_ = odd != 0 or (d % 8 != 0 if op == "read" else d not in (64, 128, 256, 512))
        seen.add(name)
        assert name == "rxw8_q8_" + op + ("_any" if any_ else "") and threads == 256 and not lds
        assert grid == (-(-t * hkv // 4) if any_ else -(-t // 4) * -(-hkv * d // 8 // 128))
    assert len(seen) == 2


def test_logits_plans(lib):
    host, rng, seen = Host(lib), random.Random(8), set()
    for _ in range(1000):
        b, v, odd = rng.choice([1, 3, 64, 700]), rng.choice([1, 7, 8, 4095, 4096, 4104, 49152, 151936, 1 << 24]), rng.choice([0, 0, 2, 8])
        kind, out = rng.choice([BF16, F32]), rng.choice([BF16, F32])
        on = {x: None for x in LOGITS}
        history, bias = rng.random() < 0.5, rng.random() < 0.5
        on.update(dict(tokens=(I32, 9), offsets=(I32, b + 1), presence=(F32, b)) if history else {})
        on.update(dict(bias_words=(I32, 9), bias=(F32, 9), bias_offsets=(I32, b + 1)) if bias else {})
        assert call(host, "logits", logits=host.buf(kind, b, v, at=(1 << 45) + odd), **on, out=host.buf(out, b, v, at=1 << 50)) == OK
        (name, grid, threads, lds), = host.launches()
        seen.add(name)
        assert name == ("rxw8_logits_any" if v % 8 or odd else "rxw8_logits_adjust") and threads == 512
        x = (c.c_int64 * 2)()
        lib.host_logits(0, x)
        assert x[0] * (x[1] - 1) < v <= x[0] * x[1] and grid == b * x[1] and grid * threads < 1 << 32
        assert lds == 4 * x[0] * (history + bias) + 2048 * bias <= 64 << 10
    assert len(seen) == 2
