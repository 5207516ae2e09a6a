"""Penalties, biases and grammar masks on logits, on the GPU."""
import numpy as np
import pytest

import serving_more_ref as more
from test_gpu_serving import STEP, check, down, dt, floats, rx, up

pytestmark = pytest.mark.gpu

I32, F32 = np.int32, np.float32


def history(rng, rows, vocab, low, high, first=0, tail=0):
    counts = rng.integers(low, high + 1, rows)
    offsets = np.concatenate([[first], first + np.cumsum(counts)]).astype(I32)
    words = np.minimum((vocab * rng.random(offsets[-1] + tail) ** 4).astype(I32), vocab - 1)
    return dict(tokens=words, offsets=offsets, prompts=(counts * rng.random(rows)).astype(I32),
                repetition=(1 + rng.random(rows)).astype(F32), frequency=rng.random(rows).astype(F32),
                presence=rng.random(rows).astype(F32))


def biases(rng, rows, vocab, high):
    counts = rng.integers(0, high + 1, rows)
    offsets = np.concatenate([[0], np.cumsum(counts)]).astype(I32)
    return dict(bias_words=rng.integers(0, vocab, offsets[-1]).astype(I32),
                bias=(5 * rng.standard_normal(offsets[-1])).astype(F32), bias_offsets=offsets)


def masks(rng, masks, vocab, share=0.5):
    bits = rng.random((masks, -(-vocab // 32) * 32)) < share
    return np.packbits(bits, axis=1, bitorder="little").view(np.uint32).view(I32)


def adjust(rt, z, kind, out=None, into=None, **options):
    bufs = {k: rt.buffer(v) for k, v in options.items()}
    zb = up(rt, z, kind)
    if into == "logits":
        assert rx().adjust_logits(rt, zb, out=zb, **bufs) is zb
        return down(zb)
    if into:
        o = rt.zeros(z.shape, dt(out))
        assert rx().adjust_logits(rt, zb, out=o, **bufs) is o
        return down(o)
    o = rx().adjust_logits(rt, zb, out_dtype=None if out is None else dt(out), **bufs)
    assert out is not None or o.dtype == dt(kind)
    return down(o)


@pytest.mark.parametrize("vocab", [1, 31, 32, 33, 999, 8192, 8193, 50000, 151936])
@pytest.mark.parametrize("kind,out", [("f32", None), ("bf16", None), ("f32", "bf16"), ("bf16", "f32")])
def test_adjust(rt, vocab, kind, out):
    """All settings at once, at vocabularies around a mask's word and a workgroup's chunk."""
    rng = np.random.default_rng(vocab)
    rows = 5
    z = floats(rng, (rows, vocab), kind, std=4.0)
    o = {**history(rng, rows, vocab, 0, 300), **biases(rng, rows, vocab, 20), "mask": masks(rng, 3, vocab),
         "mask_rows": np.array([0, -1, 2, 1, 3], I32)}
    y = adjust(rt, z, kind, out, into=out is not None, **o)
    check(y, *more.adjust(z, STEP[out or kind], **o))


@pytest.mark.parametrize("names", [("tokens", "offsets"), ("tokens", "offsets", "repetition"), ("tokens", "offsets", "frequency", "prompts"),
                                   ("tokens", "offsets", "presence"), ("bias_words", "bias", "bias_offsets"), ("mask",),
                                   ("mask", "mask_rows"), ()])
def test_settings_by_themselves(rt, names):
    rng = np.random.default_rng(len(names))
    rows, vocab = 4, 3001
    z = floats(rng, (rows, vocab), "f32", std=4.0)
    o = {**history(rng, rows, vocab, 1, 100), **biases(rng, rows, vocab, 9), "mask": masks(rng, rows, vocab),
         "mask_rows": np.array([3, 0, -1, 1], I32)}
    o = {k: o[k] for k in names}
    y = adjust(rt, z, "f32", **o)
    check(y, *more.adjust(z, STEP["f32"], **o))
    if names in ((), ("tokens", "offsets")):
        np.testing.assert_array_equal(y, z)


def test_in_place(rt):
    rng = np.random.default_rng(7)
    for kind in ("f32", "bf16"):
        z = floats(rng, (3, 20001), kind, std=4.0)
        o = {**history(rng, 3, 20001, 0, 4000), **biases(rng, 3, 20001, 50), "mask": masks(rng, 3, 20001, 0.9)}
        y = adjust(rt, z, kind, into="logits", **o)
        check(y, *more.adjust(z, STEP[kind], **o))


def test_words_and_offsets_out_of_range(rt):
    """Tokens and biased words outside the vocabulary, offsets outside the lists and rows of a history
    that others do not own, prompts longer than their rows and below 0."""
    rng = np.random.default_rng(8)
    z = floats(rng, (4, 100), "f32", std=4.0)
    o = {**history(rng, 4, 100, 30, 60, first=3, tail=2), **biases(rng, 4, 100, 30)}
    o["tokens"][::5] = np.resize(np.array([-1, 100, 2 ** 31 - 1, -2 ** 31], I32), o["tokens"][::5].size)
    o["bias_words"][::3] = np.resize(np.array([-1, 100, 2 ** 31 - 1], I32), o["bias_words"][::3].size)
    o["prompts"] = np.array([2 ** 31 - 1, -5, 0, 7], I32)
    check(adjust(rt, z, "f32", **o), *more.adjust(z, STEP["f32"], **o))
    o["offsets"] = np.array([-9, 5, 5, 50, 2 ** 31 - 1], I32)
    o["bias_offsets"] = np.array([-3, 2, 2, 9, 2 ** 31 - 1], I32)
    check(adjust(rt, z, "f32", **o), *more.adjust(z, STEP["f32"], **o))


def test_one_word_many_times(rt):
    """A history of one word alone, and its biases: the count is exact, the last entry counts."""
    z = np.full((2, 70), 10.0, F32)
    n = 100000
    o = dict(tokens=np.full(2 * n, 69, I32), offsets=np.array([0, n, 2 * n], I32), prompts=np.array([0, n - 1], I32),
             frequency=np.array([0.25, 0.25], F32), presence=np.array([1, 1], F32),
             bias_words=np.full(40, 69, I32), bias=np.arange(40, dtype=F32), bias_offsets=np.array([0, 40, 40], I32))
    y = adjust(rt, z, "f32", **o)
    assert y[0, 69] == 10 - 0.25 * n - 1 + 39 and y[1, 69] == 10 - 0.25 - 1
    assert (np.delete(y, 69, axis=1) == 10).all()


def test_special_values(rt):
    """NaN and infinities among the logits: a masked one is -inf, an allowed one stays; penalties that are
    off; infinite biases."""
    z = np.array([[np.nan, np.inf, -np.inf, 3, -3, 0, 2, 1]], F32).repeat(3, axis=0)
    o = dict(tokens=np.arange(8, dtype=I32), offsets=np.array([0, 8, 8, 8], I32), prompts=np.array([8, 0, 0], I32),
             repetition=np.array([2, np.nan, -1], F32), mask=np.array([[0b01111110], [0b11111111], [0b11110110]], I32),
             bias_words=np.array([6, 7, 6], I32), bias=np.array([-np.inf, 1, np.inf], F32), bias_offsets=np.array([0, 0, 2, 3], I32))
    y = adjust(rt, z, "f32", **o)
    inf, nan = np.inf, np.nan
    np.testing.assert_array_equal(y, np.array([[-inf, inf, -inf, 1.5, -6, 0, 1, -inf], [nan, inf, -inf, 3, -3, 0, -inf, 2],
                                               [-inf, inf, -inf, -inf, -3, 0, inf, 1]], F32))
    o["repetition"] = np.array([0, np.nan, -1], F32)  # off everywhere
    assert adjust(rt, z, "f32", **o)[0, 3:7].tolist() == [3, -3, 0, 2]


@pytest.mark.parametrize("rows,vocab,high", [(1, 248320, 20000), (64, 3000, 2000), (300, 700, 5), (1, 1 << 20, 3)])
def test_sizes(rt, rows, vocab, high):
    rng = np.random.default_rng(rows)
    z = floats(rng, (rows, vocab), "f32", std=4.0)
    o = {**history(rng, rows, vocab, 0, high), **biases(rng, rows, vocab, 5)}
    check(adjust(rt, z, "f32", **o), *more.adjust(z, STEP["f32"], **o))


def test_before_sampling(rt):
    """Greedy sampling of adjusted logits: banned and repeated words do not come again."""
    r = rx()
    z = np.zeros((2, 5000), F32)
    z[:, 100], z[:, 200], z[:, 300] = 9, 8, 7
    o = dict(tokens=np.array([100, 100, 200], I32), offsets=np.array([0, 2, 3], I32), frequency=np.array([1, 1], F32),
             bias_words=np.array([200], I32), bias=np.array([-np.inf], F32), bias_offsets=np.array([0, 1, 1], I32))
    y = r.adjust_logits(rt, rt.buffer(z), **{k: rt.buffer(v) for k, v in o.items()})
    zero = rt.buffer(np.zeros(2, F32))
    assert r.sample(rt, y, zero, zero).to_numpy().tolist() == [100, 100]
    o["frequency"] = np.array([1.5, 0], F32)
    o["tokens"][2] = 100
    y = r.adjust_logits(rt, rt.buffer(z), **{k: rt.buffer(v) for k, v in o.items()})
    assert r.sample(rt, y, zero, zero).to_numpy().tolist() == [300, 100]
