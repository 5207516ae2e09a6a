"""What the serving operators of a cache in 8 bits and of shared prefixes are timed
and checked on: rows written into 8-bit pages and read back, attention of one new
token per sequence over such pages, the same for sequences that share a prefix, and
the logits' penalties, biases and grammar masks ahead of sampling.

A case is a dict of plain values; ``prepare`` makes what a serving loop has in
hand before the call, ``run`` makes one pass and returns its outputs whole:
through the framework's entry points where ``own`` is true, else in a plain
form of elementary torch operations. ``exact`` gives the same outputs in 64
bits, ``work`` the bytes and operations that a pass cannot do without.

8-bit pages hold a row x of a kv head as codes (int8 + 128) and one f32 scale:
s = max(amax |x|, 1e-12) / 127, code = clamp(round(x / s), -127, 127) + 128, the
quotient in f32; it stands for (code - 128) s.
"""
import math
import random

import numpy as np
import torch

own = False

DEV = "cuda"
_FLOAT = {"bf16": torch.bfloat16, "f32": torch.float32}
_SIZE = {"bf16": 2, "f32": 4, "q8": 1}

# (query heads, kv heads): the dense decoder's, the hybrid model's, and from one
# query head per kv head to eight
HEADS = [(16, 8), (8, 2), (8, 8), (32, 8), (32, 4), (64, 8)]
# the vocabularies of the dense decoder and of the hybrid model
VOCABS = [151936, 248320]


def listed():
    return [
        # one new key and value for each user of a batch, and what the cache then holds of them
        dict(name="write8-step", kind="write", batch=96, kv_heads=8, dim=128, page=16, rows_low=1,
             rows_high=1, start_low=0, start_high=1500, new="f32", back="f32", whole=False),
        # prompts admitted in chunks: the chunk into its pages, then the whole context back as
        # rows for the packed attention
        dict(name="write8-chunk", kind="write", batch=12, kv_heads=8, dim=128, page=64,
             rows_low=64, rows_high=2000, start_low=0, start_high=1000, new="bf16", back="bf16",
             whole=True),
        # one user's next token over a short context: latency counts
        dict(name="decode8-step", kind="decode", batch=1, q_heads=16, kv_heads=8, dim=128, page=16,
             low=777, high=777, q="bf16"),
        # a batch of long contexts of ragged lengths
        dict(name="decode8-long", kind="decode", batch=8, q_heads=32, kv_heads=8, dim=128, page=64,
             low=512, high=8192, q="bf16"),
        # many users, from a first token on, f32 queries as the f32 projections give them
        dict(name="decode8-many", kind="decode", batch=96, q_heads=16, kv_heads=8, dim=128,
             page=16, low=1, high=1500, q="f32"),
        # a few users behind one system prompt: latency counts
        dict(name="shared-few", kind="shared", prefixes=1, prefix_low=1000, prefix_high=1000,
             batch=4, q_heads=16, kv_heads=8, dim=128, page=16, low=1, high=60, cache="bf16",
             q="bf16"),
        # one long document, many questions about it
        dict(name="shared-chat", kind="shared", prefixes=1, prefix_low=6000, prefix_high=6000,
             batch=64, q_heads=32, kv_heads=8, dim=128, page=64, low=64, high=1000, cache="bf16",
             q="bf16"),
        # three applications with a prompt of their own, f32 queries
        dict(name="shared-groups", kind="shared", prefixes=3, prefix_low=700, prefix_high=4000,
             batch=96, q_heads=16, kv_heads=8, dim=128, page=16, low=1, high=300, cache="bf16",
             q="f32"),
        # samples of one long context, over 8-bit pages, eight query heads to a kv head
        dict(name="shared-8bit", kind="shared", prefixes=1, prefix_low=8192, prefix_high=8192,
             batch=48, q_heads=32, kv_heads=4, dim=128, page=64, low=16, high=800, cache="q8",
             q="bf16"),
        # one user's next token: penalties over a chat's history
        dict(name="logits-step", kind="logits", rows=1, vocab=151936, logits="f32", low=800,
             high=800, biases=0, masks=0),
        # a batch of users with settings of their own, a third of them under a grammar
        dict(name="logits-batch", kind="logits", rows=64, vocab=248320, logits="f32", low=1,
             high=8000, biases=300, masks=5),
        # bf16 logits, every user under a grammar
        dict(name="logits-bf16", kind="logits", rows=16, vocab=151936, logits="bf16", low=100,
             high=3000, biases=20, masks=16),
    ]


def _log(rng, low, high):
    """A whole number between low and high, spread over its logarithm."""
    return max(low, min(high, round(math.exp(rng.uniform(math.log(low), math.log(high))))))


def draw(rng):
    kind = rng.choice(["write", "write", "decode", "decode", "decode", "shared", "shared",
                       "shared", "logits", "logits"])
    hq, hkv = rng.choice(HEADS)
    dim = rng.choice([64, 128, 128, 256])
    page = rng.choice([16, 16, 32, 48, 64, 128, 256])
    if kind == "write":
        high = rng.choice([1, _log(rng, 1, 2000)])
        start = _log(rng, 1, 2000)
        most = max(1, min(256, 12000 * 8 * 128 // ((high + start) * hkv * dim)))
        return dict(kind="write", batch=_log(rng, 1, most), kv_heads=hkv, dim=dim, page=page,
                    rows_low=max(1, high // rng.choice([1, 4, 2000])), rows_high=high, start_low=0,
                    start_high=start, new=rng.choice(["bf16", "f32"]),
                    back=rng.choice(["bf16", "f32"]), whole=rng.choice([True, False]))
    if kind == "decode":
        high = _log(rng, 1, 8192)
        # at most the listed long caches' bytes
        most = max(1, min(256, 8 * 4352 * 8 * 128 // (high * hkv * dim)))
        return dict(kind="decode", batch=_log(rng, 1, most), q_heads=hq, kv_heads=hkv, dim=dim,
                    page=page, low=max(1, high // rng.choice([1, 4, 16, 8192])), high=high,
                    q=rng.choice(["bf16", "f32"]))
    if kind == "shared":
        cache = rng.choice(["bf16", "bf16", "q8", "q8", "f32"])
        prefixes, prefix, high = rng.choice([1, 1, 2, 4]), _log(rng, 1, 8192), _log(rng, 1, 1000)
        # at most the listed cases' operations, and the bytes of their own keys
        most = min(256, 48 * 32 * 128 * 8192 // ((prefix + high) * hq * dim),
                   64 * 500 * 8 * 128 * 2 // (high * hkv * dim * _SIZE[cache]))
        prefixes = min(prefixes, max(1, most))
        return dict(kind="shared", prefixes=prefixes,
                    prefix_low=max(1, prefix // rng.choice([1, 4])), prefix_high=prefix,
                    batch=_log(rng, prefixes, max(prefixes, most)), q_heads=hq, kv_heads=hkv,
                    dim=dim, page=page, low=max(1, high // rng.choice([1, 4, 1000])), high=high,
                    cache=cache, q=rng.choice(["bf16", "f32"]))
    rows, vocab = _log(rng, 1, 64), rng.choice(VOCABS + [_log(rng, 1000, 248320)])
    high = _log(rng, 1, 8000)
    return dict(kind="logits", rows=rows, vocab=vocab, logits=rng.choice(["f32", "f32", "bf16"]),
                low=max(1, high // rng.choice([1, 8, 8000])), high=high,
                biases=rng.choice([0, 1, 20, 300]), masks=rng.choice([0, 1, min(rows, 7)]))


# ---- inputs ---------------------------------------------------------------------

def _spread(count, low, high, salt):
    """`count` whole numbers from low to high, the largest among them: of the case alone."""
    r = random.Random(1000003 * count + 1009 * low + high + salt)
    got = [high] + [low] * (count > 1)
    got += [_log(r, max(1, low), max(1, high)) if i % 2 else r.randint(low, high)
            for i in range(count - 2)]
    r.shuffle(got)
    return got


def _gen(seed):
    g = torch.Generator(device=DEV)
    g.manual_seed(seed)
    return g


def _normal(g, *shape, std=1.0):
    return torch.randn(*shape, generator=g, device=DEV) * std


def _int(values):
    return torch.tensor(values, dtype=torch.int32, device=DEV)


def _offsets(counts):
    at = [0]
    for n in counts:
        at.append(at[-1] + n)
    return at


def _encode(x):
    """Rows [..., D] f32 as codes and scales."""
    top = x.abs().amax(dim=-1).clamp_min(1e-12)
    scale = top / torch.full_like(top, 127.0)  # (a number here would be multiplied by its inverse)
    code = (x / scale[..., None]).round().clamp_(-127, 127) + 128
    return code.to(torch.uint8), scale


def _decode(codes, scale):
    return (codes.float() - 128.0) * scale[..., None]


def _pages(g, lens, page, hkv, d, cache):
    """A pool of key and value pages with old contents, and for each entry of `lens`
    the pages of that many positions, in no order."""
    need = [-(-n // page) for n in lens]
    pool = sum(need) + 3
    order = torch.randperm(pool, generator=g, device=DEV).to(torch.int32)
    got, at = {}, 0
    for kv in ("k", "v"):
        x = _normal(g, pool, hkv, page, d)
        if cache == "q8":
            got[kv + "_pages"], got[kv + "_scales"] = _encode(x)
        else:
            got[kv + "_pages"] = x.to(_FLOAT[cache])
    ids = []
    for n in need:
        ids.append(order[at:at + n])
        at += n
    return got, ids


def _table(ids, entries):
    """The page tables [len(ids), entries]; -1 where a sequence has none."""
    table = torch.full((len(ids), max(1, entries)), -1, dtype=torch.int32, device=DEV)
    for b, pages in enumerate(ids):
        table[b, :pages.numel()] = pages
    return table


def _write_inputs(case, seed):
    g, page, hkv, d = _gen(seed), case["page"], case["kv_heads"], case["dim"]
    counts = _spread(case["batch"], case["rows_low"], case["rows_high"], 3)
    starts = _spread(case["batch"], case["start_low"], case["start_high"], 4)
    ends = [s + n for s, n in zip(starts, counts)]
    state, ids = _pages(g, ends, page, hkv, d, "q8")
    state["table"] = _table(ids, -(-max(ends) // page))
    offsets = _offsets(counts)
    for kv in ("k", "v"):
        state[kv] = _normal(g, offsets[-1], hkv, d).to(_FLOAT[case["new"]])
    state.update(starts=_int(starts), offsets=_int(offsets))
    if case["whole"]:
        offsets, starts = _offsets(ends), [0] * len(ends)
    state.update(read_starts=_int(starts), read_offsets=_int(offsets))
    for kv in ("k", "v"):
        state[kv + "_back"] = torch.zeros(offsets[-1], hkv, d, dtype=_FLOAT[case["back"]],
                                          device=DEV)
    return state


def _decode_inputs(case, seed):
    g, page = _gen(seed), case["page"]
    lens = _spread(case["batch"], case["low"], case["high"], 1)
    state, ids = _pages(g, lens, page, case["kv_heads"], case["dim"], "q8")
    q = _normal(g, case["batch"], case["q_heads"], case["dim"]).to(_FLOAT[case["q"]])
    state.update(q=q, y=torch.zeros_like(q), table=_table(ids, -(-case["high"] // page)),
                 lens=_int(lens))
    return state


def _shares(case):
    """How many sequences each prefix has: all have one at least."""
    n, b = case["prefixes"], case["batch"]
    got = [b // (2 * n)] * n
    got[n // 2] += b - sum(got)
    if b // (2 * n) == 0:
        got = [b // n + (i < b % n) for i in range(n)]
    return got


def _shared_inputs(case, seed):
    g, page = _gen(seed), case["page"]
    prefix = _spread(case["prefixes"], case["prefix_low"], case["prefix_high"], 5)
    lens = _spread(case["batch"], case["low"], case["high"], 6)
    state, ids = _pages(g, prefix + lens, page, case["kv_heads"], case["dim"], case["cache"])
    q = _normal(g, case["batch"], case["q_heads"], case["dim"]).to(_FLOAT[case["q"]])
    state.update(q=q, y=torch.zeros_like(q), groups=_int(_offsets(_shares(case))),
                 prefixes=_table(ids[:len(prefix)], -(-case["prefix_high"] // page)),
                 prefix_lens=_int(prefix),
                 table=_table(ids[len(prefix):], -(-case["high"] // page)), lens=_int(lens),
                 most=max(_shares(case)))
    return state


def _logits_inputs(case, seed):
    g, rows, vocab = _gen(seed), case["rows"], case["vocab"]
    rank = torch.rand(rows, vocab, generator=g, device=DEV).mul_(vocab).add_(1)
    logits = 12.0 - 2.0 * rank.log_() + _normal(g, rows, vocab, std=0.5)
    counts = _spread(rows, case["low"], case["high"], 7)
    total = sum(counts)
    # a text repeats its frequent words many times over
    words = torch.rand(total, generator=g, device=DEV).mul_(math.log(vocab)).exp_().long() - 1
    words = (words * 7919 % vocab).to(torch.int32)
    draw_ = torch.rand(5, rows, generator=g, device=DEV)
    n = _int(counts)
    state = dict(logits=logits.to(_FLOAT[case["logits"]]), tokens=words,
                 offsets=_int(_offsets(counts)), prompts=(n * draw_[0]).to(torch.int32),
                 repetition=1 + 0.4 * draw_[1], frequency=0.5 * draw_[2],
                 presence=0.8 * draw_[3])
    state["repetition"][draw_[4] < 0.2] = 1.0  # switched off by some users
    if case["biases"]:
        r = random.Random(seed)
        each = [r.randint(0, case["biases"]) for _ in range(rows)]
        each[-1] = case["biases"]
        state["bias_words"] = torch.randint(vocab, (sum(each),), generator=g, device=DEV,
                                            dtype=torch.int32)
        state["bias"] = _normal(g, sum(each), std=5.0)
        state["bias_offsets"] = _int(_offsets(each))
    if case["masks"]:
        # the words that a grammar's states allow, a few of them or almost all; and the state
        # that each user is in (-1: no grammar)
        words_of = -(-vocab // 32)
        few = torch.rand(case["masks"], words_of, 32, generator=g, device=DEV)
        share = 0.001 + 0.998 * (torch.arange(case["masks"], device=DEV) % 2)[:, None, None]
        bits = (few < share).long() << torch.arange(32, device=DEV)
        state["mask"] = bits.sum(dim=2).to(torch.int32)
        pick = torch.arange(rows, device=DEV, dtype=torch.int32)
        state["mask_rows"] = torch.where((pick % 3 == 0) | (case["masks"] >= rows),
                                         pick % case["masks"], -1).to(torch.int32)
    state["y"] = torch.zeros_like(state["logits"])
    return state


_INPUTS = {"write": _write_inputs, "decode": _decode_inputs, "shared": _shared_inputs,
           "logits": _logits_inputs}

_rt = None


def _runtime():
    global _rt
    if _rt is None:
        import rxla_amd as rx
        _rt = rx.Runtime(0)
    return _rt


def prepare(case, seed):
    state = _INPUTS[case["kind"]](case, seed)
    if own:  # the handles of these tensors, which a serving loop makes once
        wrap = _runtime().wrap_tensor
        state["handles"] = {k: wrap(t) for k, t in state.items() if isinstance(t, torch.Tensor)}
    state["kind"] = case["kind"]
    torch.cuda.synchronize()
    return state


# ---- one pass -------------------------------------------------------------------

def run(state):
    if own:
        return _run_own(state)
    return _PLAIN[state["kind"]](state)


def _run_own(state):
    import rxla_amd as rx
    rt, h, kind = _runtime(), state["handles"], state["kind"]
    if kind == "write":
        rx.paged_kv_append_q8(rt, h["k_pages"], h["v_pages"], h["k_scales"], h["v_scales"], h["k"],
                              h["v"], h["table"], h["starts"], h["offsets"])
        rx.paged_kv_read(rt, h["k_pages"], h["v_pages"], h["table"], h["read_starts"],
                         h["read_offsets"], h["k_back"], h["v_back"], k_scales=h["k_scales"],
                         v_scales=h["v_scales"])
        return state["k_back"], state["v_back"]
    if kind == "decode":
        rx.grouped_query_attention_paged_q8(rt, h["q"], h["k_pages"], h["v_pages"], h["k_scales"],
                                            h["v_scales"], h["table"], h["lens"], out=h["y"])
        return state["y"]
    if kind == "shared":
        rx.grouped_query_attention_shared(rt, h["q"], h["k_pages"], h["v_pages"], h["prefixes"],
                                          h["prefix_lens"], h["groups"], h["table"], h["lens"],
                                          k_scales=h.get("k_scales"), v_scales=h.get("v_scales"),
                                          out=h["y"])
        return state["y"]
    rx.adjust_logits(rt, h["logits"], tokens=h["tokens"], offsets=h["offsets"],
                     prompts=h["prompts"], repetition=h["repetition"], frequency=h["frequency"],
                     presence=h["presence"], bias_words=h.get("bias_words"), bias=h.get("bias"),
                     bias_offsets=h.get("bias_offsets"), mask=h.get("mask"),
                     mask_rows=h.get("mask_rows"), out=h["y"])
    return state["y"]


def _rows_of(offsets, starts, total):
    """Sequence and position of each of `total` packed rows."""
    row, at = torch.arange(total, device=DEV), offsets.long()
    seq = torch.bucketize(row, at[1:], right=True)
    return seq, starts.long()[seq] + row - at[seq]


def _plain_write(s):
    page = s["k_pages"].shape[2]
    seq, pos = _rows_of(s["offsets"], s["starts"], s["k"].shape[0])
    to = s["table"].long()[seq, pos // page]
    (kc, ks), (vc, vs) = _encode(s["k"].float()), _encode(s["v"].float())
    s["k_pages"][to, :, pos % page], s["k_scales"][to, :, pos % page] = kc, ks
    s["v_pages"][to, :, pos % page], s["v_scales"][to, :, pos % page] = vc, vs
    seq, pos = _rows_of(s["read_offsets"], s["read_starts"], s["k_back"].shape[0])
    of = s["table"].long()[seq, pos // page]
    k = _decode(s["k_pages"][of, :, pos % page], s["k_scales"][of, :, pos % page])
    v = _decode(s["v_pages"][of, :, pos % page], s["v_scales"][of, :, pos % page])
    return k.to(s["k_back"].dtype), v.to(s["v_back"].dtype)


def _take(s, kv, table):
    """Keys or values [tables, kv heads, positions, D] f32 of the tables' pages."""
    ids, pages = table.long().clamp_min(0), s[kv + "_pages"]
    x = _decode(pages[ids], s[kv + "_scales"][ids]) if kv + "_scales" in s else pages[ids].float()
    n, m, hkv, page, d = x.shape
    return x.transpose(1, 2).reshape(n, hkv, m * page, d)


def _partial(q, k, v, lens):
    """Of q [n, kv heads, rows, D] over the first `lens` [n] keys: the rows' maximum,
    their sum of weights and the weighted values."""
    s = torch.matmul(q, k.transpose(-1, -2).contiguous()).mul_(1 / math.sqrt(q.shape[-1]))
    seen = torch.arange(k.shape[2], device=DEV)[None, :] < lens[:, None]
    s.masked_fill_(~seen[:, None, None, :], -math.inf)
    top = s.amax(dim=-1, keepdim=True).clamp_min(torch.finfo(s.dtype).min)
    p = s.sub_(top).exp_()
    return top, p.sum(dim=-1, keepdim=True), torch.matmul(p, v)


def _plain_decode(s):
    b, hq, d = s["q"].shape
    hkv = s["k_pages"].shape[1]
    q = s["q"].float().reshape(b, hkv, hq // hkv, d)
    _, mass, o = _partial(q, _take(s, "k", s["table"]), _take(s, "v", s["table"]), s["lens"])
    return o.div_(mass).reshape(b, hq, d).to(s["q"].dtype)


def _plain_shared(s):
    (b, hq, d), hkv, n = s["q"].shape, s["k_pages"].shape[1], s["prefix_lens"].numel()
    q, at, most = s["q"].float().reshape(b, hkv, hq // hkv, d), s["groups"].long(), s["most"]
    group, place = _rows_of(at, torch.zeros_like(at[1:]), b)
    # a prefix's sequences beside one another, up to the largest group's number
    qs = torch.zeros(n, hkv, most, hq // hkv, d, device=DEV)
    qs[group, :, place] = q
    first = _partial(qs.reshape(n, hkv, -1, d), _take(s, "k", s["prefixes"]),
                     _take(s, "v", s["prefixes"]), s["prefix_lens"])
    m1, l1, o1 = (x.reshape(n, hkv, most, hq // hkv, -1)[group, :, place] for x in first)
    m2, l2, o2 = _partial(q, _take(s, "k", s["table"]), _take(s, "v", s["table"]), s["lens"])
    m = torch.maximum(m1, m2)
    w1, w2 = (m1 - m).exp(), (m2 - m).exp()
    o = (o1 * w1 + o2 * w2) / (l1 * w1 + l2 * w2)
    return o.reshape(b, hq, d).to(s["q"].dtype)


def _plain_logits(s):
    z = s["logits"].float()
    rows, vocab = z.shape
    seq, place = _rows_of(s["offsets"], torch.zeros_like(s["prompts"]), s["tokens"].numel())
    at, one = seq * vocab + s["tokens"], torch.ones_like(s["tokens"])
    seen, count = (torch.zeros(rows * vocab, dtype=torch.int32, device=DEV) for _ in range(2))
    seen = seen.index_put_((at,), one).reshape(rows, vocab) > 0
    mine = (place >= s["prompts"].long()[seq]).to(torch.int32)
    count = count.index_put_((at,), mine, accumulate=True).reshape(rows, vocab)
    r, f, p = (s[k][:, None] for k in ("repetition", "frequency", "presence"))
    z = torch.where(seen, torch.where(z > 0, z / r, z * r), z)
    z = z - f * count - p * (count > 0)
    if "bias" in s:
        seq, _ = _rows_of(s["bias_offsets"], torch.zeros_like(s["prompts"]), s["bias"].numel())
        entry = torch.arange(1, seq.numel() + 1, device=DEV)
        last = torch.zeros(rows * vocab, dtype=torch.int64, device=DEV)
        last.scatter_reduce_(0, seq * vocab + s["bias_words"], entry, "amax")
        z = z + torch.nn.functional.pad(s["bias"], (1, 0))[last].reshape(rows, vocab)
    if "mask" in s:
        bits = s["mask"][s["mask_rows"].long().clamp_min(0)]
        bits = bits[:, :, None] >> torch.arange(32, device=DEV, dtype=torch.int32) & 1
        allowed = bits.reshape(rows, -1)[:, :vocab] > 0
        z = z.masked_fill(~allowed & (s["mask_rows"] >= 0)[:, None], -math.inf)
    return z.to(s["logits"].dtype)


_PLAIN = {"write": _plain_write, "decode": _plain_decode, "shared": _plain_shared,
          "logits": _plain_logits}


# ---- the same in 64 bits ----------------------------------------------------------

def _stands_for(codes, scales):
    return (codes.double() - 128) * scales.double().unsqueeze(-1)


def _positions(x, ids, n, kv, h):
    """Keys or values [n, D] of a kv head, of the first n positions of the pages `ids`."""
    pages = x[kv + "_pages"][ids.long(), h]
    got = (_stands_for(pages, x[kv + "_scales"][ids.long(), h]) if kv + "_scales" in x
           else pages.double())
    return got.reshape(-1, got.shape[-1])[:n]


def _softmax_rows(scores):
    e = torch.exp(scores - scores.max(dim=-1, keepdim=True).values)
    return e / e.sum(dim=-1, keepdim=True)


def exact(case, seed):
    x = _INPUTS[case["kind"]](case, seed)
    page = case.get("page")
    if case["kind"] == "write":
        got = []
        for kv in ("k", "v"):
            pool = _stands_for(x[kv + "_pages"], x[kv + "_scales"])
            at = x["offsets"].tolist()
            for b, start in enumerate(x["starts"].tolist()):
                rows = x[kv][at[b]:at[b + 1]].double()
                amax = rows.abs().max(dim=-1, keepdim=True).values.clamp_min(
                    float(np.float32(1e-12)))
                scale = (amax / 127).float().double()  # (53 bits rounded to 24: f32's own quotient)
                code = torch.round((rows / scale).float()).double().clamp(-127, 127)
                pos = torch.arange(start, start + rows.shape[0], device=DEV)
                pool[x["table"][b].long()[pos // page], :, pos % page] = code * scale
            back = torch.zeros(x[kv + "_back"].shape, dtype=torch.float64, device=DEV)
            at = x["read_offsets"].tolist()
            for b, start in enumerate(x["read_starts"].tolist()):
                pos = torch.arange(start, start + at[b + 1] - at[b], device=DEV)
                back[at[b]:at[b + 1]] = pool[x["table"][b].long()[pos // page], :, pos % page]
            got.append(back)
        return tuple(got)
    if case["kind"] in ("decode", "shared"):
        q, g = x["q"].double(), case["q_heads"] // case["kv_heads"]
        y, lens = torch.zeros_like(q), x["lens"].tolist()
        groups = x["groups"].tolist() if case["kind"] == "shared" else []
        for h in range(case["kv_heads"]):
            before = [[_positions(x, x["prefixes"][i, :-(-n // page)], n, kv, h)
                       for kv in ("k", "v")]
                      for i, n in enumerate(x["prefix_lens"].tolist())] if groups else []
            for b, n in enumerate(lens):
                k, v = (_positions(x, x["table"][b, :-(-n // page)], n, kv, h)
                        for kv in ("k", "v"))
                for i, (pk, pv) in enumerate(before):
                    if groups[i] <= b < groups[i + 1]:
                        k, v = torch.cat([pk, k]), torch.cat([pv, v])
                mine = slice(h * g, h * g + g)
                y[b, mine] = _softmax_rows(q[b, mine] @ k.T / math.sqrt(case["dim"])) @ v
        return y
    y = x["logits"].double().cpu().numpy()
    v = {k: t.cpu().numpy() for k, t in x.items()
         if isinstance(t, torch.Tensor) and k not in ("logits", "y")}
    for b in range(case["rows"]):
        words = v["tokens"][v["offsets"][b]:v["offsets"][b + 1]]
        r, f, p = (float(v[k][b]) for k in ("repetition", "frequency", "presence"))
        for w in np.unique(words):
            y[b, w] = y[b, w] / r if y[b, w] > 0 else y[b, w] * r
        for w, n in zip(*np.unique(words[v["prompts"][b]:], return_counts=True)):
            y[b, w] -= f * n + p
        if "bias" in v:
            a, e = v["bias_offsets"][b:b + 2]
            for w, add in dict(zip(v["bias_words"][a:e].tolist(), v["bias"][a:e].tolist())).items():
                y[b, w] += add
        if "mask" in v and v["mask_rows"][b] >= 0:
            bits = np.ascontiguousarray(v["mask"][v["mask_rows"][b]]).view(np.uint8)
            off = np.unpackbits(bits, bitorder="little")[:case["vocab"]] == 0
            y[b, off] = -np.inf
    return torch.from_numpy(y)


# ---- what a pass cannot do without ------------------------------------------------

def work(case):
    d, page = case.get("dim"), case.get("page")
    if case["kind"] == "write":
        counts = _spread(case["batch"], case["rows_low"], case["rows_high"], 3)
        starts = _spread(case["batch"], case["start_low"], case["start_high"], 4)
        rows = sum(counts)
        back = sum(starts) + rows if case["whole"] else rows
        row = case["kv_heads"] * d
        # new rows read, their codes written; the rows asked for read (but for those just
        # written) and given back
        return {"bytes": 2 * row * (rows * (_SIZE[case["new"]] + 1) + (back - rows)
                                    + back * _SIZE[case["back"]])
                + 2 * 4 * case["kv_heads"] * back + 16 * case["batch"],
                "flops": 2 * row * (4 * rows + 2 * back)}
    if case["kind"] == "decode":
        lens = _spread(case["batch"], case["low"], case["high"], 1)
        keys, rows = sum(lens), case["batch"] * case["q_heads"]
        pages = sum(-(-n // page) for n in lens)
        return {"bytes": 2 * keys * case["kv_heads"] * (d + 4) + 2 * rows * d * _SIZE[case["q"]]
                + 4 * pages + 4 * case["batch"], "flops": 4 * keys * case["q_heads"] * d}
    if case["kind"] == "shared":
        prefix = _spread(case["prefixes"], case["prefix_low"], case["prefix_high"], 5)
        lens = _spread(case["batch"], case["low"], case["high"], 6)
        held, rows = sum(prefix) + sum(lens), case["batch"] * case["q_heads"]
        seen = sum(lens) + sum(n * p for n, p in zip(_shares(case), prefix))
        row = d * _SIZE[case["cache"]] + 4 * (case["cache"] == "q8")
        pages = sum(-(-n // page) for n in prefix + lens)
        return {"bytes": 2 * held * case["kv_heads"] * row + 2 * rows * d * _SIZE[case["q"]]
                + 4 * pages + 4 * case["batch"], "flops": 4 * seen * case["q_heads"] * d}
    tokens = sum(_spread(case["rows"], case["low"], case["high"], 7))
    values = case["rows"] * case["vocab"]
    return {"bytes": 2 * values * _SIZE[case["logits"]] + 4 * tokens
            + case["rows"] * case["biases"] * 4 + case["masks"] * case["vocab"] / 8
            + 20 * case["rows"], "flops": 4 * tokens}
