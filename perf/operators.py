"""What the serving operators are timed and checked on: attention of one new
token per sequence over a paged key/value cache, causal attention of packed
prompts, the append that fills the pages, and sampling of the next token.

A case is a dict of plain values; ``prepare`` makes what a serving loop has in
hand before the call, ``run`` makes one pass and returns its outputs whole:
through the framework's entry points where ``own`` is true, else in a plain
form of elementary torch operations. ``exact`` gives the same outputs in 64
bits, ``work`` the bytes and operations that a pass cannot do without.
"""
import math
import random

import numpy as np
import torch

own = False

DEV = "cuda"
_FLOAT = {"bf16": torch.bfloat16, "f32": torch.float32}
_SIZE = {"bf16": 2, "f32": 4}

# (query heads, kv heads): the dense decoder's, the hybrid model's, and from one
# query head per kv head to eight
HEADS = [(16, 8), (8, 2), (8, 8), (32, 8), (32, 4), (64, 8)]
# the vocabularies of the dense decoder and of the hybrid model
VOCABS = [151936, 248320]


def listed():
    return [
        # one user's next token over a short context: latency counts
        dict(name="decode-step", kind="decode", batch=1, q_heads=16, kv_heads=8, dim=128, page=16,
             low=777, high=777, cache="bf16", q="bf16"),
        # a batch of long contexts of ragged lengths
        dict(name="decode-long", kind="decode", batch=8, q_heads=32, kv_heads=8, dim=128, page=64,
             low=512, high=8192, cache="bf16", q="bf16"),
        # many users, from a first token on, f32 queries as the f32 projections give them
        dict(name="decode-many", kind="decode", batch=96, q_heads=16, kv_heads=8, dim=128, page=16,
             low=1, high=1500, cache="bf16", q="f32"),
        # the hybrid model's attention heads over f32 caches, a page size that is no power of two
        dict(name="decode-f32", kind="decode", batch=4, q_heads=8, kv_heads=2, dim=256, page=48,
             low=300, high=2048, cache="f32", q="f32"),
        # a handful of short chat turns admitted together
        dict(name="prompt-short", kind="prompt", batch=16, q_heads=16, kv_heads=8, dim=128, low=1,
             high=60, q="bf16", pad=0),
        # prompts of very different lengths in one batch, padded behind the last one
        dict(name="prompt-ragged", kind="prompt", batch=12, q_heads=32, kv_heads=8, dim=128,
             low=64, high=2000, q="bf16", pad=100),
        # two long documents, eight query heads to a kv head
        dict(name="prompt-long", kind="prompt", batch=2, q_heads=64, kv_heads=8, dim=128, low=5000,
             high=7000, q="bf16", pad=0),
        # the hybrid model's attention heads, f32 queries and outputs
        dict(name="prompt-f32", kind="prompt", batch=3, q_heads=8, kv_heads=2, dim=256, low=100,
             high=900, q="f32", pad=0),
        # one new key and value for each user of a batch
        dict(name="append-step", kind="append", batch=96, kv_heads=8, dim=128, page=16, rows_low=1,
             rows_high=1, start_low=0, start_high=1500, new="f32", cache="bf16"),
        # whole prompts into their pages
        dict(name="append-prompt", kind="append", batch=12, kv_heads=8, dim=128, page=64,
             rows_low=64, rows_high=2000, start_low=0, start_high=200, new="bf16", cache="bf16"),
        # one user's next token, filtered the way chat programs do by default
        dict(name="sample-step", kind="sample", rows=1, vocab=151936, logits="f32", greedy=0.0,
             top_k=20, top_p=0.8, min_p=0.0),
        # a batch of users with settings of their own, some greedy, the larger vocabulary
        dict(name="sample-batch", kind="sample", rows=64, vocab=248320, logits="f32", greedy=0.1,
             top_k=200, top_p=0.95, min_p=0.02),
    ]


def _log(rng, low, high):
    """A whole number between low and high, spread over its logarithm."""
    return max(low, min(high, round(math.exp(rng.uniform(math.log(low), math.log(high))))))


def draw(rng):
    kind = rng.choice(["decode", "decode", "decode", "prompt", "prompt", "prompt", "append",
                       "sample", "sample"])
    hq, hkv = rng.choice(HEADS)
    dim = rng.choice([64, 128, 128, 256])
    page = rng.choice([16, 16, 32, 48, 64, 128, 256])
    if kind == "decode":
        cache = rng.choice(["bf16", "bf16", "f32"])
        high = _log(rng, 1, 8192)
        # at most the listed long caches' bytes
        most = max(1, min(256, 8 * 4352 * 8 * 128 * 2 // (high * hkv * dim * _SIZE[cache])))
        return dict(kind="decode", batch=_log(rng, 1, most), q_heads=hq, kv_heads=hkv, dim=dim,
                    page=page, low=max(1, high // rng.choice([1, 4, 16, 8192])), high=high,
                    cache=cache, q=rng.choice(["bf16", "f32"]))
    if kind == "prompt":
        high = _log(rng, 1, 7000)
        low = max(1, high // rng.choice([1, 2, 8, 7000]))
        # at most the listed long documents' operations
        most = max(1, min(64, 2 * 64 * 128 * 5000 ** 2 // (hq * dim * high ** 2)))
        if high ** 2 * hq * dim > 2 * 64 * 128 * 6000 ** 2:
            dim = 64
        return dict(kind="prompt", batch=_log(rng, 1, most), q_heads=hq, kv_heads=hkv, dim=dim,
                    low=low, high=high, q=rng.choice(["bf16", "bf16", "f32"]),
                    pad=rng.choice([0, 0, 7, 100]))
    if kind == "append":
        high = rng.choice([1, _log(rng, 1, 2000)])
        most = max(1, min(256, 12000 * 8 * 128 // (high * hkv * dim)))
        return dict(kind="append", batch=_log(rng, 1, most), kv_heads=hkv, dim=dim, page=page,
                    rows_low=max(1, high // rng.choice([1, 4, 2000])), rows_high=high, start_low=0,
                    start_high=_log(rng, 1, 2000), new=rng.choice(["bf16", "f32"]),
                    cache=rng.choice(["bf16", "bf16", "f32"]))
    vocab = rng.choice(VOCABS + [_log(rng, 1000, 248320)])
    return dict(kind="sample", rows=_log(rng, 1, 64), vocab=vocab,
                logits=rng.choice(["f32", "f32", "bf16"]), greedy=rng.choice([0.0, 0.2]),
                top_k=rng.choice([0, 1, 20, 50, 200, 1000]),
                top_p=rng.choice([1.0, 0.5, 0.8, 0.9, 0.95, 0.99]),
                min_p=rng.choice([0.0, 0.0, 0.02, 0.1]))


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


def _pages(g, case, lens, entries):
    """A pool of key and value pages with old contents, and a table that gives each
    sequence the pages of its `lens` positions, in no order; -1 where it has none."""
    page, hkv, d = case["page"], case["kv_heads"], case["dim"]
    need = [-(-n // page) for n in lens]
    pool = sum(need) + 3
    order = torch.randperm(pool, generator=g, device=DEV).to(torch.int32)
    table = torch.full((len(lens), entries), -1, dtype=torch.int32, device=DEV)
    at = 0
    for b, n in enumerate(need):
        table[b, :n] = order[at:at + n]
        at += n
    kp, vp = (_normal(g, pool, hkv, page, d).to(_FLOAT[case["cache"]]) for _ in range(2))
    return kp, vp, table


def _decode_inputs(case, seed):
    g = _gen(seed)
    lens = _spread(case["batch"], case["low"], case["high"], 1)
    kp, vp, table = _pages(g, case, lens, -(-case["high"] // case["page"]))
    q = _normal(g, case["batch"], case["q_heads"], case["dim"]).to(_FLOAT[case["q"]])
    return dict(q=q, k_pages=kp, v_pages=vp, table=table, lens=_int(lens))


def _offsets(counts):
    at = [0]
    for n in counts:
        at.append(at[-1] + n)
    return at


def _prompt_inputs(case, seed):
    g = _gen(seed)
    offsets = _offsets(_spread(case["batch"], case["low"], case["high"], 2))
    t, d = offsets[-1] + case["pad"], case["dim"]
    q = _normal(g, t, case["q_heads"], d).to(_FLOAT[case["q"]])
    k, v = (_normal(g, t, case["kv_heads"], d).bfloat16() for _ in range(2))
    return dict(q=q, k=k, v=v, offsets=_int(offsets), longest=case["high"])


def _append_inputs(case, seed):
    g = _gen(seed)
    counts = _spread(case["batch"], case["rows_low"], case["rows_high"], 3)
    starts = _spread(case["batch"], case["start_low"], case["start_high"], 4)
    most = case["rows_high"] + case["start_high"]
    kp, vp, table = _pages(g, case, [s + n for s, n in zip(starts, counts)],
                           -(-most // case["page"]))
    offsets = _offsets(counts)
    k, v = (_normal(g, offsets[-1], case["kv_heads"], case["dim"]).to(_FLOAT[case["new"]])
            for _ in range(2))
    return dict(k=k, v=v, k_pages=kp, v_pages=vp, table=table, offsets=_int(offsets),
                starts=_int(starts))


def _sample_inputs(case, seed):
    g = _gen(seed)
    rows, vocab = case["rows"], case["vocab"]
    # a word's logit falls with the logarithm of its rank, more steeply where the
    # model is sure of itself; bf16 values, as the output layer rounds them (many ties)
    rank = torch.rand(rows, vocab, generator=g, device=DEV).mul_(vocab).add_(1)
    slope = 1.0 + 1.2 * torch.rand(rows, 1, generator=g, device=DEV)
    logits = (12.0 - slope * rank.log_() + _normal(g, rows, vocab, std=0.5)).bfloat16()
    uniform = torch.rand(rows, generator=g, device=DEV)
    draw_ = torch.rand(4, rows, generator=g, device=DEV)
    temperature = 0.6 + 0.6 * draw_[0]
    temperature[draw_[1] < case["greedy"]] = 0.0
    top_k = torch.full((rows,), case["top_k"], dtype=torch.int32, device=DEV)
    if rows > 1:  # every user has settings of their own
        top_k = (top_k * (0.5 + draw_[2])).to(torch.int32)
    top_p = torch.full((rows,), case["top_p"], device=DEV)
    min_p = torch.full((rows,), case["min_p"], device=DEV)
    if rows > 1:
        top_p, min_p = 1 - (1 - top_p) * (0.5 + draw_[3]), min_p * (0.5 + draw_[3])
    return dict(logits=logits.to(_FLOAT[case["logits"]]), uniform=uniform, temperature=temperature,
                top_k=top_k, top_p=top_p, min_p=min_p)


_INPUTS = {"decode": _decode_inputs, "prompt": _prompt_inputs, "append": _append_inputs,
           "sample": _sample_inputs}

_rt = None


def _runtime():
    global _rt
    if _rt is None:
        import rxla_amd as rx
        _rt = rx.Runtime(0)
    return _rt


def prepare(case, seed):
    state = _INPUTS[case["kind"]](case, seed)
    if case["kind"] in ("decode", "prompt"):
        state["y"] = torch.zeros_like(state["q"])
    elif case["kind"] == "sample":
        state["y"] = torch.zeros(case["rows"], dtype=torch.int32, device=DEV)
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
    if kind == "decode":
        rx.grouped_query_attention_paged(rt, h["q"], h["k_pages"], h["v_pages"], h["table"],
                                         h["lens"], out=h["y"])
        return state["y"]
    if kind == "prompt":
        rx.grouped_query_attention_packed(rt, h["q"], h["k"], h["v"], h["offsets"], out=h["y"])
        return state["y"]
    if kind == "append":
        rx.paged_kv_append(rt, h["k_pages"], h["v_pages"], h["k"], h["v"], h["table"],
                           h["starts"], h["offsets"])
        return state["k_pages"], state["v_pages"]
    rx.sample(rt, h["logits"], h["uniform"], h["temperature"], h["top_k"], h["top_p"], h["min_p"],
              out=h["y"])
    return state["y"]


def _attend(q, k, v, seen):
    """softmax(q k^T / sqrt(d)) v over the keys that `seen` leaves; 0 for a row without any."""
    s = torch.matmul(q, k.transpose(-1, -2).contiguous()).mul_(1 / math.sqrt(q.shape[-1]))
    s.masked_fill_(~seen, -math.inf)
    top = s.amax(dim=-1, keepdim=True).clamp_min(torch.finfo(s.dtype).min)
    p = s.sub_(top).exp_()
    return torch.matmul(p, v).div_(p.sum(dim=-1, keepdim=True).clamp_min(1e-30))


def _plain_decode(s):
    q, table, lens = s["q"].float(), s["table"].long(), s["lens"]
    b, hq, d = q.shape
    hkv, page = s["k_pages"].shape[1:3]
    n = table.shape[1] * page
    k, v = (p[table.clamp_min(0)].float().transpose(1, 2).reshape(b, hkv, n, d)
            for p in (s["k_pages"], s["v_pages"]))
    seen = torch.arange(n, device=DEV)[None, :] < lens[:, None]
    o = _attend(q.reshape(b, hkv, hq // hkv, d), k, v, seen[:, None, None, :])
    return o.reshape(b, hq, d).to(s["q"].dtype)


def _plain_prompt(s):
    q, k, v, offsets, n = s["q"], s["k"], s["v"], s["offsets"].long(), s["longest"]
    (t, hq, d), hkv, b = q.shape, k.shape[1], offsets.numel() - 1
    at = torch.arange(n, device=DEV)
    rows = offsets[:-1, None] + at[None, :]
    there = rows < offsets[1:, None]
    take = rows.clamp_max(t - 1)
    qs = q[take].float().permute(0, 2, 1, 3).reshape(b, hkv, hq // hkv * n, d)
    ks, vs = (x[take].float().transpose(1, 2).contiguous() for x in (k, v))
    seen = (at[None, :] <= at[:, None]).repeat(hq // hkv, 1)
    o = _attend(qs, ks, vs, seen).reshape(b, hq, n, d).transpose(1, 2)
    y = torch.zeros(t + 1, hq, d, device=DEV)  # one row more, for the places behind each prompt
    y[torch.where(there, rows, t)] = o
    return y[:t].to(q.dtype)


def _plain_append(s):
    t, (pool, hkv, page, d) = s["k"].shape[0], s["k_pages"].shape
    row = torch.arange(t, device=DEV)
    offsets = s["offsets"].long()
    seq = torch.bucketize(row, offsets[1:], right=True)
    pos = s["starts"].long()[seq] + row - offsets[seq]
    to = s["table"].long()[seq, pos // page]
    s["k_pages"][to, :, pos % page] = s["k"].to(s["k_pages"].dtype)
    s["v_pages"][to, :, pos % page] = s["v"].to(s["v_pages"].dtype)
    return s["k_pages"], s["v_pages"]


def _plain_sample(s):
    # in 64 bits: which word a random number falls on is decided at the borders
    # between words, and there are a quarter of a million of them
    logits = s["logits"].double()
    v = logits.shape[1]
    greedy = s["temperature"] <= 0
    t = torch.where(greedy, 1.0, s["temperature"]).double()[:, None]
    z, order = logits.sort(dim=1, descending=True, stable=True)
    w = ((z - z[:, :1]) / t).exp()
    k = torch.where(s["top_k"] <= 0, v, s["top_k"]).clamp_max(v).long()[:, None]
    keep = torch.arange(v, device=DEV)[None, :] < k
    mass = (w * keep).cumsum(dim=1)
    p = s["top_p"].double()[:, None]
    keep &= (p >= 1) | (mass - w < p * mass[:, -1:])
    keep &= w >= s["min_p"].double()[:, None]
    keep[:, 0] = True
    mass = (w * keep).cumsum(dim=1)
    at = (mass <= s["uniform"].double()[:, None] * mass[:, -1:]).sum(dim=1, keepdim=True)
    at = torch.where(greedy[:, None], 0, at)
    return order.gather(1, at)[:, 0].to(torch.int32)


_PLAIN = {"decode": _plain_decode, "prompt": _plain_prompt, "append": _plain_append,
          "sample": _plain_sample}


# ---- the same in 64 bits ----------------------------------------------------------

def _softmax_rows(scores):
    e = torch.exp(scores - scores.max(dim=-1, keepdim=True).values)
    return e / e.sum(dim=-1, keepdim=True)


def exact(case, seed):
    x = _INPUTS[case["kind"]](case, seed)
    if case["kind"] == "decode":
        q, page, g = x["q"].double(), case["page"], case["q_heads"] // case["kv_heads"]
        y = torch.zeros_like(q)
        for b, n in enumerate(x["lens"].tolist()):
            ids = x["table"][b, :-(-n // page)].long()
            for h in range(case["kv_heads"]):
                k, v = (p[ids, h].reshape(-1, case["dim"])[:n].double()
                        for p in (x["k_pages"], x["v_pages"]))
                mine = slice(h * g, h * g + g)
                y[b, mine] = _softmax_rows(q[b, mine] @ k.T / math.sqrt(case["dim"])) @ v
        return y
    if case["kind"] == "prompt":
        g, at = case["q_heads"] // case["kv_heads"], x["offsets"].tolist()
        y = torch.zeros(x["q"].shape, dtype=torch.float64, device=DEV)
        for a, e in zip(at, at[1:]):
            future = torch.ones(e - a, e - a, dtype=torch.bool, device=DEV).triu(1)
            for h in range(case["q_heads"]):
                q, k, v = x["q"][a:e, h], x["k"][a:e, h // g], x["v"][a:e, h // g]
                s = q.double() @ k.double().T / math.sqrt(case["dim"])
                y[a:e, h] = _softmax_rows(s.masked_fill(future, -math.inf)) @ v.double()
        return y
    if case["kind"] == "append":
        page, at = case["page"], x["offsets"].tolist()
        got = [x["k_pages"].double(), x["v_pages"].double()]
        for b, start in enumerate(x["starts"].tolist()):
            for new, pool in zip((x["k"], x["v"]), got):
                rows = new[at[b]:at[b + 1]].double()
                pos = torch.arange(start, start + rows.shape[0], device=DEV)
                pool[x["table"][b].long()[pos // page], :, pos % page] = rows
        return tuple(got)
    ids = []
    for row in range(case["rows"]):
        z = x["logits"][row].double().cpu().numpy()
        t, k, p, m, u = (float(x[n][row]) for n in ("temperature", "top_k", "top_p", "min_p",
                                                    "uniform"))
        order = np.lexsort((np.arange(z.size), -z))
        if t <= 0:
            ids.append(int(order[0]))
            continue
        if k > 0:
            order = order[:int(k)]
        w = np.exp((z[order] - z[order[0]]) / t)
        if p < 1:
            count = int(np.searchsorted(np.cumsum(w), p * w.sum())) + 1
            order, w = order[:count], w[:count]
        count = max(1, int((w >= m).sum()))
        order, w = order[:count], w[:count]
        ids.append(int(order[min(count - 1, int(np.searchsorted(np.cumsum(w), u * w.sum(),
                                                                side="right")))]))
    return torch.tensor(ids, dtype=torch.int32)


# ---- what a pass cannot do without ------------------------------------------------

def work(case):
    d = case.get("dim")
    if case["kind"] == "decode":
        lens = _spread(case["batch"], case["low"], case["high"], 1)
        keys, rows = sum(lens), case["batch"] * case["q_heads"]
        pages = sum(-(-n // case["page"]) for n in lens)
        return {"bytes": 2 * keys * case["kv_heads"] * d * _SIZE[case["cache"]]
                + 2 * rows * d * _SIZE[case["q"]] + 4 * pages + 4 * case["batch"],
                "flops": 4 * keys * case["q_heads"] * d}
    if case["kind"] == "prompt":
        lens = _spread(case["batch"], case["low"], case["high"], 2)
        return {"bytes": sum(lens) * d * (2 * case["q_heads"] * _SIZE[case["q"]]
                                          + 2 * case["kv_heads"] * 2) + 4 * len(lens) + 4,
                "flops": 4 * d * case["q_heads"] * sum(n * (n + 1) // 2 for n in lens)}
    if case["kind"] == "append":
        rows = sum(_spread(case["batch"], case["rows_low"], case["rows_high"], 3))
        return {"bytes": 2 * rows * case["kv_heads"] * d * (_SIZE[case["new"]]
                                                            + _SIZE[case["cache"]])
                + 8 * case["batch"], "flops": 0}
    # every logit is read; the exponential of each is the least that a row's sum takes
    values = case["rows"] * case["vocab"]
    return {"bytes": values * _SIZE[case["logits"]] + 24 * case["rows"], "flops": 2 * values}
