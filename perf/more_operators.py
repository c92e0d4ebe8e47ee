"""Cases for the operators of generation with a quantised cache: writing keys and
values into 8- or 4-bit pages and reading them back, attention of new tokens
over such pages, and the choice of the next token from the logits.

A cached row of head_dim values is kept in blocks of 32: whole numbers n of 8
bits (stored as n + 128, |n| <= 127) or 4 bits (n + 8, |n| <= 7, the even
dimension in the low half of a byte), and one exponent byte e per block; the
block's values are n * 2^(e - 127).  e is the exponent of the block's largest
magnitude less 6 (8 bits) or 2 (4 bits), so n is rounded to the nearest whole
number and cut to the largest; f16 caches stop at 2^-24, a block of zeros has
e = 0.

Every case has a plain form (elementary torch operations) and, where ``own`` is
set, the framework's own calls.  Lengths, pages and settings of a case follow
from its numbers alone; the values of the tensors follow from the seed.
"""
import os
import random
import sys

import numpy as np
import torch

own = False

DEV = "cuda"
DTYPES = {"f16": torch.float16, "bf16": torch.bfloat16, "f32": torch.float32}
BLOCK = 32          # values under one exponent byte
FORMATS = {"i8": (6, 127), "i4": (2, 7)}  # what the exponent is lowered by, the largest whole number
DEPTH = 40.0        # a token this far below the top (in natural units of the scaled logits) is never chosen


def _bb():
    path = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "bonsai.cpp_b200")
    if path not in sys.path:
        sys.path.insert(0, path)
    import bonsai_b200
    return bonsai_b200


# ------------------------------------------------------------------- cases
def _cached(kind, name, n, ctx_lo, ctx_hi, q_lo, q_hi, page, heads, kv_heads, dim, dtype, fmt, chunks=None, pick=1):
    """chunks: how many of the n sequences have q_lo to q_hi new tokens (the others one); None: all."""
    c = {"kind": kind, "n": n, "ctx_lo": ctx_lo, "ctx_hi": ctx_hi, "q_lo": q_lo, "q_hi": q_hi, "page": page,
         "heads": heads, "kv_heads": kv_heads, "dim": dim, "dtype": dtype, "fmt": fmt,
         "chunks": n if chunks is None else chunks, "pick": pick}
    return dict(c, name=name) if name else c


def _sample(name, rows, vocab, dtype, spread, temperature, top_k, top_p, min_p, masked=0.0, pick=1):
    """The settings are the ends of ranges that the rows are spread over."""
    c = {"kind": "sample", "rows": rows, "vocab": vocab, "dtype": dtype, "spread": spread, "t_lo": temperature[0],
         "t_hi": temperature[1], "k_lo": top_k[0], "k_hi": top_k[1], "p_lo": top_p[0], "p_hi": top_p[1],
         "m_lo": min_p[0], "m_hi": min_p[1], "masked": masked, "pick": pick}
    return dict(c, name=name) if name else c


def listed():
    return [
        # prompt rewriting, one token at a time, one user: latency counts
        _cached("attend", "attend-one", 1, 901, 901, 1, 1, 16, 32, 8, 128, "f16", "i8"),
        # the same for a batch of users
        _cached("attend", "attend-tokens", 64, 130, 4000, 1, 1, 16, 32, 8, 128, "bf16", "i8", pick=6),
        # few users with a long cache, in the smaller format
        _cached("attend", "attend-long", 4, 30000, 65536, 1, 1, 64, 32, 8, 128, "f16", "i4", pick=7),
        # prompts behind a cached shared prefix, or a long prompt taken in chunks
        _cached("attend", "attend-chunk", 6, 1000, 8192, 33, 512, 32, 32, 8, 128, "bf16", "i8", pick=8),
        # a served batch: most users at one token, the prompts of a few taken in chunks beside them
        _cached("attend", "attend-mixed", 40, 300, 5000, 100, 400, 16, 28, 4, 128, "f16", "i4", chunks=3, pick=9),
        # what a step of a batch of users adds to the cache
        _cached("store", "store-tokens", 64, 130, 4000, 1, 1, 16, 32, 8, 128, "bf16", "i8", pick=6),
        # the prompts of a batch, up to the 512-token limit of the image model's text input
        _cached("store", "store-prompts", 48, 7, 512, 7, 512, 16, 32, 8, 128, "f16", "i8", pick=3),
        # long documents, in the smaller format
        _cached("store", "store-long", 3, 8000, 20007, 8000, 20007, 64, 32, 8, 128, "bf16", "i4", pick=4),
        # one user's next token
        _sample("sample-one", 1, 150001, "f32", 2.5, (0.7, 0.7), (50, 50), (0.9, 0.9), (0.0, 0.0)),
        # a batch of users with settings of their own, some of them greedy, some without any limit
        _sample("sample-batch", 64, 128000, "f32", 2.0, (0.0, 1.3), (0, 200), (0.5, 1.0), (0.0, 0.1), pick=2),
        # flat distributions cut by their mass alone: many tokens are left to choose from
        _sample("sample-flat", 32, 150001, "bf16", 1.0, (1.0, 1.5), (0, 0), (0.8, 0.95), (0.0, 0.0), pick=3),
        # many short rows, most tokens ruled out by a grammar
        _sample("sample-masked", 256, 32000, "f16", 2.0, (0.6, 1.0), (0, 40), (0.9, 1.0), (0.02, 0.1), masked=0.7, pick=4),
    ]


def _log(rng, lo, hi):
    return int(round(lo * (hi / lo) ** rng.random()))


def draw(rng):
    kind = rng.choice(["attend", "attend", "store", "sample"])
    pick = rng.randrange(1 << 20)
    if kind == "sample":
        vocab = _log(rng, 300, 200000)
        rows = _log(rng, 1, max(1, min(256, 8000000 // vocab)))
        t, k, p = rng.choice([(0.6, 1.0), (0.0, 2.0), (1.0, 1.0)]), rng.choice([(0, 0), (1, 60), (0, 2000)]), \
            rng.choice([(1.0, 1.0), (0.3, 1.0), (0.85, 0.95)])
        return _sample(None, rows, vocab, rng.choice(["f32", "f16", "bf16"]), rng.choice([0.5, 1.5, 3.0]), t, k, p,
                       rng.choice([(0.0, 0.0), (0.0, 0.2)]), rng.choice([0.0, 0.0, 0.9]), pick)
    heads, kv_heads = rng.choice([(32, 8), (24, 24), (28, 4), (16, 2), (12, 4), (20, 4), (8, 1)])
    dim, dtype, fmt = rng.choice([128, 128, 64]), rng.choice(["f16", "bf16"]), rng.choice(["i8", "i4"])
    page = rng.choice([16, 32, 64, 128])
    if kind == "store":
        q_hi = _log(rng, 1, 8000)
        n = _log(rng, 1, max(1, min(200, 200000 // (q_hi * kv_heads))))
        q_lo = max(1, q_hi // rng.choice([1, 3, 30]))
        ctx_hi = q_hi + rng.choice([0, rng.randrange(3000)])
        return _cached("store", None, n, q_lo, ctx_hi, q_lo, q_hi, page, heads, kv_heads, dim, dtype, fmt, None, pick)
    hi = _log(rng, 1, 65536)
    n = _log(rng, 1, max(1, min(200, 1500000 // (hi * kv_heads))))
    q_hi = rng.choice([1, 1, _log(rng, 1, max(1, min(hi, 1024, int(2.5e8 / (n * hi * heads)))))])
    ctx_lo = max(q_hi, hi // rng.choice([1, 3, 20]))
    return _cached("attend", None, n, ctx_lo, hi, max(1, q_hi // rng.choice([1, 4])), q_hi, page, heads, kv_heads, dim,
                   dtype, fmt, rng.choice([None, n // 3]), pick)


def _lengths(case):
    """(new tokens, cached tokens with the new ones) of each sequence; the longest of each reach the upper ends."""
    r = random.Random(case["pick"] * 16)
    q = [r.randint(case["q_lo"], case["q_hi"]) if i < case["chunks"] else 1 for i in range(case["n"])]
    if case["chunks"]:
        q[r.randrange(case["chunks"])] = case["q_hi"]
    r.shuffle(q)
    ctx = [r.randint(case["ctx_lo"], case["ctx_hi"]) for _ in q]
    ctx[r.randrange(case["n"])] = case["ctx_hi"]
    return q, [max(a, b) for a, b in zip(q, ctx)]


def _settings(case):
    """(temperature, top_k, top_p, min_p) of each row; at a range's ends some rows have exactly the end."""
    r = random.Random(case["pick"] * 16 + 3)

    def spread(lo, hi, whole=False):
        v = [lo if (x := r.random()) < 0.15 else hi if x > 0.85 else lo + (hi - lo) * r.random() for _ in range(case["rows"])]
        return [int(x) for x in v] if whole else v

    return (spread(case["t_lo"], case["t_hi"]), spread(case["k_lo"], case["k_hi"], True),
            spread(case["p_lo"], case["p_hi"]), spread(case["m_lo"], case["m_hi"]))


def _cumulated(lens):
    cu = [0]
    for x in lens:
        cu.append(cu[-1] + x)
    return cu


# ----------------------------------------------------------------- prepare
def _ints(v):
    return torch.tensor(v, dtype=torch.int32, device=DEV)


def _randn(g, *shape, dtype=torch.float32, std=1.0):
    return (torch.randn(*shape, device=DEV, generator=g) * std).to(dtype)


def prepare(case, seed):
    g = torch.Generator(device=DEV)
    g.manual_seed(seed)
    return {"attend": _prepare_attend, "store": _prepare_store, "sample": _prepare_sample}[case["kind"]](case, g)


def _new_pages(c, n_pages):
    """Codes [page][slot][head][bytes] and exponents [page][slot][head][dim / 32], these with a head's
    slots one after another in memory."""
    width = c["dim"] if c["fmt"] == "i8" else c["dim"] // 2
    codes = torch.zeros(n_pages, c["page"], c["kv_heads"], width, dtype=torch.uint8, device=DEV)
    exps = torch.zeros(n_pages, c["kv_heads"], c["page"], c["dim"] // BLOCK, dtype=torch.uint8, device=DEV)
    return codes, exps.transpose(1, 2)


def _prepare_pages(c):
    q, ctx = _lengths(c)
    per = [-(-x // c["page"]) for x in ctx]
    total = sum(per) + 3
    r = random.Random(c["pick"])
    free = list(range(total))
    r.shuffle(free)  # pages in the order of their allocation by many requests
    table, at = [], 0
    for k in per:
        table.append(free[at:at + k] + [0] * (max(per) - k))
        at += k
    s = {"case": c, "cu": _ints(_cumulated(q)), "ctx": _ints(ctx), "table": _ints(table), "max_q": max(q),
         "max_ctx": max(ctx), "scale": c["dim"] ** -0.5, "k_pages": _new_pages(c, total),
         "v_pages": _new_pages(c, total)}
    if own:
        s["k_cache"], s["v_cache"] = (_bb().QuantPages(codes, exps, c["fmt"]) for codes, exps in (s["k_pages"], s["v_pages"]))
    return s, sum(q), total


def _prepare_attend(c, g):
    s, t, total = _prepare_pages(c)
    for codes, exps in (s["k_pages"], s["v_pages"]):
        step = max(1, (1 << 26) // codes[0].numel())
        for a in range(0, total, step):  # what earlier steps have written
            part = slice(a, min(total, a + step))
            x = _randn(g, part.stop - a, c["page"], c["kv_heads"], c["dim"], dtype=DTYPES[c["dtype"]], std=1.2)
            codes[part], exps[part] = _plain_quantise(x, c["fmt"])
    s["q"] = _randn(g, t, c["heads"], c["dim"], dtype=DTYPES[c["dtype"]], std=1.2)
    return s


def _prepare_store(c, g):
    s, t, _ = _prepare_pages(c)
    # a few channels of the keys are much larger than the others
    gain = _randn(g, c["kv_heads"], c["dim"]).mul_(0.8).exp_()
    s["k"] = (_randn(g, t, c["kv_heads"], c["dim"]) * gain).to(DTYPES[c["dtype"]])
    s["v"] = _randn(g, t, c["kv_heads"], c["dim"], dtype=DTYPES[c["dtype"]], std=1.2)
    s["first"] = s["ctx"] - (s["cu"][1:] - s["cu"][:-1])  # place of each sequence's first new token
    return s


def _prepare_sample(c, g):
    n, v = c["rows"], c["vocab"]
    logits = _randn(g, n, v, std=c["spread"])
    # a few likely tokens above the bulk
    at = torch.randint(0, v, (n, 24), device=DEV, generator=g)
    logits.scatter_(1, at, _randn(g, n, 24, std=1.5) + 4.5 * c["spread"])
    if c["masked"]:
        logits[torch.rand(n, v, device=DEV, generator=g) < c["masked"]] = float("-inf")
    t, k, p, m = _settings(c)
    f = lambda x: torch.tensor(x, dtype=torch.float32, device=DEV)  # noqa: E731
    return {"case": c, "logits": logits.to(DTYPES[c["dtype"]]), "temperature": f(t), "top_k": _ints(k), "top_p": f(p),
            "min_p": f(m), "u": torch.rand(n, device=DEV, generator=g)}


# --------------------------------------------------------------------- run
def run(state):
    kind = state["case"]["kind"]
    if own:
        return {"attend": _own_attend, "store": _own_store, "sample": _own_sample}[kind](state)
    return {"attend": _plain_attend, "store": _plain_store, "sample": _plain_sample}[kind](state)


def _own_attend(s):
    out = torch.empty_like(s["q"])
    _bb().paged_attention_quant(s["q"], s["k_cache"], s["v_cache"], s["table"], s["cu"], s["ctx"], s["max_ctx"], out,
                                max_q=s["max_q"], scale=s["scale"])
    return out


def _own_store(s):
    bb = _bb()
    k, v = torch.empty_like(s["k"]), torch.empty_like(s["v"])
    bb.paged_append_quant(s["k"], s["v"], s["k_cache"], s["v_cache"], s["table"], s["cu"], s["ctx"])
    bb.paged_read_quant(s["k_cache"], s["v_cache"], s["table"], s["cu"], s["first"], k, v)
    return {"k": k, "v": v}


def _own_sample(s):
    n = s["logits"].shape[0]
    tokens, probs = torch.empty(n, dtype=torch.int32, device=DEV), torch.empty(n, device=DEV)
    _bb().sample_tokens(s["logits"], s["u"], tokens, probs=probs, temperature=s["temperature"], top_k=s["top_k"],
                        top_p=s["top_p"], min_p=s["min_p"])
    return {"tokens": tokens, "probs": probs}


# ------------------------------------------------------------- plain forms
def _power(n):
    """2^n in f32, n from -127 (a zero) to 127."""
    return ((n + 127) << 23).view(torch.float32)


def _plain_quantise(x, fmt):
    """16-bit values [..., dim] -> codes and exponents."""
    lower, most = FORMATS[fmt]
    b = x.float().unflatten(-1, (-1, BLOCK))
    top = b.abs().amax(-1, keepdim=True)
    e = ((top.view(torch.int32) >> 23) - lower).clamp(min=103 if x.dtype == torch.float16 else 1)
    n = (b * _power(127 - e)).round_().clamp_(-most, most).to(torch.int32)
    n, e = torch.where(top > 0, n, 0).flatten(-2), torch.where(top > 0, e, 0).squeeze(-1).to(torch.uint8)
    if fmt == "i8":
        return (n + 128).to(torch.uint8), e
    return ((n[..., 0::2] + 8) | ((n[..., 1::2] + 8) << 4)).to(torch.uint8), e


def _plain_values(codes, exps, fmt):
    """Codes and exponents -> f32 values [..., dim]."""
    if fmt == "i8":
        n = codes.float() - 128
    else:
        n = torch.stack([codes & 15, codes >> 4], -1).flatten(-2).float() - 8
    return (n.unflatten(-1, (-1, BLOCK)) * _power(exps.int() - 127)[..., None]).flatten(-2)


def _rows(cu, longest, total):
    """Packed rows as [n][longest] indices, and which of them are real."""
    pos = torch.arange(longest, device=DEV)
    real = pos < (cu[1:] - cu[:-1])[:, None]
    return (cu[:-1, None] + pos).clamp(max=total - 1), real


def _places(s):
    """Place in its sequence of every new token [n][max_q]."""
    return torch.arange(s["max_q"], device=DEV) + (s["ctx"] - (s["cu"][1:] - s["cu"][:-1]))[:, None]


def _plain_attend(s):
    c, q = s["case"], s["q"].float()
    at, real = _rows(s["cu"], s["max_q"], q.shape[0])
    k, v = (_plain_values(codes[s["table"].long()], exps[s["table"].long()], c["fmt"]).flatten(1, 2)
            for codes, exps in (s["k_pages"], s["v_pages"]))
    seen = torch.arange(k.shape[1], device=DEV)
    keep = (seen <= _places(s)[:, :, None]) & (seen < s["ctx"][:, None, None])
    hk, m = k.shape[2], s["max_q"]
    x = q[at].unflatten(2, (hk, -1)).permute(0, 2, 3, 1, 4).flatten(2, 3)  # n Hk (g i) D
    scores = torch.matmul(x, k.permute(0, 2, 3, 1)).mul_(s["scale"]).unflatten(2, (-1, m))
    scores.masked_fill_(~keep[:, None, None], float("-inf"))
    top = scores.amax(-1, keepdim=True)
    scores.sub_(top.masked_fill_(top == float("-inf"), 0.0)).exp_()
    total = scores.sum(-1, keepdim=True)
    p = scores.div_(total.masked_fill_(total == 0, 1.0)).flatten(2, 3)
    out = torch.matmul(p, v.transpose(1, 2)).unflatten(2, (-1, m)).permute(0, 3, 1, 2, 4).flatten(2, 3)
    return out[real].to(s["q"].dtype)


def _plain_store(s):
    c, page = s["case"], s["case"]["page"]
    _, real = _rows(s["cu"], s["max_q"], s["k"].shape[0])
    pos = _places(s)
    slot = s["table"].gather(1, (pos // page).clamp(max=s["table"].shape[1] - 1).long())[real].long(), (pos % page)[real]
    out = {}
    for name, pages in (("k", s["k_pages"]), ("v", s["v_pages"])):
        codes, exps = pages
        codes[slot], exps[slot] = _plain_quantise(s[name], c["fmt"])
        out[name] = _plain_values(codes[slot], exps[slot], c["fmt"]).to(s[name].dtype)
    return out


def _plain_sample(s):
    # in 64 bits: a choice next to a border goes by sums over the whole row
    logits = s["logits"].float()
    n, vocab = logits.shape
    logits = torch.where(logits.isnan(), float("-inf"), logits)
    t = s["temperature"].double()[:, None]
    greedy = ~(t > 0)
    top = logits.amax(1, keepdim=True)
    z = (logits.double() - top.double()) / torch.where(greedy, 1.0, t)
    z = torch.where(logits == top, 0.0, z)
    w = torch.where((z >= -DEPTH) & (logits > float("-inf")), torch.exp(z), 0.0)
    order = torch.sort(logits, dim=1, descending=True, stable=True).indices
    w = w.gather(1, order)
    rank = torch.arange(vocab, device=DEV)
    k = torch.where(greedy, 1, torch.where(s["top_k"][:, None] <= 0, vocab, s["top_k"][:, None]))
    w = torch.where(rank < k, w, 0.0)
    limit = s["top_p"].double()[:, None]
    over = (w.cumsum(1) - w >= limit * w.sum(1, keepdim=True)) & (limit < 1)
    w = torch.where((over | (w < s["min_p"].double()[:, None])) & (rank > 0), 0.0, w)
    w = torch.zeros_like(w).scatter_(1, order, w)
    cum = w.cumsum(1)
    target = s["u"].double().clamp(0, 1)[:, None] * cum[:, -1:]
    last = torch.where(w > 0, rank, -1).amax(1)
    tokens = torch.minimum((cum <= target).sum(1), last)
    probs = w.gather(1, tokens.clamp(min=0)[:, None])[:, 0] / cum[:, -1].clamp(min=1e-300)
    return {"tokens": tokens.int(), "probs": torch.where(tokens < 0, 0.0, probs).float()}


# -------------------------------------------------------------------- work
def work(case):
    c = case
    if c["kind"] == "sample":
        width = 4 if c["dtype"] == "f32" else 2
        # every logit once; a subtraction, a product and an exponential of each
        return {"bytes": c["rows"] * (c["vocab"] * width + 28), "flops": 3.0 * c["rows"] * c["vocab"]}
    q, ctx = _lengths(c)
    row = (c["dim"] if c["fmt"] == "i8" else c["dim"] // 2) + c["dim"] // BLOCK
    if c["kind"] == "store":
        # keys and values: 16-bit values in, codes out, codes in, 16-bit values out
        values = 2 * sum(q) * c["kv_heads"]
        return {"bytes": values * (4 * c["dim"] + 2 * row), "flops": 4.0 * values * c["dim"]}
    pairs = sum(a * b - a * (a - 1) // 2 for a, b in zip(q, ctx))
    return {"bytes": 2 * c["kv_heads"] * sum(ctx) * row + 4 * c["dim"] * c["heads"] * sum(q),
            "flops": 4.0 * pairs * c["heads"] * c["dim"]}


# ------------------------------------------------------------------- exact
def _exact_power(n):
    """2^n in f64 for whole n of 64 bits."""
    return ((n + 1023) << 52).view(torch.float64)


def _exact_values(pages, ids, c):
    """The cached values of some pages, [tokens][head][dim], f64."""
    codes, exps = (x[ids].flatten(0, 1).long() for x in pages)
    if c["fmt"] == "i4":
        codes = torch.cat([(codes % 16)[..., None], (codes // 16)[..., None]], -1).flatten(-2)
    n = (codes - (128 if c["fmt"] == "i8" else 8)).double()
    return n * _exact_power(exps - 127).repeat_interleave(BLOCK, -1)


def _exact_attend(s):
    c, cu, outs = s["case"], s["cu"].tolist(), []
    group = c["heads"] // c["kv_heads"]
    for i, length in enumerate(s["ctx"].tolist()):
        ids = s["table"][i, :-(-length // c["page"])].long()
        k, v = (_exact_values(pages, ids, c)[:length] for pages in (s["k_pages"], s["v_pages"]))
        q = s["q"][cu[i]:cu[i + 1]].double()
        hidden = torch.ones(q.shape[0], length, dtype=torch.bool, device=DEV).triu(length - q.shape[0] + 1)
        out = torch.empty_like(q)
        for h in range(c["heads"]):
            a = (q[:, h] @ k[:, h // group].T) * s["scale"]
            out[:, h] = torch.softmax(a.masked_fill(hidden, float("-inf")), 1) @ v[:, h // group]
        outs.append(out)
    return torch.cat(outs)


def _exact_store(s):
    lower, most = FORMATS[s["case"]["fmt"]]
    out = {}
    for name in ("k", "v"):
        x = s[name].double().unflatten(-1, (-1, BLOCK))
        exponent = torch.frexp(x.abs().amax(-1, keepdim=True)).exponent - 1 - lower
        step = _exact_power(exponent.clamp(min=-24 if s[name].dtype == torch.float16 else -126).long())
        out[name] = (torch.round(x / step).clamp(-most, most) * step).flatten(-2)
    return out


def _exact_sample(s):
    logits = s["logits"].double().cpu().numpy()
    t, k, p, m, u = (s[x].cpu().numpy() for x in ("temperature", "top_k", "top_p", "min_p", "u"))
    tokens, probs = [], []
    for r, row in enumerate(logits):
        order = np.lexsort((np.arange(row.size), -row))  # largest first, the lowest index of equals
        order = order[row[order] > -np.inf]
        if t[r] <= 0 or order.size == 0:
            tokens.append(int(order[0]) if order.size else -1)
            probs.append(1.0 if order.size else 0.0)
            continue
        if k[r] > 0:
            order = order[:k[r]]
        z = (row[order] - row[order[0]]) / np.float64(t[r])
        order, z = order[z >= -DEPTH], z[z >= -DEPTH]
        w = np.exp(z)
        if p[r] < 1:
            keep = np.concatenate([[0.0], np.cumsum(w)[:-1]]) < np.float64(p[r]) * w.sum()
            keep[0] = True
            order, w = order[keep], w[keep]
        keep = w >= np.float64(m[r])
        keep[0] = True
        order, w = order[keep], w[keep]
        by = np.argsort(order)
        order, w = order[by], w[by]
        cum = np.cumsum(w)
        at = min(int(np.searchsorted(cum, np.float64(u[r]) * cum[-1], side="right")), order.size - 1)
        tokens.append(int(order[at]))
        probs.append(w[at] / cum[-1])
    return {"tokens": torch.tensor(tokens, dtype=torch.int32, device=DEV),
            "probs": torch.tensor(probs, dtype=torch.float64, device=DEV)}


def exact(case, seed):
    return {"attend": _exact_attend, "store": _exact_store, "sample": _exact_sample}[case["kind"]](prepare(case, seed))
