"""Cases for the text-encoder operators: packed prompt attention, attention of
new tokens over a paged key/value cache (with the cache's append), and low-rank
adapters of many requests beside a shared B1_0 projection.

Every case has a plain form (elementary torch operations in f32, rounded once
at the end) and, where ``own`` is set, the framework's own calls.  Lengths,
pages and adapters of a case follow from its numbers alone; the values of the
tensors follow from the seed.
"""
import os
import random
import sys

import torch

own = False

DEV = "cuda"
DTYPES = {"f16": torch.float16, "bf16": torch.bfloat16, "f32": torch.float32}
BLOCK, BLOCK_BYTES = 32, 6  # B1_0: f16 scale + 32 sign bits


def _bb():
    path = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "bonsai.cpp_b200")
    if path not in sys.path:
        sys.path.insert(0, path)
    import bonsai_b200
    return bonsai_b200


# ------------------------------------------------------------------- cases
def _prompt(name, n, lo, hi, heads, kv_heads, dim, dtype, causal=True, fused=False, pick=1):
    c = {"kind": "prompt", "n": n, "lo": lo, "hi": hi, "heads": heads, "kv_heads": kv_heads, "dim": dim,
         "dtype": dtype, "causal": causal, "fused": fused, "pick": pick}
    return dict(c, name=name) if name else c


def _paged(name, n, ctx_lo, ctx_hi, q_lo, q_hi, page, heads, kv_heads, dim, dtype, pick=1):
    c = {"kind": "paged", "n": n, "ctx_lo": ctx_lo, "ctx_hi": ctx_hi, "q_lo": q_lo, "q_hi": q_hi, "page": page,
         "heads": heads, "kv_heads": kv_heads, "dim": dim, "dtype": dtype, "pick": pick}
    return dict(c, name=name) if name else c


def _lora(name, n, lo, hi, in_dim, out_dim, slots, rank_lo, rank_hi, out, pick=1):
    c = {"kind": "lora", "n": n, "lo": lo, "hi": hi, "in_dim": in_dim, "out_dim": out_dim, "slots": slots,
         "rank_lo": rank_lo, "rank_hi": rank_hi, "out": out, "pick": pick}
    return dict(c, name=name) if name else c


def listed():
    return [
        # one image request's prompt through an encoder layer: latency counts
        _prompt("prompt-one", 1, 41, 41, 32, 8, 128, "f16"),
        # a batch of prompts up to the 512-token limit of the image model's text input
        _prompt("prompt-batch", 48, 7, 512, 32, 8, 128, "bf16", pick=3),
        # bidirectional encoder with as many key as query heads, q/k/v as slices of one fused projection
        _prompt("prompt-fused", 5, 300, 1025, 24, 24, 64, "f16", causal=False, fused=True, pick=4),
        # one long document
        _prompt("prompt-long", 1, 10007, 10007, 32, 8, 128, "bf16"),
        # prompt rewriting, one token at a time, one user: latency counts
        _paged("paged-one", 1, 901, 901, 1, 1, 16, 32, 8, 128, "f16"),
        # the same for a batch of users
        _paged("paged-tokens", 64, 130, 4000, 1, 1, 16, 32, 8, 128, "bf16", pick=6),
        # few users with a long cache
        _paged("paged-long", 4, 30000, 65536, 1, 1, 64, 32, 8, 128, "f16", pick=7),
        # prompts behind a cached shared prefix, or a long prompt taken in chunks
        _paged("paged-chunk", 6, 1000, 8192, 33, 512, 32, 32, 8, 128, "bf16", pick=8),
        # one token of one request, a square projection
        _lora("lora-one", 1, 1, 1, 3072, 3072, 4, 16, 16, "f16"),
        # one token each of many requests with adapters of their own
        _lora("lora-tokens", 64, 1, 1, 3072, 9216, 64, 8, 64, "f16", pick=10),
        # prompts of several requests, some without an adapter, f32 result
        _lora("lora-prompts", 24, 5, 160, 9216, 3072, 8, 4, 32, "f32", pick=11),
        # images of several requests through the up projection
        _lora("lora-images", 4, 1024, 1152, 3072, 12288, 3, 16, 64, "f16", pick=12),
    ]


def _log(rng, lo, hi):
    return int(round(lo * (hi / lo) ** rng.random()))


def draw(rng):
    kind = rng.choice(["prompt", "paged", "lora"])
    pick = rng.randrange(1 << 20)
    heads, kv_heads = rng.choice([(32, 8), (24, 24), (28, 4), (16, 2), (12, 4), (20, 4), (8, 1)])
    dim, dtype = rng.choice([128, 128, 64]), rng.choice(["f16", "bf16"])
    if kind == "prompt":
        hi = _log(rng, 1, 10000)
        n = _log(rng, 1, max(1, min(200, int(1e8 / hi ** 2), 40000 // hi)))
        return _prompt(None, n, max(1, hi // rng.choice([1, 2, 8, 50])), hi, heads, kv_heads, dim, dtype,
                       rng.random() < 0.75, rng.random() < 0.5, pick)
    if kind == "paged":
        hi = _log(rng, 1, 65536)
        n = _log(rng, 1, max(1, min(200, 250000 // hi)))
        q_hi = rng.choice([1, 1, _log(rng, 1, max(1, min(hi, 1024, int(8e8 / (n * hi * heads)))))])
        ctx_lo = max(q_hi, hi // rng.choice([1, 3, 20]))
        return _paged(None, n, ctx_lo, hi, max(1, q_hi // rng.choice([1, 4])), q_hi, rng.choice([16, 32, 64, 128]),
                      heads, kv_heads, dim, dtype, pick)
    in_dim, out_dim = rng.choice([(3072, 3072), (3072, 9216), (9216, 3072), (2560, 4096), (4096, 1024), (7680, 3072),
                                  (3072, 12288), (96, 1000), (2080, 1330)])
    hi = _log(rng, 1, 1500)
    n = _log(rng, 1, max(1, min(128, 4000 // hi)))
    rank = _log(rng, 1, 128)
    return _lora(None, n, max(1, hi // rng.choice([1, 3, 20])), hi, in_dim, out_dim, rng.randrange(1, n + 2),
                 max(1, rank // rng.choice([1, 4])), rank, rng.choice(["f16", "f32"]), pick)


def _lengths(case, lo, hi, salt):
    """n lengths in [lo, hi], the longest exactly hi."""
    r = random.Random(case["pick"] * 16 + salt)
    v = [r.randint(lo, hi) for _ in range(case["n"])]
    v[r.randrange(case["n"])] = hi
    return v


def _cumulated(lens):
    cu = [0]
    for x in lens:
        cu.append(cu[-1] + x)
    return cu


def _paged_lengths(case):
    q = _lengths(case, case["q_lo"], case["q_hi"], 0)
    ctx = _lengths(case, case["ctx_lo"], case["ctx_hi"], 1)
    return q, [max(a, b) for a, b in zip(q, ctx)]


def _adapters(case):
    """(rank of each adapter, scale of each, adapter of each request: -1 = none)."""
    r = random.Random(case["pick"] * 16 + 5)
    ranks = [r.randint(case["rank_lo"], case["rank_hi"]) for _ in range(case["slots"])]
    ranks[0] = case["rank_hi"]
    scales = [r.choice([0.5, 1.0, 2.0]) * 0.7 for _ in ranks]
    of = [i % case["slots"] for i in range(case["n"])]
    r.shuffle(of)
    if case["n"] > 4:
        of[r.randrange(case["n"])] = -1
    return ranks, scales, of


# ----------------------------------------------------------------- prepare
def _ints(v):
    return torch.tensor(v, dtype=torch.int32, device=DEV)


def _randn(g, *shape, dtype=torch.float32, std=1.0):
    return (torch.randn(*shape, device=DEV, generator=g) * std).to(dtype)


def prepare(case, seed):
    g = torch.Generator(device=DEV)
    g.manual_seed(seed)
    return {"prompt": _prepare_prompt, "paged": _prepare_paged, "lora": _prepare_lora}[case["kind"]](case, g)


def _prepare_prompt(c, g):
    lens = _lengths(c, c["lo"], c["hi"], 0)
    cu, dt = _cumulated(lens), DTYPES[c["dtype"]]
    t, h, hk, d = cu[-1], c["heads"], c["kv_heads"], c["dim"]
    s = {"case": c, "cu": _ints(cu), "max_len": max(lens), "scale": d ** -0.5}
    if c["fused"]:
        qkv = _randn(g, t, (h + 2 * hk) * d, dtype=dt, std=1.2)
        s["q"], s["k"], s["v"] = (x.unflatten(1, (-1, d)) for x in qkv.split([h * d, hk * d, hk * d], 1))
    else:
        s["q"], s["k"], s["v"] = (_randn(g, t, x, d, dtype=dt, std=1.2) for x in (h, hk, hk))
    return s


def _prepare_paged(c, g):
    q, ctx = _paged_lengths(c)
    dt, page = DTYPES[c["dtype"]], c["page"]
    h, hk, d = c["heads"], c["kv_heads"], c["dim"]
    cu = _cumulated(q)
    per = [-(-x // page) for x in ctx]
    width = max(per)
    total = sum(per) + 3
    r = random.Random(c["pick"])
    free = list(range(total))
    r.shuffle(free)  # pages in the order of their allocation by many requests
    table, at = [], 0
    for k in per:
        table.append(free[at:at + k] + [0] * (width - k))
        at += k
    return {"case": c, "cu": _ints(cu), "ctx": _ints(ctx), "table": _ints(table), "max_q": max(q),
            "max_ctx": max(ctx), "scale": d ** -0.5,
            "k_cache": _randn(g, total, page, hk, d, dtype=dt, std=1.2),
            "v_cache": _randn(g, total, page, hk, d, dtype=dt, std=1.2),
            "q": _randn(g, cu[-1], h, d, dtype=dt, std=1.2), "k": _randn(g, cu[-1], hk, d, dtype=dt, std=1.2),
            "v": _randn(g, cu[-1], hk, d, dtype=dt, std=1.2)}


def _prepare_lora(c, g):
    lens = _lengths(c, c["lo"], c["hi"], 0)
    ranks, scales, of = _adapters(c)
    cu, k, n, r = _cumulated(lens), c["in_dim"], c["out_dim"], max(ranks)
    packed = torch.empty(n, k // BLOCK, BLOCK_BYTES, dtype=torch.uint8, device=DEV)
    packed[..., 2:] = torch.randint(0, 256, (n, k // BLOCK, 4), device=DEV, generator=g, dtype=torch.uint8)
    packed[..., :2] = _randn(g, n, k // BLOCK, 1, std=0.02).abs().half().view(torch.uint8)
    live = (torch.arange(r, device=DEV) < _ints(ranks)[:, None])
    s = {"case": c, "cu": _ints(cu), "max_len": max(lens), "of": _ints(of), "packed": packed,
         "x": _randn(g, cu[-1], k, dtype=torch.float16),
         "down": _randn(g, len(ranks), r, k, std=k ** -0.5).mul(live[:, :, None]).half(),
         "up": _randn(g, len(ranks), n, r, std=0.3).mul(live[:, None, :]).half(),
         "scales": torch.tensor(scales, device=DEV)}
    if own:
        bb = _bb()
        s["w"] = bb.B1Weight(packed.cpu().numpy(), n, k)
        s["lora"] = bb.LoraSet(n, k, r, len(ranks))
        for i, rank in enumerate(ranks):
            s["lora"].set(i, s["down"][i, :rank].contiguous(), s["up"][i, :, :rank].contiguous(), scales[i])
    return s


# --------------------------------------------------------------------- run
def run(state):
    kind = state["case"]["kind"]
    if own:
        return {"prompt": _own_prompt, "paged": _own_paged, "lora": _own_lora}[kind](state)
    return {"prompt": _plain_prompt, "paged": _plain_paged, "lora": _plain_lora}[kind](state)


def _own_prompt(s):
    out = torch.empty(s["q"].shape, dtype=s["q"].dtype, device=DEV)
    _bb().prompt_attention(s["q"], s["k"], s["v"], s["cu"], out, scale=s["scale"], causal=s["case"]["causal"])
    return out


def _own_paged(s):
    bb = _bb()
    out = torch.empty_like(s["q"])
    bb.paged_append(s["k"], s["v"], s["k_cache"], s["v_cache"], s["table"], s["cu"], s["ctx"])
    bb.paged_attention(s["q"], s["k_cache"], s["v_cache"], s["table"], s["cu"], s["ctx"], s["max_ctx"], out,
                       scale=s["scale"])
    return {"out": out, "k_cache": s["k_cache"], "v_cache": s["v_cache"]}


def _own_lora(s):
    bb, c = _bb(), s["case"]
    out = torch.empty(s["x"].shape[0], c["out_dim"], dtype=DTYPES[c["out"]], device=DEV)
    bb.b1_gemm_lora(s["x"], s["w"], bb.BONSAI_EPI_F16 if c["out"] == "f16" else bb.BONSAI_EPI_F32, out, s["lora"],
                    s["cu"], s["of"])
    return out


def _rows(cu, longest, total):
    """Packed rows as [n][longest] indices, and which of them are real."""
    pos = torch.arange(longest, device=DEV)
    real = pos < (cu[1:] - cu[:-1])[:, None]
    return (cu[:-1, None] + pos).clamp(max=total - 1), real


def _plain_softmax(scores, keep):
    scores.masked_fill_(~keep, float("-inf"))
    top = scores.amax(-1, keepdim=True)
    scores.sub_(top.masked_fill_(top == float("-inf"), 0.0)).exp_()
    total = scores.sum(-1, keepdim=True)
    return scores.div_(total.masked_fill_(total == 0, 1.0))


def _plain_attention(q, k, v, keep, scale):
    """q [n][i][H][D], k and v [n][j][Hk][D], keep [n][i][j] -> [n][i][H][D], all f32."""
    hk = k.shape[2]
    q = q.unflatten(2, (hk, -1)).permute(0, 2, 3, 1, 4).flatten(2, 3)  # n Hk (g i) D
    scores = torch.matmul(q, k.permute(0, 2, 3, 1)).mul_(scale).unflatten(2, (-1, keep.shape[1]))
    p = _plain_softmax(scores, keep[:, None, None]).flatten(2, 3)
    out = torch.matmul(p, v.transpose(1, 2))
    return out.unflatten(2, (-1, keep.shape[1])).permute(0, 3, 1, 2, 4).flatten(2, 3)


def _plain_prompt(s):
    q, k, v = s["q"].float(), s["k"].float(), s["v"].float()
    at, real = _rows(s["cu"], s["max_len"], q.shape[0])
    keep = real[:, None, :].expand(-1, s["max_len"], -1)
    if s["case"]["causal"]:
        pos = torch.arange(s["max_len"], device=DEV)
        keep = keep & (pos[:, None] >= pos)
    return _plain_attention(q[at], k[at], v[at], keep, s["scale"])[real].to(s["q"].dtype)


def _plain_paged(s):
    cu, ctx, table, page = s["cu"], s["ctx"], s["table"], s["case"]["page"]
    at, real = _rows(cu, s["max_q"], s["q"].shape[0])
    pos = torch.arange(s["max_q"], device=DEV) + (ctx - (cu[1:] - cu[:-1]))[:, None]  # place in the sequence
    slot = table.gather(1, (pos // page).clamp(max=table.shape[1] - 1).long())[real].long(), (pos % page)[real]
    s["k_cache"][slot] = s["k"]
    s["v_cache"][slot] = s["v"]
    k = s["k_cache"][table.long()].flatten(1, 2).float()
    v = s["v_cache"][table.long()].flatten(1, 2).float()
    seen = torch.arange(k.shape[1], device=DEV)
    keep = (seen <= pos[:, :, None]) & (seen < ctx[:, None, None])
    out = _plain_attention(s["q"].float()[at], k, v, keep, s["scale"])[real].to(s["q"].dtype)
    return {"out": out, "k_cache": s["k_cache"], "v_cache": s["v_cache"]}


def _plain_weight(packed, dtype):
    scale = packed[..., :2].contiguous().view(torch.float16).to(dtype)
    bits = (packed[..., 2:, None] >> torch.arange(8, device=DEV, dtype=torch.uint8)) & 1
    return ((bits.flatten(2).to(dtype) * 2 - 1) * scale).flatten(1)


def _plain_lora(s):
    x = s["x"].float()
    y = torch.matmul(x, _plain_weight(s["packed"], torch.float32).t())
    at, real = _rows(s["cu"], s["max_len"], x.shape[0])
    of = s["of"].clamp(min=0).long()
    scale = s["scales"][of] * (s["of"] >= 0)
    low = torch.matmul(x[at], s["down"][of].float().transpose(1, 2)) * scale[:, None, None]
    return (y + torch.matmul(low, s["up"][of].float().transpose(1, 2))[real]).to(DTYPES[s["case"]["out"]])


# -------------------------------------------------------------------- work
def work(case):
    c = case
    if c["kind"] == "prompt":
        lens = _lengths(c, c["lo"], c["hi"], 0)
        pairs = sum(x * (x + 1) // 2 if c["causal"] else x * x for x in lens)
        return {"bytes": sum(lens) * c["dim"] * 2 * (2 * c["heads"] + 2 * c["kv_heads"]),
                "flops": 4.0 * pairs * c["heads"] * c["dim"]}
    if c["kind"] == "paged":
        q, ctx = _paged_lengths(c)
        pairs = sum(a * b - a * (a - 1) // 2 for a, b in zip(q, ctx))
        # cached keys and values once; new ones read and written; queries, outputs
        return {"bytes": c["dim"] * 2 * (2 * c["kv_heads"] * (sum(ctx) + sum(q)) + 2 * c["heads"] * sum(q)),
                "flops": 4.0 * pairs * c["heads"] * c["dim"]}
    lens = _lengths(c, c["lo"], c["hi"], 0)
    ranks, _, of = _adapters(c)
    t, k, n = sum(lens), c["in_dim"], c["out_dim"]
    used = sum(ranks[i] for i in set(of) if i >= 0)
    low = sum(x * ranks[i] for x, i in zip(lens, of) if i >= 0)
    return {"bytes": t * k * 2 + n * k // BLOCK * BLOCK_BYTES + used * (k + n) * 2 + t * n * (2 if c["out"] == "f16" else 4),
            "flops": 2.0 * t * k * n + 2.0 * low * (k + n)}


# ------------------------------------------------------------------- exact
def _exact_rows(q, k, v, scale, first):
    """softmax(q k' scale) v of one sequence in f64, head by head; query i sees the keys up to first + i."""
    out = torch.empty(q.shape, dtype=torch.float64, device=DEV)
    group = q.shape[1] // k.shape[1]
    for h in range(q.shape[1]):
        a = (q[:, h].double() @ k[:, h // group].double().T) * scale
        if first is not None:
            a = a.masked_fill(torch.ones_like(a, dtype=torch.bool).triu(first + 1), float("-inf"))
        out[:, h] = torch.softmax(a, 1) @ v[:, h // group].double()
    return out


def exact(case, seed):
    s = prepare(case, seed)
    if case["kind"] == "prompt":
        cu = s["cu"].tolist()
        return torch.cat([_exact_rows(s["q"][a:b], s["k"][a:b], s["v"][a:b], s["scale"], 0 if case["causal"] else None)
                          for a, b in zip(cu, cu[1:])])
    if case["kind"] == "paged":
        cu, outs = s["cu"].tolist(), []
        for i, length in enumerate(s["ctx"].tolist()):
            a, b = cu[i], cu[i + 1]
            pages = s["table"][i, :-(-length // case["page"])].long()
            # the cached tokens before the new ones, then the new ones
            k = torch.cat([s["k_cache"][pages].flatten(0, 1)[:length - (b - a)], s["k"][a:b]])
            v = torch.cat([s["v_cache"][pages].flatten(0, 1)[:length - (b - a)], s["v"][a:b]])
            outs.append(_exact_rows(s["q"][a:b], k, v, s["scale"], length - (b - a)))
        return {"out": torch.cat(outs), "k_cache": None, "v_cache": None}
    raw = s["packed"].cpu().numpy()
    import numpy as np
    scale = np.ascontiguousarray(raw[..., :2]).view(np.float16).astype(np.float64)
    sign = np.unpackbits(np.ascontiguousarray(raw[..., 2:]), axis=-1, bitorder="little").astype(np.int8)
    weight = (torch.from_numpy(sign).to(DEV).double().mul_(2).sub_(1) * torch.from_numpy(scale).to(DEV)).flatten(1)
    x = s["x"].double()
    y = x @ weight.T
    cu = s["cu"].tolist()
    for i, slot in enumerate(s["of"].tolist()):
        if slot >= 0:
            rows = slice(cu[i], cu[i + 1])
            y[rows] += float(s["scales"][slot]) * ((x[rows] @ s["down"][slot].double().T) @ s["up"][slot].double().T)
    return y
