"""TextLayer over a quantised cache against one over 16 bits with the same weights: what the cache
holds is the plain quantisation of the 16-bit cache's rows, at the places that the lengths say, and a step
behind it gives what attention in 16 bits over those very values gives (the layer's parity bar: the
two round differently)."""
import numpy as np
import pytest
import torch

import quant_ref as qr
from bonsai_b200 import text_layer
from bonsai_b200.text_layer import generate, run_both_ways
from test_text_generate_gpu import HIDDEN, PROMPTS, VOCAB, ints, model

pytestmark = pytest.mark.gpu

LENS, PAGES = [37, 5, 64], 5
SLOTS = [-1] * 3


def cum(v):
    return ints(np.cumsum([0] + list(v)).tolist())


def table(seed):
    return torch.randperm(PAGES * 3, generator=torch.Generator().manual_seed(seed)).int().cuda().view(3, PAGES)


def rows(cache, pages, length):
    """The first `length` places of a 16-bit cache."""
    return torch.cat([cache[i] for i in pages])[:length]


def read(bb, layer, t, lens):
    """Keys and values of a quantised cache, packed."""
    k, v = (torch.empty(sum(lens), layer.kv_heads, 128, dtype=torch.float16, device="cuda") for _ in range(2))
    bb.paged_read_quant(layer.k_cache, layer.v_cache, t, cum(lens), None, k, v)
    return k, v


@pytest.mark.parametrize("cache", ["i8", "i4"])
def test_the_cache_holds_the_quantised_rows(gpu, cache):
    codes, plain = model(gpu, cache)[0], model(gpu, "f16")[0]
    x = torch.randn(sum(LENS), HIDDEN, device="cuda", generator=torch.Generator(device="cuda").manual_seed(1))
    for layer, seed in ((codes, 1), (plain, 2)):
        layer.forward(x.clone(), cum(LENS), ints(LENS), table(seed), ints(SLOTS))
    got = read(gpu, codes, table(1), LENS)
    for g, c in zip(got, (plain.k_cache, plain.v_cache)):
        want = torch.cat([rows(c, p, n) for p, n in zip(table(2).tolist(), LENS)])
        n, e = qr.quantise(want, cache)
        assert torch.equal(g.double(), qr.values(qr.codes_of(n, cache), e, cache))


@pytest.mark.parametrize("cache", ["i8", "i4"])
@pytest.mark.parametrize("new", [1, 3, 20])
def test_a_step_over_the_cached_values(gpu, cache, new, monkeypatch):
    codes, plain = model(gpu, cache)[0], model(gpu, "f16")[0]
    g = torch.Generator(device="cuda").manual_seed(1)
    lens = [x - 1 for x in LENS]
    total = [x + new for x in lens]
    tc, tp = (torch.arange(3 * 6, dtype=torch.int32, device="cuda").view(3, 6).flip(d).contiguous() for d in (0, 1))
    codes.forward(torch.randn(sum(lens), HIDDEN, device="cuda", generator=g), cum(lens), ints(lens), tc, ints(SLOTS))
    x = torch.randn(3 * new, HIDDEN, device="cuda", generator=g)
    got = codes.forward(x.clone(), cum([new] * 3), ints(total), tc, ints(SLOTS), max_ctx=max(total), max_q=new)
    k, v = read(gpu, codes, tc, total)
    gpu.paged_append(k, v, plain.k_cache, plain.v_cache, tp, cum(total), ints(total))
    monkeypatch.setattr(text_layer.bb, "paged_append", lambda *a, **kw: None)  # the values are there, quantised
    want = plain.forward(x.clone(), cum([new] * 3), ints(total), tp, ints(SLOTS), max_ctx=max(total), max_q=new)
    a, b = got.double().flatten(), want.double().flatten()
    assert float(a @ b / (a.norm() * b.norm())) >= 0.9999
    assert float((a - b).abs().max() / a.square().mean().sqrt()) <= 1e-2
    # without the cache's part the outputs are something else
    assert float((a - x.double().flatten()).abs().max() / a.square().mean().sqrt()) > 0.1


@pytest.mark.parametrize("cache", ["i8", "i4"])
def test_generated_tokens_follow_from_the_cached_text(gpu, cache):
    """Greedy tokens are the largest logits of single tokens fed by hand, in pages of another order."""
    layer, embedding, head = model(gpu, cache)
    steps, n = 5, len(PROMPTS)
    tokens = generate(layer, embedding, head, PROMPTS, steps, torch.zeros(steps, n, device="cuda"), temperature=torch.zeros(n, device="cuda"))
    layer, _, _ = model(gpu, cache)
    lens = [len(p) for p in PROMPTS]
    t = torch.arange(63, 63 - n * 4, -1, dtype=torch.int32, device="cuda").view(n, 4)
    h = layer.forward(embedding[ints(sum(PROMPTS, [])).long()].float(), cum(lens), ints(lens), t, ints(SLOTS))[(cum(lens)[1:] - 1).long()]
    for i in range(steps):
        logits = torch.empty(n, VOCAB, device="cuda")
        gpu.b1_gemm(h.half().contiguous(), head, gpu.BONSAI_EPI_F32, logits)
        chosen = logits.gather(1, tokens[:, i:i + 1].long())[:, 0]
        assert bool((chosen >= logits.amax(1) - 1e-2 * logits.square().mean(1).sqrt()).all())
        ctx = [x + i + 1 for x in lens]
        h = layer.forward(embedding[tokens[:, i].long()].float(), cum([1] * n), ints(ctx), t, ints(SLOTS), max_ctx=max(ctx), max_q=1)


@pytest.mark.parametrize("cache", ["i8", "i4"])
def test_nothing_is_read_that_was_not_written(gpu, cache):
    """Between its two ways run_both_ways makes every cached block a NaN: what comes after is finite."""
    whole, parts = run_both_ways(cache=cache)
    assert bool(whole.isfinite().all()) and bool(parts.isfinite().all())
