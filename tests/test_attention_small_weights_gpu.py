"""Many keys of a small weight each beside one that dominates: together they count.

One key has weight 1, n others 2^-25.4, below half of f16's smallest step; the
values are 0 for the one and 1 for the others, so the output is w / (1 + w),
w = n 2^-25.4.  Bound: f16 weights are rounded to 2^-11 relative or, below
2^-14 of what the largest may be (2^15 with the moving maximum's slack of 2^8
and no key above it: 2^7 times the weight), to 2^-25 / 2^7 absolute; the
exponential and its argument (|x| < 64) are off by 2^-17 relative; the output
by 2^-11 relative."""
import pytest
import torch

from test_text_attention_gpu import bf16, f16, ints

pytestmark = pytest.mark.gpu

UNIT = {f16: 2.0 ** -11, bf16: 2.0 ** -8}


@pytest.mark.parametrize("dtype", [f16, bf16], ids=["f16", "bf16"])
@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("paged", [True, False], ids=["paged", "prompt"])
def test_small_weights_count_together(gpu, dtype, dim, paged):
    n, big = 65535, 25.4
    k, v = torch.zeros(n + 1, 1, dim, device="cuda", dtype=dtype), torch.ones(n + 1, 1, dim, device="cuda", dtype=dtype)
    q = torch.zeros(1, 4, dim, device="cuda", dtype=dtype)
    k[5, 0, 0], v[5] = 8.0, 0.0
    q[..., 0] = 2.0
    scale = big * 0.6931471805599453 / 16.0
    w = n * 2.0 ** -big
    want = w / (1 + w)
    if paged:
        table = ints([list(range((n + 1) // 64))])
        out = torch.empty_like(q)
        # max_ctx 0: one part, in which the dominating key is
        gpu.paged_attention(q, k.view(-1, 64, 1, dim), v.view(-1, 64, 1, dim), table, ints([0, 1]), ints([n + 1]), 0, out,
                            scale=scale)
    else:
        q = torch.cat([torch.zeros(n, 4, dim, device="cuda", dtype=dtype), q])
        out = torch.empty_like(q)
        gpu.prompt_attention(q, k, v, ints([0, n + 1]), out, scale=scale, causal=True)
    u = UNIT[dtype]
    bound = want * (2 * u + 2.0 ** -17) + (n * 2.0 ** -32 if dtype is f16 else 0.0) + 2.0 ** -25
    assert float((out[-1].double() - want).abs().max()) <= bound
