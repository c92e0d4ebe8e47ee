"""bonsai_paged_attention_quant rounds to 16 bits once, at the output: the softmax weights
go to their product as two 16-bit values, within r of what they are (r = 2^-16 in bf16,
2^-22 in f16: each of the two roundings leaves at most the unit roundoff u).

Error bound of an output element, p the exact weights: u |out| for the output's rounding,
and (r + 2 e) * sum_j p_j |v_j| with e as in test_text_attention_gpu.py (f32 dot products,
the exponential), and as much of u again since the rounding is of the value so found.  With
weights rounded to 16 bits u itself would stand in r's place: values of both signs make
sums that are small beside sum_j p_j |v_j|, where that is far outside.
"""
import pytest
import torch

from test_quant_attention_gpu import cached_rows, caches_of, tables
from test_text_attention_gpu import UNIT, bf16, cumulated, f16, ints, randn, ref_rows

pytestmark = pytest.mark.gpu

LEFT = {f16: 2.0 ** -22, bf16: 2.0 ** -16}


@pytest.mark.parametrize("lens,ctx", [([1, 1], [20, 900]), ([3, 40], [50, 60]), ([200, 1], [3000, 64])], ids=str)
@pytest.mark.parametrize("dtype", [f16, bf16], ids=["f16", "bf16"])
@pytest.mark.parametrize("fmt", ["i8", "i4"])
@pytest.mark.parametrize("dim", [64, 128])
def test_one_rounding(gpu, lens, ctx, dtype, fmt, dim):
    table, total = tables(ctx, 16)
    k, v = caches_of(gpu, 2, total, 16, 2, dim, dtype, fmt, std=0.3)
    q, cu = randn(11, sum(lens), 8, dim, dtype=dtype, std=0.3), cumulated(lens)
    out = torch.full_like(q, 7.0)
    gpu.paged_attention_quant(q, k, v, table, ints(cu), ints(ctx), max(ctx), out, max_q=max(lens))
    torch.cuda.synchronize()
    u = UNIT[dtype]
    for s, row in enumerate(table.tolist()):
        kk, vv = (cached_rows(c, row, ctx[s], dtype) for c in (k, v))
        part = q[cu[s]:cu[s + 1]]
        ref, _ = ref_rows(part, kk, vv, ctx[s] - lens[s], dim ** -0.5)
        weight, _ = ref_rows(part, kk, vv.abs(), ctx[s] - lens[s], dim ** -0.5)  # sum_j p_j |v_j|
        mag = torch.einsum("ihd,jhd->hij", part.double().abs(), kk.abs().repeat_interleave(4, 1)).max() * dim ** -0.5
        e = 2 * (dim + 8) * 2.0 ** -24 * float(mag) + 2.0 ** -20
        over = (out[cu[s]:cu[s + 1]].double() - ref).abs() - u * ref.abs() - (1 + u) * (LEFT[dtype] + 2 * e) * weight
        assert float(over.max()) <= 0.0, f"off by {float(over.max())} more than the bound"
