"""Sequences of up to 2^31 - 1 places over a quantised cache: one page of 65536 slots at every place
of the table, so that every slot counts 2^15 times, those past the length once less.

The sums are f32 over n = 2^31 / 2^17 weights in a row at most (a lane of the 296 CTAs' warps has two keys
of 16, or a thread 64 of a block): their rounding is n 2^-24 = 2^-10 of the sum at worst, the output's
as much of sum_j p_j |v_j|.  Counting only part of the keys gives something else: over the first 128 alone
the outputs are ten times as large as over all of them.
"""
import pytest
import torch

import quant_ref as qr
from test_quant_attention_gpu import caches_of
from test_text_attention_gpu import bf16, f16, ints, randn

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("new", [1, 33])
@pytest.mark.parametrize("ctx", [2 ** 31 - 1, 2 ** 31 - 60, 2 ** 31 - 700, 2 ** 30 + 5])
@pytest.mark.parametrize("dtype,fmt", [(f16, "i4"), (bf16, "i8")])
def test_far_places(gpu, new, ctx, dtype, fmt):
    page, dim = 1 << 16, 64
    k, v = caches_of(gpu, 3, 1, page, 1, dim, dtype, fmt)
    table = torch.zeros(1, (1 << 31) // page, dtype=torch.int32, device="cuda")
    q, out = randn(5, new, 2, dim, dtype=dtype), torch.full((new, 2, dim), 7.0, dtype=dtype, device="cuda")
    gpu.paged_attention_quant(q, k, v, table, ints([0, new]), ints([ctx]), ctx, out, max_q=new)
    torch.cuda.synchronize()
    assert gpu.device_error() == 0
    kk, vv = (qr.values(c.codes, c.scales, fmt)[0, :, 0] for c in (k, v))
    for i in range(new):
        seen = ctx - new + i + 1
        count = seen // page + (torch.arange(page, device="cuda") < seen % page).double()
        w = torch.exp(q[i].double() @ kk.T * dim ** -0.5) * count
        w /= w.sum(1, keepdim=True)
        off = (out[i].double() - w @ vv).abs()
        assert bool((off <= 2.0 ** -8 * (w @ vv).abs() + 2 * 2.0 ** -10 * (w @ vv.abs())).all()), float(off.max())
