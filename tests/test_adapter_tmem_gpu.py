"""Adapters of high rank with more CTAs than SMs, alone and beside attention whose
key split is a cluster (see test_adapter_tmem_cpu).  Against f64."""
import numpy as np
import pytest
import torch

from test_lora_gpu import Problem, check_f32, ints, within
from test_text_attention_gpu import f16, make_cache, randn, run_paged

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("rank", [65, 80, 96, 128])
def test_more_ctas_than_sms(gpu, rank):
    p = Problem(gpu, 256, 3072, [rank, 7], max_rank=rank, seed=rank)
    lens = [1300, 700, 1900, 30, 2570]
    check_f32(p, p.x(sum(lens)), np.cumsum([0] + lens).tolist(), [0, 1, 0, -1, 0])


@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("rank", [16, 48, 80, 128])
def test_beside_attention_on_another_stream(gpu, dim, rank):
    p = Problem(gpu, 256, 1024, [rank], max_rank=rank, seed=rank)
    x, cu, slots = p.x(3000), ints([0, 3000]), ints([0])
    want = torch.empty(3000, 256, device="cuda")
    gpu.b1_gemm_lora(x, p.w, gpu.BONSAI_EPI_F32, want, p.lora, cu, slots)
    within(want, *p.accumulators(x, [0, 3000], [0]))
    ctx = [6000, 2000]
    kc, vc, table = make_cache(40, ctx, 16, 2, dim, f16)
    q, cq, cx = randn(41, 2, 16, dim), ints([0, 1, 2]), ints(ctx)
    attn = run_paged(gpu, q, kc, vc, table, [0, 1, 2], ctx, 16)
    a, b = torch.cuda.Stream(), torch.cuda.Stream()
    outs = [(torch.empty_like(want), torch.empty_like(attn)) for _ in range(8)]
    torch.cuda.synchronize()
    for y, o in outs:
        gpu.b1_gemm_lora(x, p.w, gpu.BONSAI_EPI_F32, y, p.lora, cu, slots, stream=a)
        for _ in range(3):
            gpu.paged_attention(q, kc, vc, table, cq, cx, max(ctx), o, stream=b)
    torch.cuda.synchronize()
    assert all(torch.equal(y, want) and torch.equal(o, attn) for y, o in outs)
