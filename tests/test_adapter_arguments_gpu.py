"""Arguments that b1_gemm_lora refuses before anything is launched: a gate that the
epilogue could not read."""
import pytest
import torch

from test_lora_gpu import Problem, ints, within

pytestmark = pytest.mark.gpu


def test_gate(gpu):
    p = Problem(gpu, 64, 64, [16])
    x, cu, slots = p.x(4), ints([0, 4]), ints([0])
    good = torch.randn(64, device="cuda", generator=p.g)
    out = torch.zeros(4, 64, device="cuda")
    for gate in (good.cpu(), good.half(), good[:63].contiguous(), torch.randn(128, device="cuda")[::2], good.double()):
        with pytest.raises(gpu.BonsaiError, match="gate"):
            gpu.b1_gemm_lora(x, p.w, gpu.BONSAI_EPI_RESID, out, p.lora, cu, slots, gate=gate)
    torch.cuda.synchronize()
    assert (out == 0).all()
    y, b = p.accumulators(x, [0, 4], [0])
    gpu.b1_gemm_lora(x, p.w, gpu.BONSAI_EPI_RESID, out, p.lora, cu, slots, gate=good)
    within(out, good.double() * y, good.abs().double() * b + 2.0 ** -23 * (good.double() * y).abs())
