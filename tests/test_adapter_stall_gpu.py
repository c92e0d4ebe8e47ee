"""The bounded waits of a projection with adapters, made to run out by the test hook
(bonsai_debug_stall_next_gemm): the launch runs the one-CTA kernel with its
load warp idle, whichever form and tile size the call would have taken; the
code is reported, nothing is written, and the next call is right."""
import numpy as np
import pytest
import torch

from test_lora_gpu import Problem, check_f32, ints

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("lens", [[1, 1, 1], [300, 5, 700]], ids=str)
def test_stalled_launch_reports_and_recovers(gpu, monkeypatch, lens):
    monkeypatch.setenv("BONSAI_B1_KERNEL", "pair")  # long requests: laid out for tiles of 256 tokens
    p = Problem(gpu, 512, 256, [16, 40])
    cu, slots = np.cumsum([0] + lens).tolist(), [1, 0, 1]
    x, out = p.x(cu[-1]), torch.full((cu[-1], 512), float("nan"), device="cuda")
    assert gpu.device_error() == 0
    gpu.check(gpu.lib().bonsai_debug_stall_next_gemm(), "bonsai_debug_stall_next_gemm")
    gpu.b1_gemm_lora(x, p.w, gpu.BONSAI_EPI_F32, out, p.lora, ints(cu), ints(slots))
    assert gpu.device_error() in (1, 2, 3, 4)
    assert gpu.device_error() == 0 and out.isnan().all()
    check_f32(p, x, cu, slots)
