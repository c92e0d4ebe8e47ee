"""Adapters whose low-rank values are far from one: small scales beside large B,
values past f16's largest, values near f32's.  Both forms of
bonsai_b1_gemm_lora, against f64 with the bounds of test_lora_gpu."""
import numpy as np
import pytest
import torch

from test_lora_gpu import Problem, check_f32

pytestmark = pytest.mark.gpu


class Ranged(Problem):
    up_std = 0.3

    def put(self, slot, rank, scale, host=False):
        d = (torch.randn(rank, self.k, device="cuda", generator=self.g) * self.k ** -0.5).half()
        u = (torch.randn(self.n, rank, device="cuda", generator=self.g) * self.up_std).half()
        self.down[slot], self.up[slot], self.scale[slot] = d, u, self.scales[slot]
        self.lora.set(slot, d, u, self.scales[slot])


@pytest.mark.parametrize("lens", [[1, 1, 1], [40, 300, 9], [300, 70]], ids=str)
@pytest.mark.parametrize("scales,up", [((1e-5, 3e-5), 1e3), ((1e-8, 1e-3), 1e4), ((3e6, 1.0), 0.3), ((1e25, 1e5), 1e-6),
                                       ((-1e30, 1e-30), 1e3)], ids=str)
def test_any_magnitude(gpu, lens, scales, up):
    class P(Ranged):
        pass
    P.scales, P.up_std = [float(np.float32(s)) for s in scales], up
    p = P(gpu, 300, 320, [16, 40])
    check_f32(p, p.x(sum(lens)), np.cumsum([0] + lens).tolist(), [0, 1, 0][:len(lens)])


def test_the_request_does_not_depend_on_its_batch(gpu):
    """Eight tokens of one request alone (few) and with a long neighbour (many)
    are within the sum of both forms' bounds of each other."""
    class P(Ranged):
        scales, up_std = [2e5, 1e-5], 30.0
    p = P(gpu, 256, 512, [16, 16])
    x = p.x(208)
    a = p.run(x[:8], [0, 8], [0], gpu.BONSAI_EPI_F32, torch.empty(8, 256, device="cuda"))
    b = p.run(x, [0, 8, 208], [0, 1], gpu.BONSAI_EPI_F32, torch.empty(208, 256, device="cuda"))[:8]
    _, bound = p.accumulators(x[:8], [0, 8], [0])
    assert a.isfinite().all() and float(((a - b).double().abs() - 2 * bound).max()) <= 0
