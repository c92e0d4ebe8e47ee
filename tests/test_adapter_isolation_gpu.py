"""Values that are not finite stay with the request that brings them.  Both forms of
bonsai_b1_gemm_lora and both tile sizes, against f64."""
import numpy as np
import pytest
import torch

from test_lora_gpu import Problem, kernel  # noqa: F401 (a fixture)

pytestmark = pytest.mark.gpu

INF = float("inf")
LENS = [([1, 1, 1, 1], [0, 1, -1, 0]), ([40, 9, 20, 300, 17], [1, 0, -1, 1, 0]), ([300, 70, 200], [1, 0, 1])]


def pattern(y):
    return torch.where(y.isnan(), 2, torch.where(y.isinf(), y.sign(), 0)).int()


@pytest.mark.parametrize("lens,slots", LENS, ids=str)
@pytest.mark.parametrize("rank", [1, 3, 16])
def test_infinite_x(gpu, kernel, lens, slots, rank):  # noqa: F811
    """W x and the adapter's part are infinite with signs of their own; ranks that
    the adapter does not have make no NaN of them."""
    p = Problem(gpu, 256, 512, [rank, 4], seed=rank)
    # B's columns have one sign each, as A's row has where x is infinite, so that B low is infinite in one direction
    p.up[0] = p.up[0].abs()
    p.down[0][:, 77] = p.down[0][:, 77].abs()
    p.up[0][:, 0] = p.up[0][:, 0].bfloat16().half()  # exact in one piece
    p.lora.set(0, p.down[0], p.up[0], p.scale[0])
    cu = np.cumsum([0] + lens).tolist()
    x = p.x(cu[-1])
    clean = p.run(x, cu, slots, gpu.BONSAI_EPI_F32, torch.empty(cu[-1], 256, device="cuda"))
    at = cu[slots.index(0)]
    x[at, 77] = INF
    out = p.run(x, cu, slots, gpu.BONSAI_EPI_F32, torch.empty(cu[-1], 256, device="cuda"))
    y = x[at].double() @ p.dense.double().T + p.scale[0] * (x[at].double() @ p.down[0].double().T) @ p.up[0].double().T
    assert y.isinf().any() and y.isnan().any()
    assert torch.equal(pattern(out[at]), pattern(y))
    keep = [i for i in range(cu[-1]) if i != at]
    assert torch.equal(out[keep], clean[keep])
