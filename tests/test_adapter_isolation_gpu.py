"""Values that are not finite stay with the request that brings them: in an
adapter's up or down matrix, and in x.  Both forms of bonsai_b1_gemm_lora and
both tile sizes, against f64 with the bounds of test_lora_gpu, and bit by bit
against the same call with an adapter that is finite."""
import numpy as np
import pytest
import torch

from test_lora_gpu import Problem, kernel, within  # noqa: F401 (a fixture)

pytestmark = pytest.mark.gpu

INF, NAN = float("inf"), float("nan")
LENS = [([1, 1, 1, 1], [0, 1, -1, 0]), ([40, 9, 20, 300, 17], [1, 0, -1, 1, 0]), ([300, 70, 200], [1, 0, 1])]


def pattern(y):
    return torch.where(y.isnan(), 2, torch.where(y.isinf(), y.sign(), 0)).int()


def broken(p, slot, values, which="up"):
    """The adapter with values put at (row, column) of one matrix."""
    d, u = p.down[slot].clone(), p.up[slot].clone()
    for (i, j), x in values.items():
        (u if which == "up" else d)[i, j] = x
    return d, u


def check(p, x, cu, slots, d, u, slot):
    """Every finite value within its bound, every other one as the formula has it."""
    out = p.run(x, cu, slots, p.bb.BONSAI_EPI_F32, torch.full((x.shape[0], p.n), 7.0, device="cuda"))
    p.down[slot], p.up[slot] = torch.nan_to_num(d, 0, 0, 0), torch.nan_to_num(u, 0, 0, 0)
    y, bound = p.accumulators(x, cu, slots)
    for i, s in enumerate(slots):
        if s == slot:
            rows = slice(cu[i], cu[i + 1])
            full = (x[rows].double() @ d.double().T) * p.scale[slot]
            full = full @ u.double().T
            y[rows] = torch.where(full.isfinite(), y[rows], full)
    bad = ~y.isfinite()
    assert torch.equal(pattern(out), pattern(y))
    within(torch.where(bad, 0, out), torch.where(bad, 0, y), bound)
    return bad


@pytest.mark.parametrize("lens,slots", LENS, ids=str)
@pytest.mark.parametrize("n,k,rank", [(256, 512, 16), (300, 320, 5), (130, 96, 37)])
def test_up(gpu, kernel, lens, slots, n, k, rank):  # noqa: F811
    p = Problem(gpu, n, k, [rank, 20], seed=n)
    d, u = broken(p, 0, {(3, 0): INF, (17, rank - 1): -INF, (n - 1, 2): NAN, (64, 1): INF, (64, 3): INF})
    p.lora.set(0, d, u, p.scale[0])
    cu = np.cumsum([0] + lens).tolist()
    bad = check(p, p.x(cu[-1]), cu, slots, d, u, 0)
    for i, s in enumerate(slots):
        assert bad[cu[i]:cu[i + 1]].any(0).sum() == (4 if s == 0 else 0)


@pytest.mark.parametrize("lens,slots", LENS, ids=str)
def test_down(gpu, kernel, lens, slots):  # noqa: F811
    p = Problem(gpu, 256, 512, [16, 20])
    d, u = broken(p, 0, {(2, 100): NAN, (7, 511): INF}, "down")
    p.lora.set(0, d, u, p.scale[0])
    cu = np.cumsum([0] + lens).tolist()
    bad = check(p, p.x(cu[-1]), cu, slots, d, u, 0)
    for i, s in enumerate(slots):
        assert bool(bad[cu[i]:cu[i + 1]].all()) == (s == 0)


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


@pytest.mark.parametrize("lens,slots", LENS, ids=str)
@pytest.mark.parametrize("mode", ["F16", "GELU", "RESID", "SWIGLU"])
def test_epilogues(gpu, kernel, lens, slots, mode):  # noqa: F811
    swiglu = mode == "SWIGLU"
    p = Problem(gpu, 512, 256, [16, 20], swiglu=swiglu)
    cu = np.cumsum([0] + lens).tolist()
    x, width = p.x(cu[-1]), 256 if swiglu else 512
    d, u = broken(p, 0, {(5, 1): INF, (300, 2): NAN})

    def run():
        out = torch.ones(cu[-1], width, device="cuda", dtype=torch.float32 if mode == "RESID" else torch.float16)
        return p.run(x, cu, slots, getattr(gpu, "BONSAI_EPI_" + mode), out)
    clean = run()
    p.lora.set(0, d, u, p.scale[0])
    out = run()
    cols = [5, 44] if swiglu else [5, 300]  # rows 256 and on are the values of the gates before them
    for i, s in enumerate(slots):
        rows = slice(cu[i], cu[i + 1])
        same = torch.ones(width, dtype=torch.bool, device="cuda")
        if s == 0:
            same[cols] = False
            assert out[rows, cols[1]].isnan().all()
        assert torch.equal(out[rows][:, same], clean[rows][:, same])
    p.lora.set(0, p.down[0], p.up[0], p.scale[0])  # finite again: nothing of it is left
    assert torch.equal(run(), clean)
