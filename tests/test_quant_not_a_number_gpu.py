"""A block whose exponent byte is 255 reads as NaN whatever its codes, in the same places for all
that read a quantised cache: rows read back, keys and values under single tokens and chunks."""
import pytest
import torch

import quant_ref as qr
from test_quant_attention_gpu import run, setup
from test_text_attention_gpu import bf16, f16, ints

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [f16, bf16], ids=["f16", "bf16"])
@pytest.mark.parametrize("fmt", ["i8", "i4"])
@pytest.mark.parametrize("dim", [64, 128])
def test_read_back(gpu, dtype, fmt, dim):
    _, caches, table = setup(gpu, [1], [40], 2, 2, dim, 8, dtype, fmt)
    for i, c in enumerate(caches):
        c.scales[:, i::3, :, i] = 255
    k, v = (torch.empty(40, 2, dim, dtype=dtype, device="cuda") for _ in range(2))
    gpu.paged_read_quant(*caches, table, ints([0, 40]), None, k, v)
    for c, got in zip(caches, (k, v)):
        want = torch.cat([qr.values(c.codes, c.scales, fmt)[i] for i in table[0].tolist()])[:40]
        assert torch.equal(got.isnan(), want.isnan()) and bool(want.isnan().any())
        assert torch.equal(got[~want.isnan()].double(), want[~want.isnan()])


@pytest.mark.parametrize("lens", [[1, 1], [3, 2], [90, 5]], ids=str)
@pytest.mark.parametrize("dtype", [f16, bf16], ids=["f16", "bf16"])
@pytest.mark.parametrize("fmt", ["i8", "i4"])
@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("side", ["k", "v"])
def test_attention(gpu, lens, dtype, fmt, dim, side):
    """The last key of the first sequence, the 33rd of the second and one that nobody sees."""
    ctx = [150, 200]
    q, caches, table = setup(gpu, lens, ctx, 4, 2, dim, 16, dtype, fmt, seed=4)
    c = caches["kv".index(side)]
    for s, pos, head in ((0, 149, 0), (1, 33, 1), (0, 155, 1)):
        c.scales[int(table[s, pos // 16]), pos % 16, head, 1] = 255
    out = run(gpu, q, caches, table, lens, ctx)
    assert not bool(out[:lens[0], 2:].isnan().any()) and bool(out[lens[0]:, 2:].isnan().any())


@pytest.mark.parametrize("lens", [[1, 1], [90, 5]], ids=str)
@pytest.mark.parametrize("dtype", [f16, bf16], ids=["f16", "bf16"])
@pytest.mark.parametrize("fmt", ["i8", "i4"])
@pytest.mark.parametrize("dim", [64, 128])
def test_a_key_whose_codes_are_of_one_sign(gpu, lens, dtype, fmt, dim):
    """With an infinite scale its product with a query of the other sign would be -inf, a key that counts nothing."""
    ctx = [150, 200]
    q, caches, table = setup(gpu, lens, ctx, 4, 2, dim, 16, dtype, fmt, seed=6)
    q[..., 32:64] = -q[..., 32:64].abs() - 0.1
    page, width = int(table[0, 2]), 32 if fmt == "i8" else 16
    caches[0].codes[page, 5, 1, width:2 * width] = 128 + 9 if fmt == "i8" else 0xbb
    caches[0].scales[page, 5, 1, 1] = 255
    out = run(gpu, q, caches, table, lens, ctx)
    assert bool(out[:lens[0], 2:].isnan().all()) and int(out.isnan().sum()) == lens[0] * 2 * dim
