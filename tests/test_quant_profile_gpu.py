"""The profile counts a call over a quantised cache once, whichever kernels it takes."""
import pytest
import torch

from test_quant_attention_gpu import setup
from test_text_attention_gpu import bf16, cumulated, ints

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("lens,ctx", [([1, 1], [300, 40]), ([40, 1], [300, 40]), ([40, 33], [300, 40])], ids=str)
def test_bytes_of_a_call(gpu, lens, ctx):
    q, caches, table = setup(gpu, lens, ctx, 8, 2, 128, 16, bf16, "i8")
    out = torch.empty_like(q)
    gpu.profile_start()
    gpu.paged_attention_quant(q, *caches, table, ints(cumulated(lens)), ints(ctx), max(ctx), out, max_q=max(lens))
    kinds = {k: v for k, v in gpu.profile_stop().items() if "attention" in k}
    assert list(kinds) == ["paged_attention_quant"]
    got = kinds["paged_attention_quant"]
    rows, keys = 2 * 2 * 128 * 8 * sum(lens), 2 * 2 * (128 + 4) * len(ctx) * max(ctx)  # Q and O; codes of K and V, at the bound
    assert got["launches"] == 1 and got["bytes"] == pytest.approx(rows + keys, rel=1e-6)
