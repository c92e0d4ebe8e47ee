"""generate takes random numbers with any strides, and refuses those of another type or place before it
writes to the cache."""
import pytest
import torch

import bonsai_b200 as bb
from bonsai_b200.text_layer import generate
from test_text_generate_gpu import PROMPTS, model

pytestmark = pytest.mark.gpu


def test_strides(gpu):
    u = torch.rand(4, 3, generator=torch.Generator().manual_seed(3)).cuda()
    layer, embedding, head = model(gpu, "i8")
    want = generate(layer, embedding, head, PROMPTS, 4, u)
    for other in (u.t().contiguous().t(), torch.stack([u, u], -1)[..., 1]):
        assert not other.is_contiguous()
        assert torch.equal(generate(layer, embedding, head, PROMPTS, 4, other), want)
    same = u[:1].expand(4, 3)
    assert torch.equal(generate(layer, embedding, head, PROMPTS, 4, same), generate(layer, embedding, head, PROMPTS, 4, same.contiguous()))


@pytest.mark.parametrize("bad", [torch.zeros(2, 3), torch.zeros(2, 3, dtype=torch.float64)], ids=["host", "f64"])
def test_refused_before_the_cache(gpu, bad):
    layer, embedding, head = model(gpu, "i8")
    with pytest.raises(bb.BonsaiError):
        generate(layer, embedding, head, PROMPTS, 2, bad if bad.dtype is torch.float32 else bad.cuda())
    torch.cuda.synchronize()
    assert not bool(layer.k_cache.scales.any())
