"""A request whose logits are not numbers ends: -1 from there on, and the others go on as if alone."""
import pytest
import torch

from bonsai_b200.text_layer import generate
from test_text_generate_gpu import model

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("cache", ["f16", "i8"])
def test_a_request_without_a_token_ends(gpu, cache):
    layer, embedding, head = model(gpu, cache)
    embedding = embedding.float()
    u = torch.zeros(5, 2, device="cuda")
    greedy = dict(temperature=torch.zeros(2, device="cuda"))
    free = generate(layer, embedding, head, [[5, 9], [7, 4]], 5, u, **greedy)
    embedding[3] *= 1e6  # its hidden state is past f16: logits NaN, keys and values (of normed rows) numbers
    assert not bool((free == 3).any())
    ended = generate(layer, embedding, head, [[5, 9], [7, 3]], 5, u, **greedy)
    assert torch.equal(ended[0], free[0]) and ended[1].tolist() == [-1] * 5
    # in the middle: the second token of request 1
    embedding[3] /= 1e6
    middle = int(free[1, 1])
    assert not bool((free[0] == middle).any()) and int(free[1, 0]) != middle
    embedding[middle] *= 1e6
    ended = generate(layer, embedding, head, [[5, 9], [7, 4]], 5, u, **greedy)
    assert torch.equal(ended[0], free[0]) and ended[1].tolist() == free[1, :2].tolist() + [-1] * 3
