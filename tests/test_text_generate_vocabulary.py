"""generate refuses tokens that its embedding does not have, before any device work: in a prompt,
or that the output projection could choose; and widths other than the layer's."""
import types

import pytest
import torch

import bonsai_b200 as bb
from bonsai_b200.text_layer import generate

LAYER = types.SimpleNamespace(page_size=16, hidden=8, k_cache=types.SimpleNamespace(shape=(4, 16, 2, 128)))


def head(out_dim=10, in_dim=8):
    return types.SimpleNamespace(out_dim=out_dim, in_dim=in_dim)


@pytest.mark.parametrize("rows,width,out_dim,in_dim,prompts", [
    (10, 8, 10, 8, [[1, 10], [2]]), (10, 8, 10, 8, [[1], [2, -1]]), (10, 8, 11, 8, [[1], [2]]),
    (10, 16, 10, 8, [[1], [2]]), (10, 8, 10, 16, [[1], [2]])], ids=str)
def test_refuses(rows, width, out_dim, in_dim, prompts):
    with pytest.raises(bb.BonsaiError):
        generate(LAYER, torch.zeros(rows, width), head(out_dim, in_dim), prompts, 2, torch.zeros(2, 2))
