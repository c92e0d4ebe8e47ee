"""The text-stage operators together: tokens that come behind a cache, in chunks
or one by one, get what they get as part of one prompt (same bar as the
engine's parity tests: cos >= 0.9999, max-abs <= 1e-2 of the RMS)."""
import pytest

from bonsai_b200.text_layer import run_both_ways

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("lens,new", [((37, 5, 64), 4), ((1, 130, 16), 2), ((600, 3, 77), 40)], ids=str)
def test_chunks_and_single_tokens_match_the_prompt(gpu, lens, new):
    whole, parts = run_both_ways(lens=lens, new=new, pages=256)
    a, b = whole.double().flatten(), parts.double().flatten()
    assert float(a @ b / (a.norm() * b.norm())) >= 0.9999
    assert float((a - b).abs().max() / a.square().mean().sqrt()) <= 1e-2


def test_adapters_change_only_their_requests(gpu):
    """Request 1 has no adapter: its tokens do not move with the others' adapters."""
    a, _ = run_both_ways()
    b, _ = run_both_ways(adapters=(1, -1, 0))
    assert not a[0].equal(b[0]) and not a[2].equal(b[2])
    assert a[1].equal(b[1])
