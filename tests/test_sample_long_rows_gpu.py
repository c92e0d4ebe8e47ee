"""bonsai_sample_tokens over a row of 2^25 tokens, where a bin's mass is counted in units of 1/1024 of a
token's weight and more, and top-p and min-p both cut.

Three values: one token at 0, n_b at -(1 + a), n_c at -(2 + c), one at -8, so that a bin is 1/256 wide.
a and c make a token of the one level fall short of its weight by 0.95 units of 1023, of the other by 0.05:
by those masses the share of the first two levels is too small by a quarter of the difference, 2.2e-4
of the whole.  top-p lies below their true share by 5e-5, so it cuts some of n_b; min-p cuts n_c.
"""
import math

import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu

V, UNIT = 1 << 25, 1024


@pytest.mark.parametrize("short", [(0.95, 0.05), (0.05, 0.95)], ids=str)
@pytest.mark.parametrize("off", [-5e-5, 5e-5])
def test_mass_border_of_a_long_row(gpu, short, off):
    xb, xc = (np.float32(-(i + 1 - math.log((UNIT - 2 + s) / UNIT))) for i, s in enumerate(short))
    wb, wc = math.exp(float(xb)), math.exp(float(xc))
    n_b = int((V - 2) * wc / (wb + wc))
    n_c = V - 2 - n_b
    whole = 1 + n_b * wb + n_c * wc + math.exp(-8.0)
    p = float(np.float32((1 + n_b * wb) / whole + off))
    kept = (p * whole - 1) / wb  # tokens of the second level with a mass before them of less than p of the whole
    # far from a border compared with the error of f64 sums of 2^25 weights within 1e-13
    assert 1e-3 < kept - math.floor(kept) < 1 - 1e-3
    kept = min(n_b, math.ceil(kept))
    u = float(np.float32(1 - 2.0 ** -20))
    at = (u * (1 + kept * wb) - 1) / wb
    assert 1e-3 < at - math.floor(at) < 1 - 1e-3
    x = torch.empty(1, V, device="cuda")
    x[0, 0], x[0, 1:1 + n_b], x[0, 1 + n_b:V - 1], x[0, V - 1] = 0.0, float(xb), float(xc), -8.0
    f = lambda v: torch.tensor([v], device="cuda")  # noqa: E731
    tokens, probs = torch.empty(1, dtype=torch.int32, device="cuda"), torch.empty(1, device="cuda")
    gpu.sample_tokens(x, f(u), tokens, probs=probs, top_p=f(p), min_p=f(math.exp(-1.5)))
    torch.cuda.synchronize()
    assert int(tokens) == 1 + math.floor(at)
    assert abs(float(probs) - wb / (1 + kept * wb)) <= (2.0 ** -24 + 1e-12) * wb / (1 + kept * wb)
