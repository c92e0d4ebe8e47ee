"""bonsai_sample_tokens next to a border of its sums: a row of two values, first n tokens of
weight w = e^x, then n of weight 1, and u so that u * n (1 + w) lies within `gap` of a
token's weight of the end of token j.  A weight that is off by a relative d moves that border by
d u n tokens' weights; with weights within 1e-13 and f64 sums (1e-15 per addition of a chain
of a few hundred) that is below 1e-7 here, with weights within 5e-10 it was up to 6e-5.
"""
import math

import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu

N = 1 << 17
GAP = 4e-6, 2e-5  # in weights of a token: far above 1e-7, below what single precision in a weight's parts gives


def near_borders(x, seed, count):
    """f32 u whose target lies within GAP of the end of a token of the first n, and the token that it chooses."""
    w = math.exp(float(x))
    u = np.random.default_rng(seed).random(1 << 19, dtype=np.float32)
    u = u[(u > 0.1) & (u < 0.9 * w / (1 + w))]
    at = u.astype(np.longdouble) * N * ((1 + np.longdouble(w)) / np.longdouble(w))  # in weights of the first n
    off = at - np.rint(at)
    near = (np.abs(off) > GAP[0]) & (np.abs(off) < GAP[1])
    # token j ends at j + 1; a sum that exceeds the target
    return u[near][:count], np.floor(at[near][:count]).astype(np.int64)


@pytest.mark.parametrize("seed", range(4))
def test_choice_next_to_a_border(gpu, seed):
    rows, us, want = [], [], []
    for i in range(24):
        # between two entries of a table of 64 steps, where a polynomial's roundings count most
        x = np.float32(-(2 * i + 0.5 + 0.02 * (seed - 2)) * math.log(2) / 64)
        u, j = near_borders(x, 100 * seed + i, 2)
        rows += [x] * len(u)
        us += u.tolist()
        want += j.tolist()
    logits = torch.zeros(len(rows), 2 * N, device="cuda")
    logits[:, :N] = torch.tensor(np.array(rows), device="cuda")[:, None]
    tokens, probs = torch.empty(len(rows), dtype=torch.int32, device="cuda"), torch.empty(len(rows), device="cuda")
    gpu.sample_tokens(logits, torch.tensor(us, device="cuda"), tokens, probs=probs)
    torch.cuda.synchronize()
    assert len(rows) >= 12 and tokens.tolist() == want
    for p, x in zip(probs.tolist(), rows):
        w = math.exp(float(x))
        assert abs(p - w / (N * (1 + w))) <= (2.0 ** -24 + 1e-12) * p
