"""Which rows of the output a paged attention call writes where its keys are split
over a second kernel that merges the parts: the rows of its sequences, each
from its own parts, and no others.  Against f64, with the bounds of
test_text_attention_gpu."""
import pytest
import torch

from test_text_attention_gpu import check, f16, gather, ints, make_cache, randn, ref_rows, run_paged

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("lens,ctx", [([1], [20000]), ([2, 0, 1], [9000, 500, 30000])], ids=str)
def test_wide_split_leaves_rows_of_no_sequence(gpu, dim, lens, ctx):
    """q and out with rows before and after the sequences (a batch padded to a
    captured size)."""
    page, before, after = 64, 3, 2
    kc, vc, table = make_cache(30, ctx, page, 1, dim, f16, fill=float("nan"))
    run_paged(gpu, randn(32, 1, 8, dim), kc, vc, table[:1], [0, 1], ctx[:1], page)  # scratch has been used
    cu = [before]
    for n in lens:
        cu.append(cu[-1] + n)
    q = randn(31, cu[-1] + after, 8, dim)
    out = run_paged(gpu, q, kc, vc, table, cu, ctx, page)
    assert (out[:before] == 7).all() and (out[cu[-1]:] == 7).all()


@pytest.mark.parametrize("heads,kv", [(8, 1), (16, 2)])
@pytest.mark.parametrize("n", [257, 300])
def test_split_of_a_later_launch_keeps_the_rows_of_the_first(gpu, heads, kv, n):
    """More sequences than one launch takes: the last launch has few units and
    splits their keys, the first has many and does not."""
    page, dim = 64, 64
    ctx = [2000 + (i * 797) % 8000 for i in range(n)]
    kc, vc, table = make_cache(33, [8000, 9000], page, kv, dim, f16)
    run_paged(gpu, randn(34, 2, heads, dim), kc, vc, table, [0, 1, 2], [8000, 9000], page)  # scratch has been used
    # the sequences share the cache's pages, each in an order of its own
    g = torch.Generator().manual_seed(n)
    width = -(-max(ctx) // page)
    table = torch.stack([torch.randperm(kc.shape[0], generator=g)[:width] for _ in range(n)]).int().cuda()
    run_paged(gpu, randn(35, n, heads, dim), kc, vc, table, list(range(n + 1)), ctx, page)


def test_few_active_sequences_among_many(gpu):
    """300 places of a server's batch, four of them active, in both launches."""
    page, dim, n, active = 64, 128, 300, {10: 30000, 200: 17000, 256: 24000, 299: 9001}
    ctx = [active.get(i, 0) for i in range(n)]
    kc, vc, table = make_cache(36, ctx, page, 8, dim, f16, fill=float("nan"))
    lens = [1 if i in active else 0 for i in range(n)]
    cu = [sum(lens[:i]) for i in range(n + 1)]
    q = randn(37, 6, 32, dim)  # two rows past the last sequence
    out = torch.full(q.shape, 7.0, dtype=f16, device="cuda")
    for _ in range(2):
        out.fill_(7.0)
        gpu.paged_attention(q, kc, vc, table, ints(cu), ints(ctx), 30000, out)
    torch.cuda.synchronize()
    for i, c in active.items():
        a = cu[i]
        check(out[a:a + 1], *ref_rows(q[a:a + 1], gather(kc, table[i], c, page), gather(vc, table[i], c, page), c - 1,
                                      dim ** -0.5))
    assert (out[4:] == 7).all()
