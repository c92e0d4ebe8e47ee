"""Tensor memory of kernels whose CTAs wait for one another in clusters: whichever
of them an SM's shared memory admits together, of one launch or of several
streams, have to fit its tensor memory.  Otherwise a CTA could wait for
columns behind a CTA that waits for its own cluster."""
import ctypes

import bonsai_b200 as bb

SMEM, COLUMNS = 228 * 1024, 512


def shares():
    L = bb.lib()
    n = L.bonsai_debug_tmem_shares(None, None, 0)
    smem, cols = (ctypes.c_int * n)(), (ctypes.c_int * n)()
    assert L.bonsai_debug_tmem_shares(smem, cols, n) == n
    return list(zip(smem, cols))


def most_columns(kinds, smem):
    """The most columns of any set of CTAs, kinds repeated, within `smem` bytes."""
    return max((c + most_columns(kinds[i:], smem - s) for i, (s, c) in enumerate(kinds) if s <= smem), default=0)


def test_ctas_that_fit_an_sm_fit_its_tensor_memory():
    kinds = shares()
    assert len(kinds) >= 15 and all(1024 < s <= SMEM and 32 <= c <= COLUMNS for s, c in kinds)
    assert most_columns(kinds, SMEM) <= COLUMNS


def test_the_sum_sees_what_does_not_fit():
    """Two CTAs of 107776 bytes and 512 columns, or one beside an attention CTA."""
    assert most_columns([(107776 + 1024, 512)], SMEM) == 1024
    assert most_columns([(132352 + 1024, 512), (64000 + 1024, 256)], SMEM) == 768
    assert most_columns([(65024, 256)], SMEM) == 768


def test_shares_refuses_no_room():
    assert bb.lib().bonsai_debug_tmem_shares(None, None, 4) == -1
    assert bb.lib().bonsai_debug_tmem_shares(None, None, -1) == -1
