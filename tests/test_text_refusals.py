"""Arguments that the text-stage entry points refuse: the checks run before any
device work, so a CPU sees them too."""
import ctypes

import pytest

import bonsai_b200 as bb

ARG, UNSUPPORTED = -1, -2


def heads(data=1 << 20, token=1024, head=128):
    return ctypes.byref(bb.HeadsDesc(data, token, head))


def pages(data=1 << 20, page=16384, token=1024, head=128, n=4, size=16):
    return ctypes.byref(bb.PagesDesc(data, page, token, head, n, size))


def prompt(q=heads(), k=heads(), v=heads(), cu=64, n=1, T=5, H=8, Hk=8, D=128, dtype=0, scale=0.1, out=heads()):
    return bb.lib().bonsai_prompt_attention(q, k, v, cu, n, T, H, Hk, D, dtype, 1, scale, out, None)


def paged(q=heads(), kc=pages(), vc=pages(), table=64, ld=9, width=9, cu=64, ctx=64, n=1, T=5, max_ctx=20, H=8, Hk=8,
          D=128, dtype=0, scale=0.1, out=heads()):
    return bb.lib().bonsai_paged_attention(q, kc, vc, table, ld, width, cu, ctx, n, T, max_ctx, H, Hk, D, dtype, scale,
                                           out, None)


def append(k=heads(), v=heads(), kc=pages(), vc=pages(), table=64, ld=9, width=9, cu=64, ctx=64, n=1, T=5, Hk=8, D=128):
    return bb.lib().bonsai_paged_append(k, v, kc, vc, table, ld, width, cu, ctx, n, T, Hk, D, None)


SHAPES = [(dict(n=-1), ARG), (dict(T=-1), ARG), (dict(Hk=0), ARG), (dict(D=96), UNSUPPORTED)]
ATTENTION = [(dict(H=0), ARG), (dict(H=9, Hk=2), ARG), (dict(H=129, Hk=1), UNSUPPORTED), (dict(dtype=2), ARG),
             (dict(scale=0.0), ARG), (dict(scale=-1.0), ARG), (dict(scale=float("nan")), ARG),
             (dict(scale=float("inf")), ARG), (dict(out=None), ARG), (dict(out=heads(data=8)), ARG),
             (dict(out=heads(head=100)), ARG), (dict(q=None), ARG), (dict(q=heads(token=0)), ARG),
             (dict(q=heads(token=-1024)), ARG), (dict(q=heads(data=(1 << 20) + 2)), ARG)]
PAGES = [(dict(kc=None), ARG), (dict(vc=pages(size=12)), UNSUPPORTED), (dict(vc=pages(size=4)), UNSUPPORTED),
         (dict(kc=pages(size=32)), ARG), (dict(kc=pages(n=5)), ARG), (dict(kc=pages(n=0)), ARG),
         (dict(kc=pages(data=0)), ARG), (dict(kc=pages(head=4)), ARG), (dict(table=None), ARG), (dict(cu=None), ARG),
         (dict(ctx=None), ARG), (dict(ld=8), ARG), (dict(width=-1, ld=3), ARG)]


@pytest.mark.parametrize("bad,code", SHAPES + ATTENTION + [(dict(cu=None), ARG),
                                                           (dict(k=heads(token=1001)), ARG)], ids=str)
def test_prompt_attention_refuses(bad, code):
    assert prompt(**bad) == code
    assert b"attention" in bb.lib().bonsai_last_error()


@pytest.mark.parametrize("bad,code", SHAPES + ATTENTION + PAGES + [(dict(max_ctx=-1), ARG)], ids=str)
def test_paged_attention_refuses(bad, code):
    assert paged(**bad) == code
    assert b"attention" in bb.lib().bonsai_last_error()


@pytest.mark.parametrize("bad,code", SHAPES + PAGES + [(dict(k=None), ARG), (dict(v=heads(head=12)), ARG)], ids=str)
def test_paged_append_refuses(bad, code):
    assert append(**bad) == code
    assert b"paged_append" in bb.lib().bonsai_last_error()


def test_nothing_to_do_is_no_error():
    assert prompt(n=0, cu=None, q=None) == 0 and prompt(T=0, out=None) == 0
    assert paged(T=0, q=None) == 0 and append(n=0, table=None) == 0
