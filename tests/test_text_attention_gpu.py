"""Prompt attention over packed sequences and attention over a paged cache
(bonsai_prompt_attention, bonsai_paged_append, bonsai_paged_attention) against
a plain implementation in f64.

Error bound of an output element, with p the exact softmax weights and u the
unit roundoff of the tensors' type (2^-11 f16, 2^-8 bf16): P is rounded to that
type and so is the output, each at most u relative; the f32 dot products and
the exponential add e = 2 * (D + 8) * 2^-24 * max(scale * sum|q||k|) + 2^-20 to
each weight (and as much to their sum); P below f16's normal range is rounded
to a multiple of 2^-24 while the row's sum is at least 1, which is 2^-25 per
key.  So |err| <= (2 u + 2 e) * sum_j p_j |v_j| + n_keys * 2^-25 * max|v|.
"""
import pytest
import torch

pytestmark = pytest.mark.gpu

UNIT = {torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}
f16, bf16 = torch.float16, torch.bfloat16


def ref_rows(q, k, v, first, scale, causal=True):
    """f64 attention of one sequence: q [n][H][D], k, v [m][Hk][D]; query i is at
    place first + i.  Returns the outputs and the error bound; rows that see
    no key are zero.  Only the keys a row sees enter its sum."""
    n, H, D = q.shape
    m, Hk = k.shape[:2]
    g = H // Hk
    qd, kd, vd = q.double(), k.double().repeat_interleave(g, 1), v.double().repeat_interleave(g, 1)
    s = torch.einsum("ihd,jhd->hij", qd, kd) * scale
    mag = torch.einsum("ihd,jhd->hij", qd.abs(), kd.abs()) * scale
    see = torch.ones(n, m, dtype=torch.bool, device=q.device)
    if causal:
        see = torch.arange(m, device=q.device) <= (torch.arange(n, device=q.device) + first)[:, None]
    s = s.masked_fill(~see, float("-inf"))
    p = torch.where(see.any(1)[:, None], torch.softmax(s, -1), torch.zeros((), dtype=s.dtype, device=s.device))
    p = torch.where(see, p, torch.zeros_like(p))
    # 0 * inf of an unseen key is not part of the sum
    out = torch.stack([torch.stack([(p[h, i, see[i]][:, None] * vd[see[i], h]).sum(0) if not vd.isfinite().all()
                                    else p[h, i] @ vd[:, h] for h in range(H)]) for i in range(n)]) \
        if not vd.isfinite().all() else torch.einsum("hij,jhd->ihd", p, vd)
    fin = lambda x: torch.nan_to_num(x, 0.0, 0.0, 0.0)  # noqa: E731
    u = UNIT[q.dtype]
    e = 2 * (D + 8) * 2.0 ** -24 * float(fin(mag).max() if mag.numel() else 0.0) + 2.0 ** -20
    va = fin(vd).abs()
    bound = (2 * u + 2 * e) * torch.einsum("hij,jhd->ihd", fin(p), va) + m * 2.0 ** -25 * (va.max() if m else 0.0)
    return out, bound


def check(out, ref, bound):
    out = out.double()
    bad = ~ref.isfinite()
    assert torch.equal(out.isfinite(), ref.isfinite()), "finite where the reference is not, or the other way around"
    assert torch.equal(out[bad].isnan(), ref[bad].isnan())
    over = ((out - ref).abs() - bound)[~bad]
    assert over.numel() == 0 or float(over.max()) <= 0.0, f"off by {float(over.max())} more than the bound"


def randn(seed, *shape, dtype=f16, std=1.2):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return (torch.randn(*shape, device="cuda", generator=g) * std).to(dtype)


def ints(v):
    return torch.tensor(v, dtype=torch.int32, device="cuda")


def cumulated(lens):
    cu = [0]
    for x in lens:
        cu.append(cu[-1] + x)
    return cu


def run_prompt(bb, q, k, v, cu, causal=True, scale=None, out=None, check_all=True):
    D = q.shape[2]
    scale = D ** -0.5 if scale is None else scale
    out = torch.full(q.shape, 7.0, dtype=q.dtype, device="cuda") if out is None else out
    bb.prompt_attention(q, k, v, ints(cu), out, scale=scale, causal=causal)
    torch.cuda.synchronize()
    for a, b in zip(cu, cu[1:]):
        if b > a:
            check(out[a:b], *ref_rows(q[a:b], k[a:b], v[a:b], 0, scale, causal))
    return out


LENS = [[1], [2], [41], [64], [65], [128], [129], [1, 1, 1], [31, 0, 33, 1], [0, 5, 0], [127, 255, 64, 63], [300],
        [513, 7, 190]]


@pytest.mark.parametrize("lens", LENS, ids=str)
@pytest.mark.parametrize("dtype", [f16, bf16], ids=["f16", "bf16"])
@pytest.mark.parametrize("causal", [True, False], ids=["causal", "full"])
def test_prompt_lengths(gpu, lens, dtype, causal):
    T = sum(lens)
    q, k, v = (randn(i, T, h, 128, dtype=dtype) for i, h in enumerate((8, 2, 2)))
    run_prompt(gpu, q, k, v, cumulated(lens), causal)


@pytest.mark.parametrize("heads,kv", [(1, 1), (3, 3), (24, 24), (32, 8), (12, 4), (28, 4), (20, 4), (8, 1), (33, 1),
                                      (128, 1), (65, 1)])
@pytest.mark.parametrize("dim", [64, 128])
def test_prompt_heads(gpu, heads, kv, dim):
    lens = [70, 3, 130]
    q, k, v = (randn(i, sum(lens), h, dim, dtype=bf16 if dim == 64 else f16) for i, h in enumerate((heads, kv, kv)))
    run_prompt(gpu, q, k, v, cumulated(lens))


def test_prompt_many_sequences(gpu):
    lens = [(i * 37) % 90 for i in range(700)]
    q, k, v = (randn(i, sum(lens), h, 64) for i, h in enumerate((4, 2, 2)))
    run_prompt(gpu, q, k, v, cumulated(lens))


@pytest.mark.parametrize("dim", [64, 128])
def test_prompt_long(gpu, dim):
    lens = [2999, 4097]
    q, k, v = (randn(i, sum(lens), h, dim, dtype=bf16) for i, h in enumerate((8, 2, 2)))
    run_prompt(gpu, q, k, v, cumulated(lens))


@pytest.mark.parametrize("causal", [True, False])
def test_prompt_large_scores(gpu, causal):
    """Row maxima that keep growing along the keys: the rescaling path."""
    T = 700
    q, k, v = (randn(i, T, h, 128) for i, h in enumerate((4, 2, 2)))
    k *= torch.linspace(0.1, 4.0, T, device="cuda")[:, None, None].half()
    q *= 3
    run_prompt(gpu, q, k, v, [0, T], causal)


def test_prompt_strides(gpu):
    """Slices of one fused projection, head-major tensors, gaps in the output."""
    H, Hk, D, T = 6, 2, 128, 150
    qkv = randn(0, T, (H + 2 * Hk) * D + 8)
    q = qkv[:, :H * D].unflatten(1, (H, D))
    k = qkv[:, H * D:(H + Hk) * D].unflatten(1, (Hk, D))
    v = qkv[:, (H + Hk) * D:(H + 2 * Hk) * D].unflatten(1, (Hk, D))
    big = torch.full((T, H + 1, D + 8), 7.0, device="cuda", dtype=f16)
    run_prompt(gpu, q, k, v, [0, 60, 150], out=big[:, :H, :D])
    assert (big[:, H] == 7).all() and (big[:, :, D:] == 7).all()
    hm = [randn(i, h, T, D).transpose(0, 1) for i, h in enumerate((H, Hk, Hk))]
    run_prompt(gpu, *hm, [0, 60, 150], out=torch.empty(H, T, D, device="cuda", dtype=f16).transpose(0, 1))


def test_prompt_gaps_are_not_used_or_written(gpu):
    """cu_seqlens that begins after row 0 and ends before the last: rows of no
    sequence hold NaN, are not read into any result and not written."""
    q, k, v = (randn(i, 200, h, 128) for i, h in enumerate((4, 2, 2)))
    for t in (q, k, v):
        t[:10] = float("nan")
        t[171:] = float("nan")
    out = run_prompt(gpu, q, k, v, [10, 60, 171])
    assert (out[:10] == 7).all() and (out[171:] == 7).all()


@pytest.mark.parametrize("bad", [float("nan"), float("inf"), float("-inf")], ids=str)
@pytest.mark.parametrize("which", ["k", "v", "q"])
def test_prompt_nonfinite_reaches_only_rows_that_see_it(gpu, bad, which):
    q, k, v = (randn(i, 260, h, 128) for i, h in enumerate((4, 2, 2)))
    if which == "v":
        v[77, 1, 5] = bad
        v[130, 0, 100] = bad
        run_prompt(gpu, q, k, v, [0, 90, 260])
        return
    (q if which == "q" else k)[77, 1, 5] = bad
    out = torch.empty_like(q)
    gpu.prompt_attention(q, k, v, ints([0, 90, 260]), out)
    clean = [t.clone() for t in (q, k, v)]
    for t in clean:
        t[77:90] = 0
    ref, bound = ref_rows(clean[0][:77], clean[1][:77], clean[2][:77], 0, 128 ** -0.5)
    check(out[:77], ref, bound)
    ref, bound = ref_rows(q[90:], k[90:], v[90:], 0, 128 ** -0.5)
    check(out[90:], ref, bound)


# ------------------------------------------------------------------- paged
def make_cache(seed, ctx, page, heads, dim, dtype, extra=2, fill=None, shuffle=True):
    """A cache with the pages of the sequences in shuffled order, and the table.
    `fill`: value of every slot that no sequence has (None: random)."""
    per = [-(-x // page) for x in ctx]
    total = sum(per) + extra
    g = torch.Generator().manual_seed(seed)
    order = torch.randperm(total, generator=g).tolist() if shuffle else list(range(total))
    kc, vc = (randn(seed + i, total, page, heads, dim, dtype=dtype) for i in range(2))
    width = max(max(per), 1) + 1
    table = torch.full((len(ctx), width), -1, dtype=torch.int32)
    used = torch.zeros(total, page, dtype=torch.bool)
    at = 0
    for i, n in enumerate(per):
        table[i, :n] = torch.tensor(order[at:at + n], dtype=torch.int32)
        for j in range(n):
            used[order[at + j], :min(page, ctx[i] - j * page)] = True
        at += n
    if fill is not None:
        kc[~used.cuda()] = fill
        vc[~used.cuda()] = fill
    return kc, vc, table.cuda()


def gather(cache, table, length, page):
    pages = table[:-(-length // page)].long() if length > 0 else table[:0].long()
    return cache[pages].flatten(0, 1)[:length]


def run_paged(bb, q, kc, vc, table, cu, ctx, page, max_ctx=None):
    D = q.shape[2]
    out = torch.full(q.shape, 7.0, dtype=q.dtype, device="cuda")
    bb.paged_attention(q, kc, vc, table, ints(cu), ints(ctx), max(ctx) if max_ctx is None else max_ctx, out)
    torch.cuda.synchronize()
    for i, n in enumerate(ctx):
        a, b = cu[i], cu[i + 1]
        if b > a:
            check(out[a:b], *ref_rows(q[a:b], gather(kc, table[i], n, page), gather(vc, table[i], n, page),
                                      n - (b - a), D ** -0.5))
    return out


@pytest.mark.parametrize("page", [8, 16, 32, 64, 128, 256])
@pytest.mark.parametrize("dtype", [f16, bf16], ids=["f16", "bf16"])
@pytest.mark.parametrize("dim", [64, 128])
def test_paged_single_tokens(gpu, page, dtype, dim):
    ctx = [1, 2, page - 1, page, page + 1, 63, 64, 65, 200, 999]
    kc, vc, table = make_cache(1, ctx, page, 2, dim, dtype, fill=float("nan"))
    q = randn(9, len(ctx), 8, dim, dtype=dtype)
    run_paged(gpu, q, kc, vc, table, list(range(len(ctx) + 1)), ctx, page)


@pytest.mark.parametrize("lens,ctx", [([5], [5]), ([1, 40, 129], [700, 41, 1000]), ([33, 0, 64], [33, 50, 4000]),
                                      ([200, 1, 1, 0], [201, 1, 64, 0]), ([512], [3000])], ids=str)
@pytest.mark.parametrize("heads,kv,dim", [(32, 8, 128), (4, 4, 64), (7, 1, 128)])
@pytest.mark.parametrize("page", [16, 64])
def test_paged_chunks(gpu, lens, ctx, heads, kv, dim, page):
    kc, vc, table = make_cache(2, ctx, page, kv, dim, bf16, fill=float("inf"))
    run_paged(gpu, randn(3, sum(lens), heads, dim, dtype=bf16), kc, vc, table, cumulated(lens), ctx, page)


@pytest.mark.parametrize("n", [255, 256, 257, 600])
def test_paged_many_sequences(gpu, n):
    """More sequences than one launch takes; single tokens, chunks and empty ones mixed."""
    lens = [(1, 1, 0, 5, 1, 40)[i % 6] for i in range(n)]
    ctx = [max(m, (i * 61) % 330) for i, m in enumerate(lens)]
    kc, vc, table = make_cache(21, ctx, 16, 2, 64, f16, fill=float("nan"))
    run_paged(gpu, randn(22, sum(lens), 8, 64), kc, vc, table, cumulated(lens), ctx, 16)


@pytest.mark.parametrize("max_ctx", [0, 1, 100, 100000])
def test_paged_max_ctx_only_sets_the_split(gpu, max_ctx):
    ctx = [5000, 3, 777]
    kc, vc, table = make_cache(4, ctx, 32, 2, 128, f16, fill=float("nan"))
    run_paged(gpu, randn(5, 3, 8, 128), kc, vc, table, [0, 1, 2, 3], ctx, 32, max_ctx=max_ctx)


def test_paged_rows_that_see_nothing_are_zero(gpu):
    """Lengths of zero, and more new tokens than the length holds."""
    ctx = [0, 2, 100]
    kc, vc, table = make_cache(6, ctx, 16, 2, 128, f16, fill=float("nan"))
    out = run_paged(gpu, randn(7, 12, 8, 128), kc, vc, table, [0, 3, 8, 12], ctx, 16)
    assert (out[:3] == 0).all() and (out[3:6] == 0).all() and (out[6:8] != 0).any()


def test_paged_bad_pages_read_zeros(gpu):
    """Page indices outside the cache count as pages of zeros; a length past
    the table is cut to the table."""
    ctx = [100, 40]
    kc, vc, table = make_cache(8, ctx, 16, 2, 128, f16)
    q = randn(9, 2, 8, 128)
    table = table[:, :7].contiguous()
    table[0, 2], table[1, 0] = 1 << 30, -5
    out = torch.empty_like(q)
    gpu.paged_attention(q, kc, vc, table, ints([0, 1, 2]), ints([5000, 40]), 5000, out)
    for i, n in enumerate((112, 40)):
        t = table[i].clamp(0, kc.shape[0] - 1)
        k, v = gather(kc, t, n, 16).clone(), gather(vc, t, n, 16).clone()
        lo = 32 if i == 0 else 0
        k[lo:lo + 16] = 0
        v[lo:lo + 16] = 0
        check(out[i:i + 1], *ref_rows(q[i:i + 1], k, v, n - 1, 128 ** -0.5))


def test_paged_nonfinite_new_token_reaches_only_later_rows(gpu):
    ctx, n = [300], 80
    kc, vc, table = make_cache(10, ctx, 16, 2, 128, f16)
    place = 260  # new token 40
    vc[table[0, place // 16], place % 16, 1, 7] = float("inf")
    vc[table[0, 290 // 16], 290 % 16, 0, 100] = float("nan")
    run_paged(gpu, randn(11, n, 4, 128), kc, vc, table, [0, n], ctx, 16)


def test_paged_other_layouts(gpu):
    """A head-major cache [page][head][slot][dim] and keys and values in one buffer."""
    page, Hk, D = 16, 2, 128
    ctx = [333, 90]
    kc, vc, table = make_cache(12, ctx, page, Hk, D, f16)
    both = torch.stack([kc, vc], 1).transpose(2, 3).contiguous()  # [page][2][head][slot][dim]
    q = randn(13, 2, 8, D)
    run_paged(gpu, q, both[:, 0].transpose(1, 2), both[:, 1].transpose(1, 2), table, [0, 1, 2], ctx, page)


@pytest.mark.parametrize("page", [8, 64])
def test_paged_append(gpu, page):
    lens, ctx = [3, 0, 1, 70], [3, 20, 300, 100]
    kc, vc, table = make_cache(14, ctx, page, 2, 64, bf16)
    k, v = (randn(i, sum(lens), 2, 64, dtype=bf16) for i in range(2))
    want = [kc.clone(), vc.clone()]
    cu = cumulated(lens)
    for i, n in enumerate(lens):
        for t in range(n):
            place = ctx[i] - n + t
            for w, new in zip(want, (k, v)):
                w[table[i, place // page], place % page] = new[cu[i] + t]
    gpu.paged_append(k, v, kc, vc, table, ints(cu), ints(ctx))
    assert torch.equal(kc, want[0]) and torch.equal(vc, want[1])


def test_paged_append_skips_what_has_no_place(gpu):
    kc, vc, table = make_cache(15, [16], 16, 2, 64, f16)
    table = table[:, :1].contiguous()
    before = kc.clone()
    k = randn(1, 5, 2, 64)
    for ctx, tab in (([2], table), ([900], table), ([16], torch.full_like(table, 99)), ([16], -table - 1)):
        gpu.paged_append(k, k, kc, vc, tab, ints([0, 5]), ints(ctx))
        at = [p for p in range(ctx[0] - 5, ctx[0]) if 0 <= p < 16] if tab is table else []
        for p in at:
            before[table[0, 0], p] = k[p - (ctx[0] - 5)]
        assert torch.equal(kc, before)


def test_paged_cache_beyond_32_bit_offsets(gpu):
    """Pages past 2^31 elements of the cache, and past 2^32 bytes."""
    page, Hk, D = 64, 8, 128
    pages = (1 << 31) // (page * Hk * D) + 40
    kc, vc = (torch.zeros(pages, page, Hk, D, dtype=f16, device="cuda") for _ in range(2))
    ids = [pages - 1, 3, pages - 20, 7, pages - 2]
    n = 4 * page + 9
    table = ints([ids])
    k, v = (randn(i, n, Hk, D) for i in range(2))
    gpu.paged_append(k, v, kc, vc, table, ints([0, n]), ints([n]))
    assert torch.equal(gather(kc, table[0], n, page), k)
    run_paged(gpu, randn(3, 6, 16, D), kc, vc, table, [0, 6], [n], page)


def test_text_attention_on_another_stream_and_in_a_graph(gpu):
    ctx = [2000, 70]
    kc, vc, table = make_cache(16, ctx, 16, 2, 128, f16)
    q = randn(17, 2, 8, 128)
    cu, cx = ints([0, 1, 2]), ints(ctx)
    want = run_paged(gpu, q, kc, vc, table, [0, 1, 2], ctx, 16)
    side = torch.cuda.Stream()
    out = torch.zeros_like(q)
    side.wait_stream(torch.cuda.current_stream())
    gpu.paged_attention(q, kc, vc, table, cu, cx, 2000, out, stream=side)
    side.synchronize()
    assert torch.equal(out, want)
    out.zero_()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        gpu.paged_attention(q, kc, vc, table, cu, cx, 2000, out)
    cx[0] = 1500  # lengths are read on the device: the graph follows them
    graph.replay()
    torch.cuda.synchronize()
    check(out[:1], *ref_rows(q[:1], gather(kc, table[0], 1500, 16), gather(vc, table[0], 1500, 16), 1499, 128 ** -0.5))


def test_same_call_twice_gives_the_same_bits(gpu):
    ctx = [9000, 4000]
    kc, vc, table = make_cache(18, ctx, 16, 2, 128, bf16)
    q = randn(19, 70, 8, 128, dtype=bf16)
    a = run_paged(gpu, q, kc, vc, table, [0, 1, 70], ctx, 16)
    assert torch.equal(a, run_paged(gpu, q, kc, vc, table, [0, 1, 70], ctx, 16))


@pytest.mark.parametrize("kv,ctx", [(1, [20000]), (1, [70]), (2, [3000, 9]), (2, [40000, 0, 17, 5000])], ids=str)
@pytest.mark.parametrize("dim", [64, 128])
def test_paged_key_splits(gpu, kv, ctx, dim):
    """Few units: their keys are split over a cluster, or more widely through
    global memory; sequences shorter than the split leave parts without keys."""
    kc, vc, table = make_cache(20, ctx, 64, kv, dim, bf16, fill=float("nan"))
    n = len(ctx)
    run_paged(gpu, randn(21, n, 8 * kv, dim, dtype=bf16), kc, vc, table, list(range(n + 1)), ctx, 64)


def test_prompt_more_units_than_slots(gpu):
    """Long and short sequences in one launch, several units per CTA, some of one
    block and some of many, both masks."""
    lens = [1, 900, 64, 3, 1500, 130, 0, 31] * 4
    q, k, v = (randn(i, sum(lens), h, 64) for i, h in enumerate((8, 8, 8)))
    run_prompt(gpu, q, k, v, cumulated(lens))
    run_prompt(gpu, q, k, v, cumulated(lens), causal=False)


def test_paged_negative_lengths_see_nothing(gpu):
    kc, vc, table = make_cache(22, [40, 40], 16, 2, 128, f16)
    q = randn(23, 4, 8, 128)
    out = torch.full_like(q, 7.0)
    gpu.paged_attention(q, kc, vc, table, ints([0, 2, 4]), ints([-2147483648, 40]), 40, out)
    assert (out[:2] == 0).all()
    check(out[2:], *ref_rows(q[2:], gather(kc, table[1], 40, 16), gather(vc, table[1], 40, 16), 38, 128 ** -0.5))


def test_wide_split_in_a_graph(gpu):
    """A split that goes through scratch: its allocation belongs to the graph."""
    kc, vc, table = make_cache(24, [30000], 64, 1, 128, f16)
    q, cu, ctx = randn(25, 1, 8, 128), ints([0, 1]), ints([30000])
    want = run_paged(gpu, q, kc, vc, table, [0, 1], [30000], 64)
    out = torch.zeros_like(q)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        gpu.paged_attention(q, kc, vc, table, cu, ctx, 30000, out)
    for _ in range(3):
        out.zero_()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, want)
