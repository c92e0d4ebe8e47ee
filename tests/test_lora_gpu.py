"""A B1_0 projection with the low-rank adapters of many requests beside it
(bonsai_b1_gemm_lora) against a plain implementation in f64.

Error bound of an accumulator: the tensor cores add 16 products at a time to an
f32 sum; every addition of a chunk is off by at most 2^-22 of the sum so far
and of the chunk's own magnitude (truncation in place of rounding included).
That is summed chunk by chunk for W x, for A x (whose error passes through
|B|) and for B low.  The epilogue then rounds to f16 once (2^-11 relative,
2^-25 absolute below the normal range) or not at all.
"""
import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu

EPS, U = 2.0 ** -22, 2.0 ** -11


def product(x, w):
    """f64 x w^T and the error bound of its f32 chunked sum."""
    y = torch.zeros(x.shape[0], w.shape[0], dtype=torch.float64, device=x.device)
    bound = torch.zeros_like(y)
    for k in range(0, x.shape[1], 16):
        a, b = x[:, k:k + 16].double(), w[:, k:k + 16].double()
        y += a @ b.T
        bound += EPS * (y.abs() + a.abs() @ b.abs().T)
    return y, bound


class Problem:
    def __init__(self, bb, n, k, ranks, max_rank=None, swiglu=False, seed=0):
        rng = np.random.default_rng(seed)
        g = torch.Generator(device="cuda").manual_seed(seed)
        packed = bb.random_b1_packed(n, k, rng)
        self.bb, self.n, self.k, self.swiglu, self.g = bb, n, k, swiglu, g
        self.w = bb.B1Weight(packed, n, k, 0 if swiglu else -1)
        self.dense = torch.from_numpy(bb.dequant_b1(packed, n, k)).cuda()
        self.lora = bb.LoraSet(n, k, max_rank or max(max(ranks), 1), len(ranks), 0 if swiglu else -1)
        self.down, self.up, self.scale = {}, {}, {}
        for i, r in enumerate(ranks):
            if r:
                self.put(i, r, 0.5 + i)

    def put(self, slot, rank, scale, host=False):
        d = (torch.randn(rank, self.k, device="cuda", generator=self.g) * self.k ** -0.5).half()
        u = (torch.randn(self.n, rank, device="cuda", generator=self.g) * 0.3).half()
        self.down[slot], self.up[slot], self.scale[slot] = d, u, scale
        self.lora.set(slot, d.cpu() if host else d, u.cpu() if host else u, scale)

    def x(self, tokens, ld=None):
        full = torch.randn(tokens, ld or self.k, device="cuda", generator=self.g).half()
        return full[:, :self.k]

    def accumulators(self, x, cu, slots):
        y, bound = product(x, self.dense)
        for i, s in enumerate(slots):
            if s in self.down and cu[i + 1] > cu[i]:
                rows = slice(cu[i], cu[i + 1])
                low, el = product(x[rows], self.down[s])
                low, el = low * self.scale[s], el * abs(self.scale[s])
                add, ea = product(low, self.up[s])
                y[rows] += add
                bound[rows] += ea + (el + EPS * low.abs()) @ self.up[s].double().abs().T + EPS * y[rows].abs()
        return y, bound

    def run(self, x, cu, slots, mode, out, gate=None):
        self.bb.b1_gemm_lora(x, self.w, mode, out, self.lora, ints(cu), ints(slots), gate=gate)
        torch.cuda.synchronize()
        return out


def ints(v):
    return torch.tensor(v, dtype=torch.int32, device="cuda")


def within(out, ref, bound):
    over = float(((out.double() - ref).abs() - bound).max())
    assert over <= 0, f"off by {over} more than the bound"


def check_f32(p, x, cu, slots):
    y, bound = p.accumulators(x, cu, slots)
    within(p.run(x, cu, slots, p.bb.BONSAI_EPI_F32, torch.full((x.shape[0], p.n), 7.0, device="cuda")), y, bound)


@pytest.fixture(params=["auto", "single", "pair"])
def kernel(request, monkeypatch):
    if request.param != "auto":
        monkeypatch.setenv("BONSAI_B1_KERNEL", request.param)


CASES = [([1], [0]), ([1] * 9, [0, 1, 2, 3, -1, 0, 7, 2, 1]), ([17], [2]), ([5, 0, 40, 1, 130], [1, 0, -1, 2, 0]),
         ([300, 20], [0, 1]), ([64, 64, 65], [2, 2, 1]), ([128, 256, 3], [0, 2, 1])]


@pytest.mark.parametrize("lens,slots", CASES, ids=str)
@pytest.mark.parametrize("n,k", [(256, 512), (130, 96), (1000, 2080)])
def test_lora_f32(gpu, kernel, lens, slots, n, k):
    p = Problem(gpu, n, k, [16, 5, 33, 0], seed=n)
    check_f32(p, p.x(sum(lens)), np.cumsum([0] + lens).tolist(), slots)


@pytest.mark.parametrize("rank", [1, 7, 8, 15, 16, 17, 31, 32, 33, 48, 63, 64, 65, 100, 127, 128])
@pytest.mark.parametrize("lens", [[1, 1, 1], [70, 3, 200]], ids=str)
def test_lora_ranks(gpu, rank, lens):
    p = Problem(gpu, 300, 320, [rank, 1], seed=rank)
    check_f32(p, p.x(sum(lens)), np.cumsum([0] + lens).tolist(), [0, 1, 0])


def test_lora_many_requests(gpu):
    lens = [(i * 7) % 5 for i in range(150)]
    p = Problem(gpu, 384, 256, [4, 20, 9, 0, 64])
    check_f32(p, p.x(sum(lens)), np.cumsum([0] + lens).tolist(), [i % 6 - 1 for i in range(150)])


@pytest.mark.parametrize("lens", [[1, 1], [40, 300]], ids=str)
def test_lora_epilogues(gpu, kernel, lens):
    bb = gpu
    cu, slots = np.cumsum([0] + lens).tolist(), [1, 0]
    T = cu[-1]
    p = Problem(bb, 512, 256, [16, 40])
    x = p.x(T)
    y, b = p.accumulators(x, cu, slots)
    out = p.run(x, cu, slots, bb.BONSAI_EPI_F16, torch.empty(T, 512, device="cuda", dtype=torch.float16))
    within(out, y, b + U * (y.abs() + b) + 2.0 ** -25)
    # gelu: slope at most 1.13; the hardware tanh is off by at most 2^-10.9
    out = p.run(x, cu, slots, bb.BONSAI_EPI_GELU, torch.empty(T, 512, device="cuda", dtype=torch.float16))
    ref = torch.nn.functional.gelu(y, approximate="tanh")
    within(out, ref, 1.13 * b + 0.5 * y.abs() * 2.0 ** -10.9 + U * (ref.abs() + b) + 2.0 ** -20)
    resid = torch.randn(T, 512, device="cuda", generator=p.g)
    gate = torch.randn(512, device="cuda", generator=p.g)
    out = p.run(x, cu, slots, bb.BONSAI_EPI_RESID, resid.clone(), gate=gate)
    ref = resid.double() + gate.double() * y
    within(out, ref, gate.abs().double() * b + 2.0 ** -23 * ref.abs())
    out = p.run(x, cu, slots, bb.BONSAI_EPI_RESID, resid.clone())
    within(out, resid.double() + y, b + 2.0 ** -23 * (resid.double() + y).abs())


@pytest.mark.parametrize("lens", [[1, 1], [40, 300]], ids=str)
def test_lora_swiglu_row_order(gpu, kernel, lens):
    cu, slots = np.cumsum([0] + lens).tolist(), [0, 1]
    p = Problem(gpu, 512, 256, [24, 8], swiglu=True)
    x = p.x(cu[-1])
    y, b = p.accumulators(x, cu, slots)
    g, v, bg, bv = y[:, :256], y[:, 256:], b[:, :256], b[:, 256:]
    s = g * torch.sigmoid(g)
    out = p.run(x, cu, slots, gpu.BONSAI_EPI_SWIGLU, torch.empty(cu[-1], 256, device="cuda", dtype=torch.float16))
    bound = 1.1 * bg * (v.abs() + bv) + s.abs() * bv + 2.0 ** -19 * (s * v).abs()
    within(out, s * v, bound + U * ((s * v).abs() + bound) + 2.0 ** -25)


def test_lora_strides_gaps_and_rows_of_no_request(gpu):
    """x and out with longer rows, tokens before, between and after the requests."""
    p = Problem(gpu, 200, 96, [16, 5])
    x = p.x(100, ld=136)
    out = torch.full((100, 256), 7.0, device="cuda")
    cu, slots = [10, 30, 90], [1, 0]
    p.run(x, cu, slots, gpu.BONSAI_EPI_F32, out[:, :200])
    within(out[:, :200], *p.accumulators(x, cu, slots))
    assert (out[:, 200:] == 7).all()


def test_lora_slots_change(gpu):
    p = Problem(gpu, 256, 128, [16, 0], max_rank=40)
    x, cu = p.x(60), [0, 30, 60]
    check_f32(p, x, cu, [0, 1])
    p.put(1, 40, -2.0, host=True)
    check_f32(p, x, cu, [0, 1])
    p.put(0, 3, 1.0)  # a smaller rank leaves nothing of the larger one
    check_f32(p, x, cu, [0, 1])
    p.lora.clear(1)
    del p.down[1]
    check_f32(p, x, cu, [0, 1])


def test_lora_without_requests_is_the_projection(gpu):
    p = Problem(gpu, 256, 128, [16])
    x = p.x(50)
    a, b = (torch.empty(50, 256, device="cuda") for _ in range(2))
    p.run(x, [0], [], gpu.BONSAI_EPI_F32, a)
    gpu.b1_gemm(x, p.w, gpu.BONSAI_EPI_F32, b)
    assert torch.equal(a, b)
    p.run(x, [0, 50], [-1], gpu.BONSAI_EPI_F32, a)
    assert torch.equal(a, b)


def test_lora_stays_with_its_token(gpu):
    """A non-finite token spoils its own row only, whatever shares its tile."""
    p = Problem(gpu, 256, 128, [16, 4])
    cu, slots = [0, 33, 34, 80], [0, 1, 0]
    x = p.x(80)
    x[33] = float("nan")
    out = p.run(x, cu, slots, gpu.BONSAI_EPI_F32, torch.empty(80, 256, device="cuda"))
    assert out[33].isnan().all()
    x[33] = 0
    y, b = p.accumulators(x, cu, slots)
    keep = [i for i in range(80) if i != 33]
    within(out[keep], y[keep], b[keep])


def test_lora_on_another_stream_and_repeatable(gpu):
    p = Problem(gpu, 512, 1024, [16, 64])
    x, cu, slots = p.x(300), ints([0, 100, 300]), ints([1, 0])
    want = p.run(x, [0, 100, 300], [1, 0], gpu.BONSAI_EPI_F32, torch.empty(300, 512, device="cuda"))
    side = torch.cuda.Stream()
    out = torch.zeros(300, 512, device="cuda")
    side.wait_stream(torch.cuda.current_stream())
    gpu.b1_gemm_lora(x, p.w, gpu.BONSAI_EPI_F32, out, p.lora, cu, slots, stream=side)
    side.synchronize()
    assert torch.equal(out, want)


def test_lora_refusals(gpu):
    bb = gpu
    import ctypes
    h = ctypes.c_void_p()
    L = bb.lib()
    for args, code in (((0, 64, 16, 1, -1), -1), ((64, 65, 16, 1, -1), -1), ((64, 64, 0, 1, -1), -2),
                       ((64, 64, 129, 1, -1), -2), ((64, 64, 16, 0, -1), -1), ((64, 64, 16, 1, 3), -1),
                       ((64, 64, 16, 1, 64), -1)):
        assert L.bonsai_lora_create(*args, ctypes.byref(h)) == code and not h
    assert L.bonsai_lora_create(64, 64, 16, 1, -1, None) == -1
    p = Problem(bb, 64, 64, [16])
    d, u = p.down[0], p.up[0]
    for slot, rank, down, up, scale in ((1, 16, d, u, 1.0), (-1, 16, d, u, 1.0), (0, 17, d, u, 1.0), (0, -1, d, u, 1.0),
                                        (0, 16, None, u, 1.0), (0, 16, d, u, float("nan"))):
        assert L.bonsai_lora_set(p.lora.handle, slot, None if down is None else down.data_ptr(), up.data_ptr(), rank,
                                 scale, None) == -1
    x, out = p.x(4), torch.empty(4, 64, device="cuda")
    cu, slots = ints([0, 4]), ints([0])

    def call(tokens=4, w=p.w.handle, mode=0, o=out.data_ptr(), ld=64, s=p.lora.handle, c=cu.data_ptr(),
             a=slots.data_ptr(), n=1, xp=x.data_ptr(), ldx=64):
        return L.bonsai_b1_gemm_lora(xp, ldx, tokens, w, mode, o, ld, None, s, c, a, n, None)
    other = bb.LoraSet(128, 64, 16, 1)
    assert call(w=None) == -1 and call(s=None) == -1 and call(s=other.handle) == -1
    assert call(tokens=-1) == -1 and call(n=-1) == -1 and call(c=None) == -1 and call(a=None) == -1
    assert call(mode=9) == -1 and call(mode=bb.BONSAI_EPI_SWIGLU) == -1 and call(o=None) == -1 and call(ld=63) == -1
    assert call(xp=None) == -1 and call(ldx=60) == -1 and call(xp=x.data_ptr() + 2) == -1
    assert call(tokens=0, c=None, o=None) == 0 and call() == 0
    with pytest.raises(bb.BonsaiError):
        p.lora.set(0, d.float(), u, 1.0)
    with pytest.raises(bb.BonsaiError):
        p.lora.set(0, d, u[:63].contiguous(), 1.0)


@pytest.mark.parametrize("per", [1, 20])
def test_lora_more_tiles_than_sms(gpu, per):
    """Both forms with several tiles per CTA."""
    n = 400 // per * (1 if per == 1 else 4)
    p = Problem(gpu, 4096, 128, [16, 5, 0, 33])
    cu = [i * per for i in range(n + 1)]
    check_f32(p, p.x(cu[-1]), cu, [i % 5 - 1 for i in range(n)])


@pytest.mark.parametrize("lens", [[1, 1, 1], [100, 30]], ids=str)
def test_lora_in_a_graph(gpu, lens):
    p = Problem(gpu, 512, 1024, [16, 64])
    cu, slots = np.cumsum([0] + lens).tolist(), [1, 0, 1][:len(lens)]
    x, c, s = p.x(cu[-1]), ints(cu), ints(slots)
    want = p.run(x, cu, slots, gpu.BONSAI_EPI_F32, torch.empty(cu[-1], 512, device="cuda"))
    out = torch.zeros_like(want)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        gpu.b1_gemm_lora(x, p.w, gpu.BONSAI_EPI_F32, out, p.lora, c, s)
    for _ in range(3):
        out.zero_()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, want)
