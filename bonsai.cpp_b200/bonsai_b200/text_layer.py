"""One decoder-style text layer with 1-bit projections, run the way a text
encoder or prompt rewriter in front of the diffuser is served: the prompts of
several requests at once, each with its own low-rank adapters, then single
tokens or chunks behind what the cache holds.

It shows the text-stage operators together: ``prompt_attention`` over packed
prompts, ``paged_append`` / ``paged_attention`` over a paged key/value cache,
and ``b1_gemm_lora`` for every projection, next to the framework's RMS norm
and RoPE.  ``python -m bonsai_b200.text_layer`` runs a batch and checks that
tokens that come one by one get what they get in one prompt.
"""
from __future__ import annotations

import ctypes

import numpy as np

import bonsai_b200 as bb

HEAD_DIM = 128


class TextLayer:
    """h += Wo attention(norm(h)); h += Wdown swiglu(Wup norm(h)), pre-norm, with
    per-head q/k norms and RoPE; all projections B1_0 with adapter slots.
    Weights are seeded random ones."""

    def __init__(self, hidden=512, heads=8, kv_heads=2, mlp=1024, slots=4, max_rank=16, pages=64, page_size=16,
                 theta=1e6, seed=0):
        import torch
        self.torch, self.hidden, self.heads, self.kv_heads = torch, hidden, heads, kv_heads
        self.page_size, self.theta = page_size, theta
        rng = np.random.default_rng(seed)
        q, kv = heads * HEAD_DIM, kv_heads * HEAD_DIM
        shapes = {"q": (q, hidden), "k": (kv, hidden), "v": (kv, hidden), "o": (hidden, q), "up": (2 * mlp, hidden),
                  "down": (hidden, mlp)}
        self.weights, self.adapters = {}, {}
        for name, (n, k) in shapes.items():
            swiglu = 0 if name == "up" else -1
            scale = 1.0 / (np.sqrt(2.0 / np.pi) * np.sqrt(k))  # rows of unit variance on unit inputs
            self.weights[name] = bb.B1Weight(bb.random_b1_packed(n, k, rng, scale), n, k, swiglu)
            self.adapters[name] = bb.LoraSet(n, k, max_rank, slots, swiglu)
        cuda = lambda a: torch.from_numpy(a.astype(np.float32)).cuda()  # noqa: E731
        self.norms = {n: cuda(1 + 0.1 * rng.standard_normal(d)) for n, d in
                      (("attn", hidden), ("mlp", hidden), ("q", HEAD_DIM), ("k", HEAD_DIM))}
        self.k_cache, self.v_cache = (torch.zeros(pages, page_size, kv_heads, HEAD_DIM, dtype=torch.float16,
                                                  device="cuda") for _ in range(2))

    def set_adapter(self, slot: int, rank: int, scale: float, seed: int) -> None:
        """A random adapter of that rank in a slot of every projection."""
        torch = self.torch
        g = torch.Generator(device="cuda").manual_seed(seed)
        for name, w in self.weights.items():
            down = torch.randn(rank, w.in_dim, device="cuda", generator=g).mul_(w.in_dim ** -0.5).half()
            up = torch.randn(w.out_dim, rank, device="cuda", generator=g).mul_(0.2).half()
            self.adapters[name].set(slot, down, up, scale)

    def _norm(self, x, name):
        y = self.torch.empty_like(x)
        dim = self.norms[name].numel()
        bb.check(bb.lib().bonsai_rms_norm_f32(x.data_ptr(), self.norms[name].data_ptr(), x.numel() // dim, dim, 1e-6,
                                              y.data_ptr(), bb.stream_ptr()), "bonsai_rms_norm_f32")
        return y

    def _rope(self, x, cos, sin):
        T, H, D = x.shape
        bb.check(bb.lib().bonsai_rope_2d_f32(x.data_ptr(), cos.data_ptr(), sin.data_ptr(), D, H, T, x.data_ptr(),
                                             bb.stream_ptr()), "bonsai_rope_2d_f32")
        return x

    def _project(self, name, x16, cu, slots, mode, out):
        bb.b1_gemm_lora(x16, self.weights[name], mode, out, self.adapters[name], cu, slots)
        return out

    def forward(self, h, cu, ctx_lens, page_table, slots, max_ctx=None):
        """New tokens h f32 [T][hidden] of several requests (rows [cu[i],
        cu[i + 1]), ctx_lens[i] tokens in all, the new ones included), updated
        in place.  max_ctx None: whole prompts, nothing is cached before them;
        otherwise an upper bound of ctx_lens."""
        torch = self.torch
        T = h.shape[0]
        f32 = lambda *s: torch.empty(*s, device="cuda")  # noqa: E731
        f16 = lambda *s: torch.empty(*s, device="cuda", dtype=torch.float16)  # noqa: E731
        # each token's place in its sequence, and the RoPE tables of the places
        req = torch.searchsorted(cu, torch.arange(T, dtype=torch.int32, device="cuda"), right=True) - 1
        place = (ctx_lens[req] - cu[req + 1] + torch.arange(T, device="cuda")).float()
        cos, sin = f32(T, HEAD_DIM // 2), f32(T, HEAD_DIM // 2)
        axes = (ctypes.c_int * 1)(HEAD_DIM)
        bb.check(bb.lib().bonsai_rope_tables(place.data_ptr(), T, 1, axes, self.theta, cos.data_ptr(), sin.data_ptr(),
                                             bb.stream_ptr()), "bonsai_rope_tables")
        x = self._norm(h, "attn").half()
        q, k = (self._project(n, x, cu, slots, bb.BONSAI_EPI_F32, f32(T, heads * HEAD_DIM)).view(T, heads, HEAD_DIM)
                for n, heads in (("q", self.heads), ("k", self.kv_heads)))
        v = self._project("v", x, cu, slots, bb.BONSAI_EPI_F16, f16(T, self.kv_heads * HEAD_DIM)).view(T, -1, HEAD_DIM)
        q, k = self._rope(self._norm(q, "q"), cos, sin).half(), self._rope(self._norm(k, "k"), cos, sin).half()
        out = f16(T, self.heads, HEAD_DIM)
        bb.paged_append(k, v, self.k_cache, self.v_cache, page_table, cu, ctx_lens)
        if max_ctx is None:
            bb.prompt_attention(q, k, v, cu, out)
        else:
            bb.paged_attention(q, self.k_cache, self.v_cache, page_table, cu, ctx_lens, max_ctx, out)
        self._project("o", out.view(T, -1), cu, slots, bb.BONSAI_EPI_RESID, h)
        x = self._norm(h, "mlp").half()
        x = self._project("up", x, cu, slots, bb.BONSAI_EPI_SWIGLU, f16(T, self.weights["down"].in_dim))
        self._project("down", x, cu, slots, bb.BONSAI_EPI_RESID, h)
        return h


def run_both_ways(lens=(37, 5, 64), new=4, adapters=(0, -1, 1), seed=1, **layer):
    """Prompts of `lens` tokens and `new` more each: once as one prompt each, once
    as the prompt, a chunk of all new tokens but one, and a single token.
    Returns the layer's outputs of the new tokens, both ways, f32
    [requests][new][hidden]."""
    import torch
    bb.init(torch.cuda.current_device())
    m = TextLayer(seed=seed, **layer)
    m.set_adapter(0, 16, 0.5, 3)
    m.set_adapter(1, 7, -1.0, 4)
    n, total = len(lens), [x + new for x in lens]
    ints = lambda v: torch.tensor(v, dtype=torch.int32, device="cuda")  # noqa: E731
    cum = lambda v: ints(np.cumsum([0] + list(v)).tolist())  # noqa: E731
    g = torch.Generator(device="cuda").manual_seed(seed)
    seqs = [torch.randn(t, m.hidden, device="cuda", generator=g) for t in total]
    per = -(-max(total) // m.page_size)
    table = torch.randperm(m.k_cache.shape[0], generator=torch.Generator().manual_seed(seed))[:n * per]
    table, slots = table.int().cuda().view(n, per), ints(list(adapters))
    whole = m.forward(torch.cat(seqs), cum(total), ints(total), table, slots)
    whole = torch.stack([x[-new:] for x in whole.split(total)])
    m.k_cache.fill_(float("nan"))  # nothing of the first way is left to be used
    m.v_cache.fill_(float("nan"))
    m.forward(torch.cat([s[:t] for s, t in zip(seqs, lens)]), cum(lens), ints(list(lens)), table, slots)
    parts = []
    at = list(lens)
    for step in (new - 1, 1):
        rows = torch.cat([s[a:a + step] for s, a in zip(seqs, at)])
        at = [a + step for a in at]
        parts.append(m.forward(rows, cum([step] * n), ints(at), table, slots, max_ctx=max(at)).view(n, step, -1))
    torch.cuda.synchronize()
    return whole, torch.cat(parts, 1)


if __name__ == "__main__":
    a, b = (x.double().flatten() for x in run_both_ways())
    cos = float(a @ b / (a.norm() * b.norm()))
    print(f"new tokens in one prompt and one by one: cos={cos:.7f} max-abs/rms={float((a - b).abs().max() / a.square().mean().sqrt()):.2e}")
    assert cos >= 0.9999 and bb.device_error() == 0
