"""ctypes binding of libbonsai_cuda.so (include/bonsai_cuda.h).

This is the Python-side view of the C ABI that tests and the benchmark use.
It mirrors the reference's operator surface: ``b1_linear_f32`` is the
drop-in for ``b1_linear_f32_f32`` (src/b1_0_kernel.h:37-288), ``rope_2d_f32``
for ``rope_2d_fwd_f32`` (src/b1_0_kernel.h:309-361), and the model entry
points for one pass of ``build_diffuser_graph`` (src/diffuser_graph.cpp:231-561).

Device tensors are passed as raw pointers (``tensor.data_ptr()``); PyTorch is
used only to own device memory and streams.  There is no CPU fallback: if the
shared library is missing or fails to load, every call raises.
"""
from __future__ import annotations

import ctypes
import os
import struct
import threading
from pathlib import Path

import numpy as np

PKG_DIR = Path(__file__).resolve().parent
LIB_PATH = PKG_DIR.parent / "lib" / "libbonsai_cuda.so"

BONSAI_EPI_F32 = 0
BONSAI_EPI_F16 = 1
BONSAI_EPI_GELU = 2
BONSAI_EPI_RESID = 3
BONSAI_EPI_SWIGLU = 5

PRESET_KLEIN4B = 0
PRESET_FLUX1 = 1

_lib = None

_c_int = ctypes.c_int
_c_ll = ctypes.c_longlong
_vp = ctypes.c_void_p
_fp = ctypes.c_float

# name -> (restype, argtypes); every symbol declared in include/bonsai_cuda.h
SIGNATURES = {
    "bonsai_last_error": (ctypes.c_char_p, []),
    "bonsai_init": (_c_int, [_c_int]),
    "bonsai_device_error": (_c_int, []),
    "bonsai_shutdown": (_c_int, []),
    "bonsai_count_nonfinite": (_c_int, [_vp, _c_ll, ctypes.POINTER(_c_ll), _vp]),
    "bonsai_launch_count": (_c_ll, []),
    "bonsai_debug_stall_next_gemm": (_c_int, []),
    "bonsai_debug_tmem_shares": (_c_int, [ctypes.POINTER(_c_int), ctypes.POINTER(_c_int), _c_int]),
    "bonsai_profile_start": (_c_int, []),
    "bonsai_profile_stop": (_c_int, [ctypes.c_char_p, _c_int]),
    "bonsai_b1_upload": (_c_int, [_vp, _c_int, _c_int, _c_int, ctypes.POINTER(_vp)]),
    "bonsai_b1_free": (_c_int, [_vp]),
    "bonsai_b1_shape": (_c_int, [_vp, ctypes.POINTER(_c_int), ctypes.POINTER(_c_int)]),
    "bonsai_b1_linear_f32": (_c_int, [_vp, _c_int, _vp, _vp, _vp]),
    "bonsai_b1_linear_f32_noalloc": (_c_int, [_vp, _c_int, _vp, _vp, _vp]),
    "bonsai_b1_gemm": (_c_int, [_vp, _c_ll, _c_int, _vp, _c_int, _vp, _c_ll, _vp, _vp]),
    "bonsai_lora_create": (_c_int, [_c_int, _c_int, _c_int, _c_int, _c_int, ctypes.POINTER(_vp)]),
    "bonsai_lora_set": (_c_int, [_vp, _c_int, _vp, _vp, _c_int, _fp, _vp]),
    "bonsai_lora_free": (_c_int, [_vp]),
    "bonsai_b1_gemm_lora": (_c_int, [_vp, _c_ll, _c_int, _vp, _c_int, _vp, _c_ll, _vp, _vp, _vp, _vp, _c_int, _vp]),
    "bonsai_rope_2d_f32": (_c_int, [_vp, _vp, _vp, _c_int, _c_int, _c_int, _vp, _vp]),
    "bonsai_rope_tables": (_c_int, [_vp, _c_int, _c_int, _vp, _fp, _vp, _vp, _vp]),
    "bonsai_rms_norm_f32": (_c_int, [_vp, _vp, _c_int, _c_int, _fp, _vp, _vp]),
    "bonsai_linear_f32": (_c_int, [_vp, _c_int, _c_int, _vp, _vp, _c_int, _vp, _vp]),
    "bonsai_ln_modulate": (_c_int, [_vp, _c_int, _c_int, _vp, _vp, _fp, _vp, _c_ll, _vp]),
    "bonsai_ln_modulate_f32": (_c_int, [_vp, _c_int, _c_int, _vp, _vp, _fp, _vp, _vp]),
    "bonsai_joint_attention": (_c_int, [_vp, _vp, _vp, _c_int, _c_int, _c_int, _fp, _vp, _c_ll, _vp]),
    "bonsai_qk_norm_rope": (_c_int, [_vp, _c_int, _c_int, _c_int, _vp, _vp, _c_int, _fp, _vp, _vp, _vp]),
    "bonsai_prompt_attention": (_c_int, [_vp, _vp, _vp, _vp, _c_int, _c_int, _c_int, _c_int, _c_int,
                                         _c_int, _c_int, _fp, _vp, _vp]),
    "bonsai_paged_append": (_c_int, [_vp, _vp, _vp, _vp, _vp, _c_ll, _c_int, _vp, _vp, _c_int, _c_int,
                                     _c_int, _c_int, _vp]),
    "bonsai_paged_attention": (_c_int, [_vp, _vp, _vp, _vp, _c_ll, _c_int, _vp, _vp, _c_int, _c_int,
                                        _c_int, _c_int, _c_int, _c_int, _c_int, _fp, _vp, _vp]),
    "bonsai_paged_append_quant": (_c_int, [_vp, _vp, _vp, _vp, _vp, _c_ll, _c_int, _vp, _vp, _c_int, _c_int,
                                           _c_int, _c_int, _c_int, _vp]),
    "bonsai_paged_read_quant": (_c_int, [_vp, _vp, _vp, _c_ll, _c_int, _vp, _vp, _c_int, _c_int, _c_int,
                                         _c_int, _c_int, _vp, _vp, _vp]),
    "bonsai_paged_attention_quant": (_c_int, [_vp, _vp, _vp, _vp, _c_ll, _c_int, _vp, _vp, _c_int, _c_int,
                                              _c_int, _c_int, _c_int, _c_int, _c_int, _c_int, _fp, _vp, _vp]),
    "bonsai_sample_tokens": (_c_int, [_vp, _c_ll, _c_int, _c_int, _c_int, _vp, _vp, _vp, _vp, _vp, _vp, _vp, _vp]),
    "bonsai_dit_create": (_c_int, [_vp, ctypes.POINTER(_vp)]),
    "bonsai_dit_destroy": (_c_int, [_vp]),
    "bonsai_dit_forward": (_c_int, [_vp, _vp, _vp, _vp, _fp, _vp, _vp]),
    "bonsai_dit_forward_host": (_c_int, [_vp, _vp, _vp, _vp, _fp, _vp, _vp]),
    "bonsai_dit_set_state": (_c_int, [_vp, _vp, _vp, _vp]),
    "bonsai_dit_get_state": (_c_int, [_vp, _vp, _vp]),
    "bonsai_dit_double_block": (_c_int, [_vp, _c_int, _vp]),
    "bonsai_dit_single_block": (_c_int, [_vp, _c_int, _vp]),
    "bonsai_dit_weight": (_c_ll, [_vp, ctypes.c_char_p, _vp, _c_ll]),
    "bonsai_dit_set_weight": (_c_int, [_vp, ctypes.c_char_p, _vp, _c_ll]),
    "bonsai_dit_load_safetensors": (_c_int, [_vp, ctypes.c_char_p]),
    "bonsai_safetensors_list": (_c_int, [ctypes.c_char_p, ctypes.c_char_p, _c_int]),
    "bonsai_dit_sample": (_c_int, [_vp, _vp, _vp, _vp, _c_int, _vp, _vp]),
    "bonsai_dit_set_partition": (_c_int, [_vp, _c_int, _c_int]),
    "bonsai_dit_buffer": (_c_int, [_vp, ctypes.c_char_p, ctypes.POINTER(_vp), ctypes.POINTER(_c_ll)]),
    "bonsai_dit_begin": (_c_int, [_vp, _vp, _vp, _vp, _fp, _vp]),
    "bonsai_dit_phase": (_c_int, [_vp, _c_int, _c_int, _c_int, _vp]),
    "bonsai_dit_end": (_c_int, [_vp, _vp, _vp]),
    "bonsai_dit_set_peers": (_c_int, [_vp, ctypes.POINTER(_vp), ctypes.POINTER(_vp), _c_int]),
    "bonsai_dit_ipc_handles": (_c_int, [_vp, _vp]),
    "bonsai_dit_open_peers": (_c_int, [_vp, _vp, _c_int]),
    "bonsai_dit_set_qkv_peers": (_c_int, [_vp, ctypes.POINTER(_vp), _c_int]),
    "bonsai_dit_ipc_handle": (_c_int, [_vp, ctypes.c_char_p, _vp]),
    "bonsai_dit_open_qkv_peers": (_c_int, [_vp, _vp, _c_int]),
    "bonsai_dit_set_flag_peers": (_c_int, [_vp, ctypes.POINTER(_vp), _c_int]),
    "bonsai_dit_open_flag_peers": (_c_int, [_vp, _vp, _c_int]),
    "bonsai_dit_barrier": (_c_int, [_vp, _vp]),
    "bonsai_vae_create": (_c_int, [_c_int, _c_int, ctypes.c_ulonglong, ctypes.POINTER(_vp)]),
    "bonsai_vae_destroy": (_c_int, [_vp]),
    "bonsai_vae_load_safetensors": (_c_int, [_vp, ctypes.c_char_p]),
    "bonsai_vae_decode": (_c_int, [_vp, _vp, _vp, _vp]),
    "bonsai_vae_decode_host": (_c_int, [_vp, _vp, _vp, _vp]),
    "bonsai_vae_rgb8": (_c_int, [_vp, _c_int, _c_int, _vp, _vp]),
    "bonsai_vae_info": (_c_int, [_vp, ctypes.POINTER(_c_int), ctypes.POINTER(_c_int)]),
    "bonsai_conv2d_nhwc": (_c_int, [_vp, _c_int, _c_int, _c_int, _c_int, _vp, _c_int, _c_int, _vp, _vp,
                                    _vp, _vp]),
}


class BonsaiError(RuntimeError):
    pass


def lib() -> ctypes.CDLL:
    """Load the shared library (raises if it is absent: there is no fallback)."""
    global _lib
    if _lib is None:
        if not LIB_PATH.exists():
            raise BonsaiError(
                f"{LIB_PATH} not found: build it with `make -C bonsai.cpp_b200` "
                "(or __graft_entry__.build())")
        L = ctypes.CDLL(str(LIB_PATH))
        missing = []
        for name, (res, args) in SIGNATURES.items():
            try:
                fn = getattr(L, name)
            except AttributeError:
                missing.append(name)
                continue
            fn.restype = res
            fn.argtypes = args
        L.missing_symbols = missing
        _lib = L
    return _lib


def check(rc: int, what: str = "") -> None:
    if rc != 0:
        msg = lib().bonsai_last_error().decode(errors="replace")
        raise BonsaiError(f"{what or 'bonsai call'} failed with {rc}: {msg}")


def stream_ptr(stream=None) -> int:
    import torch
    s = stream if stream is not None else torch.cuda.current_stream()
    return int(s.cuda_stream)


def init(device: int = 0) -> None:
    check(lib().bonsai_init(device), "bonsai_init")


def device_error() -> int:
    return int(lib().bonsai_device_error())


def launch_count() -> int:
    return int(lib().bonsai_launch_count())


def profile_start() -> None:
    check(lib().bonsai_profile_start(), "bonsai_profile_start")


def profile_stop() -> dict:
    import json
    buf = ctypes.create_string_buffer(1 << 16)
    n = lib().bonsai_profile_stop(buf, len(buf))
    if n < 0:
        check(n, "bonsai_profile_stop")
    return json.loads(buf.value.decode())


class B1Weight:
    """Device B1_0 weight uploaded from the reference's packed bytes."""

    def __init__(self, packed: np.ndarray, out_dim: int, in_dim: int, swiglu_from: int = -1):
        packed = np.ascontiguousarray(packed, dtype=np.uint8)
        assert packed.size == out_dim * (in_dim // 32) * 6, "packed size mismatch"
        h = _vp()
        check(lib().bonsai_b1_upload(packed.ctypes.data, out_dim, in_dim, swiglu_from,
                                     ctypes.byref(h)), "bonsai_b1_upload")
        self.handle = h
        self.out_dim = out_dim
        self.in_dim = in_dim

    def free(self):
        if self.handle:
            lib().bonsai_b1_free(self.handle)
            self.handle = None

    def __del__(self):
        try:
            self.free()
        except Exception:
            pass


def b1_linear_f32(act, w: B1Weight, out, stream=None) -> None:
    """Drop-in b1_linear_f32_f32: act f32 [T][K] -> out f32 [T][N] (device tensors)."""
    assert act.is_contiguous() and out.is_contiguous()
    T = act.shape[0]
    check(lib().bonsai_b1_linear_f32(act.data_ptr(), T, w.handle, out.data_ptr(),
                                     stream_ptr(stream)), "bonsai_b1_linear_f32")


def b1_gemm(x16, w: B1Weight, mode: int, out, gate=None, stream=None) -> None:
    """Fused-epilogue GEMM on f16 activations x16 [T][ldx]."""
    T = x16.shape[0]
    check(lib().bonsai_b1_gemm(x16.data_ptr(), x16.stride(0), T, w.handle, mode,
                               out.data_ptr(), out.stride(0),
                               gate.data_ptr() if gate is not None else None,
                               stream_ptr(stream)), "bonsai_b1_gemm")


class LoraSet:
    """Low-rank adapters for one B1_0 projection of out_dim x in_dim: n_slots
    slots of rank <= max_rank (swiglu_from as the B1Weight's)."""

    def __init__(self, out_dim: int, in_dim: int, max_rank: int, n_slots: int, swiglu_from: int = -1):
        h = _vp()
        check(lib().bonsai_lora_create(out_dim, in_dim, max_rank, n_slots, swiglu_from, ctypes.byref(h)),
              "bonsai_lora_create")
        self.handle = h
        self.out_dim, self.in_dim, self.max_rank, self.n_slots = out_dim, in_dim, max_rank, n_slots

    def set(self, slot: int, down, up, scale: float, stream=None) -> None:
        """down f16 [rank][in_dim], up f16 [out_dim][rank]: contiguous tensors, host
        or cuda; y += scale * up (down x)."""
        import torch
        rank = down.shape[0]
        if down.dtype != torch.float16 or up.dtype != torch.float16:
            raise BonsaiError("adapters must be f16")
        if tuple(down.shape) != (rank, self.in_dim) or tuple(up.shape) != (self.out_dim, rank):
            raise BonsaiError(f"adapter {tuple(down.shape)}, {tuple(up.shape)} does not fit "
                              f"{self.out_dim} x {self.in_dim}")
        if not (down.is_contiguous() and up.is_contiguous()):
            raise BonsaiError("adapters must be contiguous")
        check(lib().bonsai_lora_set(self.handle, slot, down.data_ptr(), up.data_ptr(), rank, float(scale),
                                    stream_ptr(stream)), "bonsai_lora_set")

    def clear(self, slot: int, stream=None) -> None:
        check(lib().bonsai_lora_set(self.handle, slot, None, None, 0, 0.0, stream_ptr(stream)), "bonsai_lora_set")

    def free(self):
        if getattr(self, "handle", None):
            lib().bonsai_lora_free(self.handle)
            self.handle = None

    def __del__(self):
        try:
            self.free()
        except Exception:
            pass


def b1_gemm_lora(x16, w: B1Weight, mode: int, out, lora: LoraSet, cu_tokens, slots, gate=None, stream=None) -> None:
    """b1_gemm with each request's adapter beside it: request i has the tokens
    [cu_tokens[i], cu_tokens[i + 1]) and the adapter slots[i] (-1: none); cuda int32."""
    dev, st, _ = _text_place(x16)
    n = slots.shape[0]
    if cu_tokens.shape[0] != n + 1:
        raise BonsaiError(f"cu_tokens {tuple(cu_tokens.shape)} and slots [{n}] do not match")
    T, K = x16.shape
    sx, so = x16.stride(), out.stride()
    f16 = mode in (BONSAI_EPI_F16, BONSAI_EPI_GELU, BONSAI_EPI_SWIGLU)
    if x16.dtype is not _text_torch.float16 or K != w.in_dim or K > 1 and sx[1] != 1:
        raise BonsaiError(f"x must be f16 [tokens][{w.in_dim}] with contiguous rows, got {x16.dtype} {tuple(x16.shape)}")
    width = w.out_dim // 2 if mode == BONSAI_EPI_SWIGLU else w.out_dim
    if out.dtype is not (_text_torch.float16 if f16 else _text_torch.float32) or out.shape != (T, width) \
            or out.get_device() != dev or width > 1 and so[1] != 1:
        raise BonsaiError(f"out {out.dtype} {tuple(out.shape)} does not fit the mode, {T} tokens and {width} outputs")
    if gate is not None and (gate.dtype is not _text_torch.float32 or gate.get_device() != dev
                             or gate.numel() < w.out_dim or not gate.is_contiguous()):
        raise BonsaiError(f"gate must be contiguous f32 of {w.out_dim} values on the current device, "
                          f"got {gate.dtype} {tuple(gate.shape)} on {gate.device}")
    check(lib().bonsai_b1_gemm_lora(
        x16.data_ptr(), sx[0] if T > 1 else K, T, w.handle, mode, out.data_ptr(), so[0] if T > 1 else width,
        gate.data_ptr() if gate is not None else None, lora.handle, _text_ints(dev, "cu_tokens", cu_tokens),
        _text_ints(dev, "slots", slots), n, st if stream is None else stream.cuda_stream), "bonsai_b1_gemm_lora")


def linear_f32(x, W, bias, out, stream=None) -> None:
    """f32 edge linear: out[t][o] = x[t] . W[o] (+ bias[o]); device tensors."""
    T, K = x.shape
    N = W.shape[0]
    assert x.is_contiguous() and W.is_contiguous() and out.is_contiguous()
    check(lib().bonsai_linear_f32(x.data_ptr(), T, K, W.data_ptr(),
                                  bias.data_ptr() if bias is not None else None, N,
                                  out.data_ptr(), stream_ptr(stream)), "bonsai_linear_f32")


def count_nonfinite(x, stream=None) -> int:
    """Number of NaN / Inf values in a device f32 tensor."""
    n = _c_ll()
    check(lib().bonsai_count_nonfinite(x.data_ptr(), x.numel(), ctypes.byref(n), stream_ptr(stream)),
          "bonsai_count_nonfinite")
    return int(n.value)


def safetensors_list(path) -> list:
    """[(name, dtype, shape tuple, begin, end)] of a .safetensors file (host only)."""
    p = str(path).encode()
    n = lib().bonsai_safetensors_list(p, None, 0)
    if n < 0:
        check(n, "bonsai_safetensors_list")
    buf = ctypes.create_string_buffer(n + 1)
    check(0 if lib().bonsai_safetensors_list(p, buf, n + 1) == n else -1, "bonsai_safetensors_list")
    out = []
    for line in buf.value.decode().splitlines():
        name, dtype, shape, b, e = line.split("\t")
        out.append((name, dtype, tuple(int(d) for d in shape.split(",") if d), int(b), int(e)))
    return out


def shutdown() -> None:
    check(lib().bonsai_shutdown(), "bonsai_shutdown")


def joint_attention(q, k, v, out, scale=None, stream=None) -> None:
    """softmax(Q K^T * scale) V per head: q/k/v f16 [H][L][128] head-major,
    out f16 [L][ld >= H*128] token-major (head h at columns h*128)."""
    H, L, D = q.shape
    check(lib().bonsai_joint_attention(q.data_ptr(), k.data_ptr(), v.data_ptr(), H, L, D,
                                       float(scale if scale is not None else D ** -0.5),
                                       out.data_ptr(), out.stride(0), stream_ptr(stream)),
          "bonsai_joint_attention")


# ----------------------------------------------------------------- text stage
class HeadsDesc(ctypes.Structure):
    """bonsai_heads_t: a 16-bit [token][head][dim] tensor with strides."""
    _fields_ = [("data", _vp), ("stride_token", _c_ll), ("stride_head", _c_ll)]


class PagesDesc(ctypes.Structure):
    """bonsai_pages_t: one side of a paged cache [page][slot][head][dim]."""
    _fields_ = [("data", _vp), ("stride_page", _c_ll), ("stride_token", _c_ll), ("stride_head", _c_ll),
                ("n_pages", _c_int), ("page_size", _c_int)]


# These calls run once per layer and token, so their checks are kept to a few
# microseconds: plain comparisons of what the tensors say of themselves, and
# descriptors packed into a buffer of the calling thread.
_text_torch = None
_HEADS = struct.Struct("Qqq")       # bonsai_heads_t
_PAGES = struct.Struct("Qqqqii")    # bonsai_pages_t


class _TextDescs(threading.local):
    """Up to four descriptors, 40 bytes apart, and their addresses."""

    def __init__(self):
        self.buf = bytearray(160)
        base = ctypes.addressof((ctypes.c_char * 160).from_buffer(self.buf))
        self.at = (base, base + 40, base + 80, base + 120)


_text_descs = _TextDescs()


def _text_place(first):
    """(device index of `first`, which has to be the current one, its current stream, descriptors)."""
    global _text_torch
    if _text_torch is None:
        import torch
        _text_torch = torch
    dev = first.get_device()
    if dev < 0 or dev != _text_torch._C._cuda_getDevice():
        raise BonsaiError(f"tensors must be on the current cuda device, got {first.device}")
    return dev, _text_torch._C._cuda_getCurrentRawStream(dev), _text_descs


def _text_dtype(dtype) -> int:
    if dtype is _text_torch.float16:
        return 0
    if dtype is _text_torch.bfloat16:
        return 1
    raise BonsaiError(f"text attention takes f16 or bf16 tensors, got {dtype}")


def _text_ints(dev, name, t):
    if t.dtype is not _text_torch.int32 or t.get_device() != dev or not t.is_contiguous():
        raise BonsaiError(f"{name} must be contiguous int32 on the current device")
    return t.data_ptr()


def _heads(d, i, t, dtype, dev, dim):
    """Descriptor i: a [token][head][dim] tensor."""
    s = t.stride()
    if len(s) != 3 or t.dtype is not dtype or t.get_device() != dev or s[2] != 1 and dim > 1:
        raise BonsaiError(f"want a [token][head][dim] tensor of {dtype} with contiguous dims on the current device, "
                          f"got {t.dtype} {tuple(t.shape)} {tuple(s)} on {t.device}")
    _HEADS.pack_into(d.buf, 40 * i, t.data_ptr(), s[0], s[1])
    return d.at[i]


def _pages(d, i, t, dtype, dev, dim):
    """Descriptor i: a [page][slot][head][dim] tensor."""
    s, n = t.stride(), t.shape
    if len(s) != 4 or t.dtype is not dtype or t.get_device() != dev or s[3] != 1 and dim > 1:
        raise BonsaiError(f"want a [page][slot][head][dim] cache of {dtype} with contiguous dims on the current device, "
                          f"got {t.dtype} {tuple(n)} {tuple(s)} on {t.device}")
    _PAGES.pack_into(d.buf, 40 * i, t.data_ptr(), s[0], s[1], s[2], n[0], n[1])
    return d.at[i]


def _same(what, a, b):
    if a != b:
        raise BonsaiError(f"{what} do not match: {tuple(a)}, {tuple(b)}")


def prompt_attention(q, k, v, cu_seqlens, out, scale=None, causal=True, stream=None) -> None:
    """Attention over packed prompts: q, out [T][H][D], k, v [T][Hkv][D] (f16 or
    bf16, any token / head strides that are multiples of 8), cu_seqlens cuda
    int32 [n + 1]; sequence s has the rows [cu_seqlens[s], cu_seqlens[s + 1])."""
    dev, st, d = _text_place(q)
    dtype, shape, kshape = q.dtype, q.shape, k.shape
    _same("q and out", shape, out.shape)
    _same("k and v", kshape, v.shape)
    T, H, D = shape
    if kshape[0] != T or kshape[2] != D:
        raise BonsaiError(f"k {tuple(kshape)} does not fit q {tuple(shape)}")
    check(lib().bonsai_prompt_attention(
        _heads(d, 0, q, dtype, dev, D), _heads(d, 1, k, dtype, dev, D), _heads(d, 2, v, dtype, dev, D),
        _text_ints(dev, "cu_seqlens", cu_seqlens), cu_seqlens.shape[0] - 1, T, H, kshape[1], D, _text_dtype(dtype),
        1 if causal else 0, D ** -0.5 if scale is None else scale, _heads(d, 3, out, dtype, dev, D),
        st if stream is None else stream.cuda_stream), "bonsai_prompt_attention")


def _table_args(dev, page_table, cu_q, ctx_lens):
    """(page_table, row stride, width, cu_q, ctx_lens, sequences) as the C calls take them."""
    shape, s = page_table.shape, page_table.stride()
    n = ctx_lens.numel()
    if len(shape) != 2 or shape[0] != n or cu_q.numel() != n + 1:
        raise BonsaiError(f"page_table {tuple(shape)}, cu_q {tuple(cu_q.shape)} and ctx_lens [{n}] do not match")
    if page_table.dtype is not _text_torch.int32 or page_table.get_device() != dev or s[1] != 1 and shape[1] > 1:
        raise BonsaiError("page_table must be int32 with unit stride along a row on the current device")
    return (page_table.data_ptr(), s[0] if n > 1 else shape[1], shape[1], _text_ints(dev, "cu_q", cu_q),
            _text_ints(dev, "ctx_lens", ctx_lens), n)


def paged_append(k, v, k_cache, v_cache, page_table, cu_q, ctx_lens, stream=None) -> None:
    """Write new keys / values [T][Hkv][D] into the cache [pages][page_size][Hkv][D]:
    token i of sequence s (rows [cu_q[s], cu_q[s + 1])) goes to place
    ctx_lens[s] - q_len + i of its page_table row [n][width]."""
    dev, st, d = _text_place(k)
    dtype, shape, cshape = k.dtype, k.shape, k_cache.shape
    _text_dtype(dtype)
    _same("k and v", shape, v.shape)
    _same("the caches", cshape, v_cache.shape)
    T, Hk, D = shape
    if cshape[2] != Hk or cshape[3] != D:
        raise BonsaiError(f"caches {tuple(cshape)} do not fit k {tuple(shape)}")
    check(lib().bonsai_paged_append(
        _heads(d, 0, k, dtype, dev, D), _heads(d, 1, v, dtype, dev, D), _pages(d, 2, k_cache, dtype, dev, D),
        _pages(d, 3, v_cache, dtype, dev, D), *_table_args(dev, page_table, cu_q, ctx_lens), T, Hk, D,
        st if stream is None else stream.cuda_stream), "bonsai_paged_append")


def paged_attention(q, k_cache, v_cache, page_table, cu_q, ctx_lens, max_ctx, out, scale=None,
                    stream=None) -> None:
    """Causal attention of new tokens q [T][H][D] over the paged cache
    [pages][page_size][Hkv][D], the new tokens' own keys appended before;
    max_ctx: an upper bound of ctx_lens (only sets how the work is split)."""
    dev, st, d = _text_place(q)
    dtype, shape, cshape = q.dtype, q.shape, k_cache.shape
    _same("q and out", shape, out.shape)
    _same("the caches", cshape, v_cache.shape)
    T, H, D = shape
    if cshape[3] != D:
        raise BonsaiError(f"caches {tuple(cshape)} do not fit q {tuple(shape)}")
    check(lib().bonsai_paged_attention(
        _heads(d, 0, q, dtype, dev, D), _pages(d, 1, k_cache, dtype, dev, D), _pages(d, 2, v_cache, dtype, dev, D),
        *_table_args(dev, page_table, cu_q, ctx_lens), T, max_ctx, H, cshape[2], D, _text_dtype(dtype),
        D ** -0.5 if scale is None else scale, _heads(d, 3, out, dtype, dev, D),
        st if stream is None else stream.cuda_stream), "bonsai_paged_attention")


class QuantPagesDesc(ctypes.Structure):
    """bonsai_quant_pages_t: one side of a quantised cache."""
    _fields_ = [("codes", _vp), ("stride_page", _c_ll), ("stride_token", _c_ll), ("stride_head", _c_ll),
                ("scales", _vp), ("scale_page", _c_ll), ("scale_token", _c_ll), ("scale_head", _c_ll),
                ("n_pages", _c_int), ("page_size", _c_int), ("format", _c_int)]


class QuantPages:
    """Keys or values of a paged cache in 8 ("i8") or 4 ("i4") bits: codes uint8
    [pages][page_size][Hkv][D or D / 2] and block exponents scales uint8
    [pages][page_size][Hkv][D / 32], any strides of the first three dimensions
    (codes: multiples of 16 bytes).  The format is in include/bonsai_cuda.h."""

    FORMATS = {"i8": 0, "i4": 1}

    def __init__(self, codes, scales, fmt="i8"):
        import torch
        if fmt not in self.FORMATS:
            raise BonsaiError(f"unknown cache format {fmt!r}: one of {sorted(self.FORMATS)}")
        if codes.dtype is not torch.uint8 or scales.dtype is not torch.uint8 or codes.dim() != 4 or scales.dim() != 4:
            raise BonsaiError("codes and scales must be uint8 [page][slot][head][bytes] tensors")
        dim = codes.shape[3] * (1 if fmt == "i8" else 2)
        if scales.shape != (*codes.shape[:3], dim // 32) or dim % 32:
            raise BonsaiError(f"scales {tuple(scales.shape)} do not fit codes {tuple(codes.shape)} of format {fmt}")
        if codes.stride(3) != 1 or scales.stride(3) != 1 or codes.device != scales.device or not codes.is_cuda:
            raise BonsaiError("codes and scales must be on one cuda device, with the bytes of a row side by side")
        self.codes, self.scales, self.format, self.head_dim = codes, scales, fmt, dim
        self.shape = (*codes.shape[:3], dim)
        c, s = codes.stride(), scales.stride()
        self._desc = QuantPagesDesc(codes.data_ptr(), c[0], c[1], c[2], scales.data_ptr(), s[0], s[1], s[2],
                                    codes.shape[0], codes.shape[1], self.FORMATS[fmt])
        self._at, self._dev = ctypes.addressof(self._desc), codes.get_device()

    @classmethod
    def zeros(cls, n_pages, page_size, n_kv_heads, head_dim, fmt="i8", device=None):
        """An empty cache (it reads as zeros), a head's exponents side by side."""
        import torch
        device = torch.device("cuda", torch.cuda.current_device()) if device is None else device
        width = head_dim if fmt == "i8" else head_dim // 2
        codes = torch.zeros(n_pages, page_size, n_kv_heads, width, dtype=torch.uint8, device=device)
        scales = torch.zeros(n_pages, n_kv_heads, page_size, head_dim // 32, dtype=torch.uint8, device=device)
        return cls(codes, scales.transpose(1, 2), fmt)


def _quant_pages(dev, k_cache, v_cache, heads, dim):
    """Addresses of both descriptors."""
    shape = k_cache.shape
    _same("the caches", shape, v_cache.shape)
    if shape[2] != heads and heads or shape[3] != dim:
        raise BonsaiError(f"caches {shape} do not fit [token][{heads or 'head'}][{dim}]")
    if k_cache.format != v_cache.format:
        raise BonsaiError(f"the caches have formats {k_cache.format} and {v_cache.format}")
    if k_cache._dev != dev or v_cache._dev != dev:
        raise BonsaiError("the caches must be on the current cuda device")
    return k_cache._at, v_cache._at


def paged_append_quant(k, v, k_cache: QuantPages, v_cache: QuantPages, page_table, cu_q, ctx_lens, stream=None) -> None:
    """``paged_append`` into a quantised cache: k, v [T][Hkv][D] f16 or bf16."""
    dev, st, d = _text_place(k)
    dtype, shape = k.dtype, k.shape
    _same("k and v", shape, v.shape)
    T, Hk, D = shape
    kc, vc = _quant_pages(dev, k_cache, v_cache, Hk, D)
    check(lib().bonsai_paged_append_quant(
        _heads(d, 0, k, dtype, dev, D), _heads(d, 1, v, dtype, dev, D), kc, vc,
        *_table_args(dev, page_table, cu_q, ctx_lens), T, Hk, D, _text_dtype(dtype),
        st if stream is None else stream.cuda_stream), "bonsai_paged_append_quant")


def paged_read_quant(k_cache: QuantPages, v_cache: QuantPages, page_table, cu_rows, first, k, v, stream=None) -> None:
    """Cached keys and values as rows k, v [T][Hkv][D] (f16 or bf16): row i of
    sequence s (rows [cu_rows[s], cu_rows[s + 1])) is its place first[s] + i.
    first: cuda int32 [n], or None for the sequences' beginnings."""
    dev, st, d = _text_place(k)
    dtype, shape = k.dtype, k.shape
    _same("k and v", shape, v.shape)
    T, Hk, D = shape
    kc, vc = _quant_pages(dev, k_cache, v_cache, Hk, D)
    n, ts = cu_rows.numel() - 1, page_table.stride()
    if page_table.dim() != 2 or page_table.shape[0] != n or first is not None and first.numel() != n:
        raise BonsaiError(f"page_table {tuple(page_table.shape)}, cu_rows [{n + 1}] and first do not match")
    if page_table.dtype is not _text_torch.int32 or page_table.get_device() != dev or \
            ts[1] != 1 and page_table.shape[1] > 1:
        raise BonsaiError("page_table must be int32 with unit stride along a row on the current device")
    width = page_table.shape[1]
    check(lib().bonsai_paged_read_quant(
        kc, vc, page_table.data_ptr(), ts[0] if n > 1 else width, width, _text_ints(dev, "cu_rows", cu_rows),
        None if first is None else _text_ints(dev, "first", first), n, T, Hk, D, _text_dtype(dtype),
        _heads(d, 0, k, dtype, dev, D), _heads(d, 1, v, dtype, dev, D),
        st if stream is None else stream.cuda_stream), "bonsai_paged_read_quant")


def paged_attention_quant(q, k_cache: QuantPages, v_cache: QuantPages, page_table, cu_q, ctx_lens, max_ctx, out,
                          max_q=None, scale=None, stream=None) -> None:
    """``paged_attention`` over a quantised cache.  max_q: an upper bound of the
    new tokens of a sequence (None: all of q); like max_ctx it only sets how the
    work is done."""
    dev, st, d = _text_place(q)
    dtype, shape = q.dtype, q.shape
    _same("q and out", shape, out.shape)
    T, H, D = shape
    kc, vc = _quant_pages(dev, k_cache, v_cache, 0, D)
    check(lib().bonsai_paged_attention_quant(
        _heads(d, 0, q, dtype, dev, D), kc, vc, *_table_args(dev, page_table, cu_q, ctx_lens), T,
        T if max_q is None else max_q, max_ctx, H, k_cache.shape[2], D, _text_dtype(dtype),
        D ** -0.5 if scale is None else scale, _heads(d, 1, out, dtype, dev, D),
        st if stream is None else stream.cuda_stream), "bonsai_paged_attention_quant")


def sample_tokens(logits, u, tokens, probs=None, temperature=None, top_k=None, top_p=None, min_p=None,
                  stream=None) -> None:
    """The next token of each row of logits [rows][vocab] (f16, bf16 or f32, rows
    that do not overlap): tokens int32 [rows], probs f32 [rows] or None.  u f32 [rows]
    are the random numbers; temperature, top_p, min_p f32 [rows] and top_k int32
    [rows] the rows' settings (None: 1, 1, 0, 0).  The rule, ties and special values
    are at bonsai_sample_tokens in include/bonsai_cuda.h."""
    dev, st, _ = _text_place(logits)
    torch = _text_torch
    shape, s = logits.shape, logits.stride()
    if len(shape) != 2 or s[1] != 1 and shape[1] > 1:
        raise BonsaiError(f"logits must be [rows][vocab] with contiguous rows, got {tuple(shape)} {tuple(s)}")
    n = shape[0]

    def row(name, t, dtype):
        if t is None:
            return None
        if t.dtype is not dtype or t.get_device() != dev or t.dim() != 1 or t.shape[0] != n or not t.is_contiguous():
            raise BonsaiError(f"{name} must be a contiguous {dtype} tensor [{n}] on the current device")
        return t.data_ptr()

    dtype = logits.dtype
    code = 2 if dtype is torch.float32 else 0 if dtype is torch.float16 else 1 if dtype is torch.bfloat16 else None
    if code is None:
        raise BonsaiError(f"sample_tokens takes f16, bf16 or f32 logits, got {dtype}")
    f32 = torch.float32
    check(lib().bonsai_sample_tokens(
        logits.data_ptr(), s[0] if n > 1 else shape[1], n, shape[1], code, row("temperature", temperature, f32),
        row("top_k", top_k, torch.int32), row("top_p", top_p, f32), row("min_p", min_p, f32), row("u", u, f32),
        row("tokens", tokens, torch.int32), row("probs", probs, f32),
        st if stream is None else stream.cuda_stream), "bonsai_sample_tokens")


# ----------------------------------------------------------------- host side
def random_b1_packed(out_dim: int, in_dim: int, rng: np.random.Generator,
                     scale_std: float = 0.02) -> np.ndarray:
    """Seeded random packed B1_0 matrix [out_dim][in_dim/32*6] (uint8): signs
    Bernoulli(0.5), scales |N(0, scale_std)| rounded to f16, in the layout of
    convert_to_b1_0_packed.py:21-43."""
    nb = in_dim // 32
    signs = rng.integers(0, 2, size=(out_dim, nb, 32), dtype=np.uint8)
    scales = np.abs(rng.standard_normal((out_dim, nb)) * scale_std).astype(np.float16)
    raw = np.zeros((out_dim, nb, 6), dtype=np.uint8)
    raw[:, :, 0:2] = scales.view(np.uint8).reshape(out_dim, nb, 2)
    raw[:, :, 2:6] = np.packbits(signs, axis=-1, bitorder="little")
    return raw.reshape(out_dim, nb * 6)


def dequant_b1(packed: np.ndarray, out_dim: int, in_dim: int) -> np.ndarray:
    """f32 [out_dim][in_dim] = +-scale per the B1_0 block rule
    (tests/test_diffuser.py:24-33 dequant of the reference)."""
    nb = in_dim // 32
    raw = np.ascontiguousarray(packed, dtype=np.uint8).reshape(out_dim, nb, 6)
    scales = raw[:, :, 0:2].copy().view(np.float16).reshape(out_dim, nb).astype(np.float32)
    bits = np.unpackbits(raw[:, :, 2:6], axis=-1, bitorder="little").astype(np.float32)
    return ((bits * 2.0 - 1.0) * scales[:, :, None]).reshape(out_dim, in_dim)


# ----------------------------------------------------------------- model
class DitConfig(ctypes.Structure):
    _fields_ = [("preset", ctypes.c_int), ("depth", ctypes.c_int), ("depth_single", ctypes.c_int),
                ("img_tokens", ctypes.c_int), ("txt_tokens", ctypes.c_int),
                ("grid_h", ctypes.c_int), ("grid_w", ctypes.c_int), ("seed", ctypes.c_ulonglong)]


PRESET_DIMS = {
    # preset: (depth, depth_single, mlp, swiglu, in_ch, ctx_dim, pooled, axes, theta, per_block_mod)
    PRESET_KLEIN4B: (5, 20, 9216, True, 128, 7680, 0, (32, 32, 32, 32), 2000.0, False),
    PRESET_FLUX1: (19, 38, 12288, False, 64, 4096, 768, (16, 56, 56), 10000.0, True),
}
HIDDEN, HEADS, HEAD_DIM = 3072, 24, 128


class Dit:
    """One diffuser transformer on the device (bonsai_dit_* entry points)."""

    def __init__(self, preset: int, img_tokens: int, txt_tokens: int, grid_h: int, grid_w: int,
                 depth: int = 0, depth_single: int = 0, seed: int = 1234):
        d = PRESET_DIMS[preset]
        self.preset = preset
        self.depth = depth or d[0]
        self.depth_single = depth_single or d[1]
        self.mlp, self.swiglu, self.in_ch, self.ctx_dim, self.pooled = d[2], d[3], d[4], d[5], d[6]
        self.axes, self.theta, self.per_block_mod = d[7], d[8], d[9]
        self.img, self.txt, self.L = img_tokens, txt_tokens, img_tokens + txt_tokens
        self.grid_h, self.grid_w = grid_h, grid_w
        cfg = DitConfig(preset, depth, depth_single, img_tokens, txt_tokens, grid_h, grid_w, seed)
        h = _vp()
        check(lib().bonsai_dit_create(ctypes.byref(cfg), ctypes.byref(h)), "bonsai_dit_create")
        self.handle = h

    def close(self):
        if getattr(self, "handle", None):
            lib().bonsai_dit_destroy(self.handle)
            self.handle = None

    def __del__(self):
        try:
            self.close()
        except Exception:
            pass

    def weight(self, name: str) -> np.ndarray:
        n = lib().bonsai_dit_weight(self.handle, name.encode(), None, 0)
        if n < 0:
            check(int(n), f"bonsai_dit_weight({name})")
        buf = np.empty(n, np.uint8)
        check(0 if lib().bonsai_dit_weight(self.handle, name.encode(), buf.ctypes.data, n) == n
              else -1, f"bonsai_dit_weight({name})")
        return buf

    def set_weight(self, name: str, data: np.ndarray):
        """Replace a weight from host bytes in the layout weight() returns."""
        buf = np.ascontiguousarray(data)
        check(lib().bonsai_dit_set_weight(self.handle, name.encode(), buf.ctypes.data, buf.nbytes),
              f"bonsai_dit_set_weight({name})")

    def load_safetensors(self, path):
        """Load a checkpoint in the reference's packed safetensors layout (klein4b)."""
        check(lib().bonsai_dit_load_safetensors(self.handle, str(path).encode()),
              "bonsai_dit_load_safetensors")

    def sample(self, latents, txt, pooled, n_steps: int, stream=None) -> np.ndarray:
        """Whole Euler loop on the device (latents updated in place); returns the
        per-step stats [n_steps][5] = NaN count, Inf count, min, max, mean."""
        stats = np.zeros((n_steps, 5), np.float32)
        check(lib().bonsai_dit_sample(self.handle, latents.data_ptr(),
                                      txt.data_ptr() if txt is not None else None,
                                      pooled.data_ptr() if pooled is not None else None,
                                      n_steps, stats.ctypes.data, stream_ptr(stream)),
              "bonsai_dit_sample")
        return stats

    def weight_f32(self, name: str) -> np.ndarray:
        return self.weight(name).view(np.float32)

    def rope_ids(self) -> np.ndarray:
        """Token ids [L][n_axes] (src/diffuser.cpp:240-249): text 0, image (.., y, x)."""
        na = len(self.axes)
        ids = np.zeros((self.L, na), np.float32)
        for y in range(self.grid_h):
            for x in range(self.grid_w):
                ids[self.txt + y * self.grid_w + x, na - 2] = y
                ids[self.txt + y * self.grid_w + x, na - 1] = x
        return ids

    def forward(self, img, txt, pooled, t: float, out, stream=None):
        check(lib().bonsai_dit_forward(self.handle, img.data_ptr(),
                                       txt.data_ptr() if txt is not None else None,
                                       pooled.data_ptr() if pooled is not None else None,
                                       float(t), out.data_ptr(), stream_ptr(stream)),
              "bonsai_dit_forward")

    def forward_host(self, img: np.ndarray, txt: np.ndarray, pooled, t: float,
                     out: np.ndarray, stream=None):
        check(lib().bonsai_dit_forward_host(self.handle, img.ctypes.data,
                                            txt.ctypes.data if txt is not None else None,
                                            pooled.ctypes.data if pooled is not None else None,
                                            float(t), out.ctypes.data, stream_ptr(stream)),
              "bonsai_dit_forward_host")

    def set_state(self, hidden, vec, stream=None):
        check(lib().bonsai_dit_set_state(self.handle, hidden.data_ptr(), vec.data_ptr(),
                                         stream_ptr(stream)), "bonsai_dit_set_state")

    def get_state(self, hidden, stream=None):
        check(lib().bonsai_dit_get_state(self.handle, hidden.data_ptr(), stream_ptr(stream)),
              "bonsai_dit_get_state")

    # ---- partitioned (multi-GPU) driving, see bonsai_b200.headsplit
    def set_partition(self, rank: int, world: int):
        check(lib().bonsai_dit_set_partition(self.handle, rank, world), "bonsai_dit_set_partition")

    def set_peers(self, xm_ptrs, cat_ptrs):
        """Fused exchanges: every rank's xm / cat device pointers as seen
        from this GPU ([rank] = this model's own); None switches back."""
        if xm_ptrs is None:
            check(lib().bonsai_dit_set_peers(self.handle, None, None, 0), "bonsai_dit_set_peers")
            return
        n = len(xm_ptrs)
        xa = (_vp * n)(*xm_ptrs)
        ca = (_vp * n)(*cat_ptrs)
        check(lib().bonsai_dit_set_peers(self.handle, xa, ca, n), "bonsai_dit_set_peers")

    def set_qkv_peers(self, qkv_ptrs):
        """QKV scatter: every rank's qkv device pointer as seen from this GPU
        ([rank] = this model's own); None switches back to the xm broadcast."""
        if qkv_ptrs is None:
            check(lib().bonsai_dit_set_qkv_peers(self.handle, None, 0), "bonsai_dit_set_qkv_peers")
            return
        n = len(qkv_ptrs)
        check(lib().bonsai_dit_set_qkv_peers(self.handle, (_vp * n)(*qkv_ptrs), n),
              "bonsai_dit_set_qkv_peers")

    def ipc_handle(self, name: str) -> bytes:
        buf = ctypes.create_string_buffer(64)
        check(lib().bonsai_dit_ipc_handle(self.handle, name.encode(), buf), "bonsai_dit_ipc_handle")
        return buf.raw

    def open_qkv_peers(self, handles: bytes, world: int):
        assert len(handles) == 64 * world
        check(lib().bonsai_dit_open_qkv_peers(self.handle, handles, world),
              "bonsai_dit_open_qkv_peers")

    def open_flag_peers(self, handles: bytes, world: int):
        """Every rank's "flags" IPC handle (world x 64 bytes): enables
        barrier(); order the ranks once (host barrier) before the first."""
        assert len(handles) == 64 * world
        check(lib().bonsai_dit_open_flag_peers(self.handle, handles, world),
              "bonsai_dit_open_flag_peers")

    def barrier(self, stream=None):
        """Stream-ordered barrier of the partitioned ranks over peer flags."""
        check(lib().bonsai_dit_barrier(self.handle, stream_ptr(stream)), "bonsai_dit_barrier")

    def ipc_handles(self) -> bytes:
        buf = ctypes.create_string_buffer(128)
        check(lib().bonsai_dit_ipc_handles(self.handle, buf), "bonsai_dit_ipc_handles")
        return buf.raw

    def open_peers(self, handles: bytes, world: int):
        assert len(handles) == 128 * world
        check(lib().bonsai_dit_open_peers(self.handle, handles, world), "bonsai_dit_open_peers")

    def buffer(self, name: str, dtype, shape):
        """Engine buffer as a torch tensor view (no copy)."""
        import torch
        ptr, nbytes = _vp(), _c_ll()
        check(lib().bonsai_dit_buffer(self.handle, name.encode(), ctypes.byref(ptr),
                                      ctypes.byref(nbytes)), f"bonsai_dit_buffer({name})")
        return _wrap_device(ptr.value, nbytes.value, dtype, shape)

    def begin(self, img, txt, pooled, t: float, stream=None):
        check(lib().bonsai_dit_begin(self.handle, img.data_ptr(),
                                     txt.data_ptr() if txt is not None else None,
                                     pooled.data_ptr() if pooled is not None else None,
                                     float(t), stream_ptr(stream)), "bonsai_dit_begin")

    def phase(self, kind: int, block: int, phase: int, stream=None):
        check(lib().bonsai_dit_phase(self.handle, kind, block, phase, stream_ptr(stream)),
              "bonsai_dit_phase")

    def end(self, out, stream=None):
        check(lib().bonsai_dit_end(self.handle, out.data_ptr(), stream_ptr(stream)), "bonsai_dit_end")

    def double_block(self, i: int, stream=None):
        check(lib().bonsai_dit_double_block(self.handle, i, stream_ptr(stream)), "double_block")

    def single_block(self, i: int, stream=None):
        check(lib().bonsai_dit_single_block(self.handle, i, stream_ptr(stream)), "single_block")


class Vae:
    """The Flux VAE decoder on the device (bonsai_vae_* entry points), the
    reference's bonsai_vae program (src/vae_decoder.cpp) for one encoded
    latent size: latent f32 [128][h][w] -> raw image f32 [3][16h][16w]."""

    def __init__(self, latent_h: int, latent_w: int, seed: int = 0):
        h = _vp()
        check(lib().bonsai_vae_create(latent_h, latent_w, seed, ctypes.byref(h)), "bonsai_vae_create")
        self.handle = h
        self.latent_h, self.latent_w = latent_h, latent_w
        self.image_h, self.image_w = 16 * latent_h, 16 * latent_w

    def close(self):
        if getattr(self, "handle", None):
            lib().bonsai_vae_destroy(self.handle)
            self.handle = None

    def __del__(self):
        try:
            self.close()
        except Exception:
            pass

    def load_safetensors(self, path) -> None:
        check(lib().bonsai_vae_load_safetensors(self.handle, str(path).encode()),
              "bonsai_vae_load_safetensors")

    def decode(self, latent, image, stream=None) -> None:
        """latent: cuda f32 [128][h][w]; image: cuda f32 [3][16h][16w]."""
        assert latent.is_contiguous() and image.is_contiguous()
        assert latent.numel() == 128 * self.latent_h * self.latent_w
        assert image.numel() == 3 * self.image_h * self.image_w
        check(lib().bonsai_vae_decode(self.handle, latent.data_ptr(), image.data_ptr(),
                                      stream_ptr(stream)), "bonsai_vae_decode")

    def decode_host(self, latent: np.ndarray, stream=None) -> np.ndarray:
        lat = np.ascontiguousarray(latent, dtype=np.float32)
        assert lat.size == 128 * self.latent_h * self.latent_w
        out = np.empty((3, self.image_h, self.image_w), np.float32)
        check(lib().bonsai_vae_decode_host(self.handle, lat.ctypes.data, out.ctypes.data,
                                           stream_ptr(stream)), "bonsai_vae_decode_host")
        return out


def conv2d_nhwc(x, w, bias, out, resid=None, stream=None) -> None:
    """x: cuda f16/bf16 NHWC [H][W][cin]; w: cuda f32 [cout][cin][k][k];
    bias: cuda f32 [cout] or None; out (and resid): cuda f32 NHWC [H][W][cout]."""
    import torch
    hh, ww, cin = x.shape
    cout, _, k, _ = w.shape
    assert x.is_contiguous() and w.is_contiguous() and out.is_contiguous()
    check(lib().bonsai_conv2d_nhwc(x.data_ptr(), hh, ww, cin, int(x.dtype == torch.bfloat16),
                                   w.data_ptr(), cout, k, bias.data_ptr() if bias is not None else None,
                                   resid.data_ptr() if resid is not None else None, out.data_ptr(),
                                   stream_ptr(stream)), "bonsai_conv2d_nhwc")


def vae_rgb8(image, rgb, stream=None) -> None:
    """image: cuda f32 [3][H][W]; rgb: cuda u8 [H][W][3] (sigmoid, x255, clamp)."""
    _, hh, ww = image.shape
    check(lib().bonsai_vae_rgb8(image.data_ptr(), hh, ww, rgb.data_ptr(), stream_ptr(stream)),
          "bonsai_vae_rgb8")


def _wrap_device(ptr: int, nbytes: int, dtype, shape):
    """A torch tensor aliasing device memory owned by the engine (no copy)."""
    import torch

    class _Holder:
        def __init__(self, p, n):
            self.__cuda_array_interface__ = {
                "shape": (n,), "typestr": "|u1", "data": (p, False), "version": 3}

    flat = torch.as_tensor(_Holder(ptr, nbytes), device="cuda")
    return flat.view(dtype).view(shape)
