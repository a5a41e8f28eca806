"""Python operator API over libasmllm.so.

Two layers, both going through the C ABI (no Python or torch compute path):

* Host layer -- numpy in, numpy out, through the reference's synchronous
  entry points (`asm_matmul_q4`, `asm_matmul_q8`, ...), exactly as the
  reference's ctypes callers use them (THRISHAL12345/asmllm
  tests/correctness/test_runner.py:84-111, src/runtime/generate.py:255-259).
* Device layer -- torch CUDA tensors, stream-ordered on torch's current
  stream through the `*_async` entries; this is what the decode driver and
  the benchmark use with weights resident in HBM.

Argument meanings follow the reference: qweights Q4_0 uint8 [M, K/32, 16]
(or flat), Q8_0 int8 [M, K/32, 32], scales [M, K/32], x fp32 [K], y fp32 [M].
"""
from __future__ import annotations

import ctypes
import struct

import numpy as np

from . import native
from .native import FMT_Q4_0, FMT_Q8_0, AsmError

MV_INDEPENDENT = 1  # ASM_MV_INDEPENDENT (include/asmllm.h)
MV_PACKED = 2  # ASM_MV_PACKED

# --------------------------------------------------------------------------
# Host (numpy) layer: the reference-facing synchronous ABI
# --------------------------------------------------------------------------


def _np(a, dtype):
    return np.ascontiguousarray(a, dtype=dtype)


def _mk(qw, scales, x, wdtype, bytes_per_block):
    qw = _np(qw, wdtype)
    scales = _np(scales, np.float32)
    x = _np(x, np.float32)
    K = x.shape[-1]
    M = scales.shape[0] if scales.ndim >= 2 else (qw.size // max(1, (K // 32) * bytes_per_block) if K else 0)
    return qw, scales, x, int(M), int(K)


def _sync_call(name, qw, scales, x, wdtype, bpb, *extra):
    qw, scales, x, M, K = _mk(qw, scales, x, wdtype, bpb)
    y = np.zeros(M, dtype=np.float32)
    getattr(native.lib(), name)(qw.ctypes.data, scales.ctypes.data, x.ctypes.data,
                                y.ctypes.data, M, K, *extra)
    native.check()
    return y


def matmul_q4(qweights, scales, x):
    """asm_matmul_q4: Q4_0 x Q8_0 (x quantized inside, NEON semantics)."""
    return _sync_call("asm_matmul_q4", qweights, scales, x, np.uint8, 16)


def matmul_q4_mt(qweights, scales, x, num_threads=4):
    return _sync_call("asm_matmul_q4_mt", qweights, scales, x, np.uint8, 16, int(num_threads))


def matmul_q4_avx512(qweights, scales, x):
    """asm_matmul_q4_avx512: Q4_0 x fp32 (x86 semantics)."""
    return _sync_call("asm_matmul_q4_avx512", qweights, scales, x, np.uint8, 16)


def matmul_q4_f32(qweights, scales, x):
    return _sync_call("asm_matmul_q4_f32", qweights, scales, x, np.uint8, 16)


def matmul_q8(qweights, scales, x):
    """asm_matmul_q8: Q8_0 x fp32 (x86 / NEON-scalar semantics)."""
    return _sync_call("asm_matmul_q8", qweights, scales, x, np.int8, 32)


def matmul_q8_mt(qweights, scales, x, num_threads=4):
    return _sync_call("asm_matmul_q8_mt", qweights, scales, x, np.int8, 32, int(num_threads))


def matmul_q8q8(qweights, scales, x):
    """asm_matmul_q8q8: Q8_0 x Q8_0."""
    return _sync_call("asm_matmul_q8q8", qweights, scales, x, np.int8, 32)


def quantize_q8_0(x):
    """asm_quantize_q8_0: fp32[K] -> (int8[K], fp32[K/32])."""
    x = _np(x, np.float32)
    K = x.shape[-1]
    xq = np.zeros(K, dtype=np.int8)
    xd = np.zeros(K // 32, dtype=np.float32)
    native.lib().asm_quantize_q8_0(x.ctypes.data, xq.ctypes.data, xd.ctypes.data, K)
    native.check()
    return xq, xd


def register_weights(qweights: np.ndarray, scales: np.ndarray, fmt: int) -> None:
    """asm_weights_register on host arrays (kept alive by the caller)."""
    scales = np.asarray(scales)
    if not (qweights.flags.c_contiguous and scales.flags.c_contiguous and scales.dtype == np.float32):
        raise ValueError("register_weights needs C-contiguous arrays and fp32 scales")
    M = scales.shape[0]
    K = scales.size // M * 32
    rc = native.lib().asm_weights_register(qweights.ctypes.data, scales.ctypes.data, M, K, fmt)
    native.check(rc)


def unregister_weights(qweights: np.ndarray) -> None:
    native.check(native.lib().asm_weights_unregister(qweights.ctypes.data))


def threadpool_init(num_threads: int) -> None:
    native.lib().asm_threadpool_init(int(num_threads))
    native.check()


def threadpool_shutdown() -> None:
    native.lib().asm_threadpool_shutdown()


def threadpool_get_num_threads() -> int:
    return int(native.lib().asm_threadpool_get_num_threads())


def max_k(fmt: int, fp32_activations: bool) -> int:
    return int(native.lib().asm_max_k(fmt, 1 if fp32_activations else 0))


# --------------------------------------------------------------------------
# Device (torch) layer
# --------------------------------------------------------------------------


def _torch():
    import torch  # imported lazily: the host layer needs no torch

    return torch


def _stream_handle(stream=None):
    torch = _torch()
    s = stream if stream is not None else torch.cuda.current_stream()
    return ctypes.c_void_p(s.cuda_stream)


def _ptr(t):
    return ctypes.c_void_p(t.data_ptr())


def _check_dev(t, dtypes, name):
    torch = _torch()
    if not isinstance(t, torch.Tensor) or not t.is_cuda:
        raise TypeError(f"{name}: expected a CUDA tensor")
    if t.dtype not in dtypes:
        raise TypeError(f"{name}: dtype {t.dtype} not in {dtypes}")
    if not t.is_contiguous():
        raise ValueError(f"{name}: tensor must be contiguous")


def matvec(fmt: int, qweights, scales, x, out=None, *, fp32_activations=False, stream=None, independent=False):
    """y = W x on device tensors.

    fmt: FMT_Q4_0 (qweights uint8 [M, K/32, 16]) or FMT_Q8_0 (int8 [M, K/32, 32]).
    scales: fp32 or fp16 [M, K/32].  fp32_activations selects the x86 (fp32-x)
    semantics instead of Q8_0-quantized activations (fp32 scales only).
    independent: the kernel enqueued just before this call neither writes x
    nor touches `out` (asm_matvec_ex_async with ASM_MV_INDEPENDENT), so the
    matvec may overlap it.
    """
    torch = _torch()
    wdt = torch.uint8 if fmt == FMT_Q4_0 else torch.int8
    _check_dev(qweights, (wdt,), "qweights")
    _check_dev(scales, (torch.float32, torch.float16), "scales")
    _check_dev(x, (torch.float32,), "x")
    M = scales.shape[0]
    K = x.shape[-1]
    if scales.numel() != M * (K // 32) or qweights.numel() != M * (K // 32) * (16 if fmt == FMT_Q4_0 else 32):
        raise ValueError(f"shape mismatch: qweights {tuple(qweights.shape)}, scales {tuple(scales.shape)}, K={K}")
    if out is None:
        out = torch.empty(M, dtype=torch.float32, device=x.device)
    else:
        _check_dev(out, (torch.float32,), "out")
    L = native.lib()
    f16 = scales.dtype == torch.float16
    st = _stream_handle(stream)
    args = (_ptr(qweights), _ptr(scales), _ptr(x), _ptr(out), M, K, st)
    if fp32_activations:
        if f16:
            raise ValueError("fp32-activation kernels take fp32 scales")
        rc = (L.asm_matmul_q4_f32_async if fmt == FMT_Q4_0 else L.asm_matmul_q8_async)(*args)
    elif independent:
        rc = L.asm_matvec_ex_async(fmt, _ptr(qweights), _ptr(scales), 1 if f16 else 0, _ptr(x), _ptr(out), M, K,
                                   MV_INDEPENDENT, st)
    elif fmt == FMT_Q4_0:
        rc = (L.asm_matmul_q4_f16s_async if f16 else L.asm_matmul_q4_async)(*args)
    else:
        rc = (L.asm_matmul_q8q8_f16s_async if f16 else L.asm_matmul_q8q8_async)(*args)
    native.check(rc)
    return out


def packed_row_bytes(fmt: int, K: int) -> int:
    """Bytes of one packed row (asm_packed_row_bytes); K a multiple of 256."""
    n = int(native.lib().asm_packed_row_bytes(fmt, int(K)))
    if n < 0:
        raise ValueError(f"no packed layout for fmt={fmt}, K={K} (K must be a multiple of 256)")
    return n


def pack_rows(fmt: int, qweights, scales_f16, out=None, stream=None):
    """Device qweights + fp16 scales -> packed rows uint8 [M, packed_row_bytes] (asm_pack_rows_async)."""
    torch = _torch()
    _check_dev(scales_f16, (torch.float16,), "scales")
    M, K = scales_f16.shape[0], scales_f16.shape[1] * 32
    if out is None:
        out = torch.empty((M, packed_row_bytes(fmt, K)), dtype=torch.uint8, device=qweights.device)
    native.check(native.lib().asm_pack_rows_async(fmt, _ptr(qweights), _ptr(scales_f16), _ptr(out), M, K,
                                                  _stream_handle(stream)))
    return out


def matvec_packed(fmt: int, packed, x, out=None, *, stream=None, independent=False):
    """y = W x on packed rows (asm_matvec_packed_async): Q4_0 / Q8_0 x Q8_0."""
    torch = _torch()
    _check_dev(packed, (torch.uint8,), "packed")
    _check_dev(x, (torch.float32,), "x")
    M, K = packed.shape[0], x.shape[-1]
    if packed.numel() != M * packed_row_bytes(fmt, K):
        raise ValueError(f"packed {tuple(packed.shape)} does not hold {M} rows of K={K}")
    if out is None:
        out = torch.empty(M, dtype=torch.float32, device=x.device)
    else:
        _check_dev(out, (torch.float32,), "out")
    native.check(native.lib().asm_matvec_packed_async(fmt, _ptr(packed), _ptr(x), _ptr(out), M, K,
                                                      MV_INDEPENDENT if independent else 0, _stream_handle(stream)))
    return out


def mark_static(*tensors) -> None:
    """Declares device tensors (model weights) static: see asm_weights_mark_static."""
    L = native.lib()
    for t in tensors:
        native.check(L.asm_weights_mark_static(_ptr(t), t.numel() * t.element_size()))


def unmark_static(*tensors) -> None:
    L = native.lib()
    for t in tensors:
        native.check(L.asm_weights_unmark_static(_ptr(t)))


def set_option(name: str, value: int) -> int:
    """asm_set_option: "tma" / "pdl" kernel-path switches, "image_min_k" (matvecs with
    K >= it quantize x in a pre-pass; 0 = never), "gemm_splits" (0 = automatic K split
    of the batched product, S = exactly S), "sync_map" (synchronous entries: bit 0 reads
    pinned host x in place, bit 1 writes pinned host y in place; default 3); returns the
    previous value."""
    prev = int(native.lib().asm_set_option(name.encode(), int(value)))
    if prev < 0:
        native.check()
    return prev


def device_error() -> int:
    """Reads and clears the device error word (0 = no kernel gave up a bounded wait)."""
    v = ctypes.c_uint(0)
    native.check(native.lib().asm_device_error(ctypes.byref(v)))
    return int(v.value)


def act_image_bytes(K: int) -> int:
    """Bytes of one row of the Q8_0 activation image (asm_act_image_bytes)."""
    n = int(native.lib().asm_act_image_bytes(int(K)))
    if n < 0:
        raise ValueError(f"K={K} is not a multiple of 32")
    return n


def act_image_dev(x, out=None, stream=None, prefetch=None):
    """Quantizes x fp32 [K] or [N, K] once into the activation image (uint8 [N, bytes]).

    prefetch: optional (qweights, scales) of the matvec that will read the
    image; their first bytes are streamed into L2 while the quantize waits for
    the previous kernel (a performance hint; results are unchanged)."""
    torch = _torch()
    _check_dev(x, (torch.float32,), "x")
    K = x.shape[-1]
    N = x.numel() // K if K else 0
    nbytes = act_image_bytes(K)
    if out is None:
        out = torch.empty((max(N, 1), nbytes), dtype=torch.uint8, device=x.device)
    L = native.lib()
    if prefetch is None:
        rc = L.asm_act_image_q8_0_async(_ptr(x), _ptr(out), N, K, _stream_handle(stream))
    else:
        w, s = prefetch
        rc = L.asm_act_image_q8_0_prefetch_async(_ptr(x), _ptr(out), N, K, _ptr(w), w.numel() * w.element_size(),
                                                 _ptr(s), s.numel() * s.element_size(), _stream_handle(stream))
    native.check(rc)
    return out


def matvec_image(fmt: int, qweights, scales, image, K: int, out=None, stream=None):
    """y = W x with x given as a prepared activation image (see act_image_dev)."""
    torch = _torch()
    wdt = torch.uint8 if fmt == FMT_Q4_0 else torch.int8
    _check_dev(qweights, (wdt,), "qweights")
    _check_dev(scales, (torch.float32, torch.float16), "scales")
    _check_dev(image, (torch.uint8,), "image")
    M = scales.shape[0]
    if image.numel() < act_image_bytes(K):
        raise ValueError("image too small for K")
    if out is None:
        out = torch.empty(M, dtype=torch.float32, device=image.device)
    rc = native.lib().asm_matmul_image_async(fmt, _ptr(qweights), _ptr(scales), 1 if scales.dtype == torch.float16 else 0,
                                             _ptr(image), _ptr(out), M, K, _stream_handle(stream))
    native.check(rc)
    return out


def quantize_q8_0_dev(x, xq=None, xd=None, stream=None):
    """Device quantize of x fp32 [N, K] or [K] -> (int8 same shape, fp32 [..., K/32])."""
    torch = _torch()
    _check_dev(x, (torch.float32,), "x")
    K = x.shape[-1]
    N = x.numel() // K if K else 0
    if xq is None:
        xq = torch.empty(x.shape, dtype=torch.int8, device=x.device)
    if xd is None:
        xd = torch.empty((*x.shape[:-1], K // 32), dtype=torch.float32, device=x.device)
    rc = native.lib().asm_quantize_q8_0_async(_ptr(x), _ptr(xq), _ptr(xd), N, K, _stream_handle(stream))
    native.check(rc)
    return xq, xd


def block_sums_dev(fmt: int, qweights, scales, x, stream=None):
    """(y, isums int32 [M, K/32]) from the matvec kernel's own debug instantiation."""
    torch = _torch()
    M = scales.shape[0]
    K = x.shape[-1]
    y = torch.empty(M, dtype=torch.float32, device=x.device)
    isums = torch.empty((M, K // 32), dtype=torch.int32, device=x.device)
    rc = native.lib().asm_block_sums_async(fmt, _ptr(qweights), _ptr(scales), _ptr(x), _ptr(y),
                                           _ptr(isums), M, K, _stream_handle(stream))
    native.check(rc)
    return y, isums


def gguf_split_dev(fmt: int, raw, nblocks: int, scales_f16: bool = True, stream=None):
    """Split raw GGUF Q4_0 (18 B) / Q8_0 (34 B) blocks on the device.

    Returns (qs uint8/int8 [nblocks, 16|32], scales fp16|fp32 [nblocks]).
    Mirrors the reference's host split in src/runtime/generate.py:91-119.
    """
    torch = _torch()
    _check_dev(raw, (torch.uint8,), "raw")
    qb = 16 if fmt == FMT_Q4_0 else 32
    if raw.numel() < nblocks * (qb + 2):
        raise ValueError("raw buffer shorter than nblocks blocks")
    qs = torch.empty((nblocks, qb), dtype=torch.uint8 if fmt == FMT_Q4_0 else torch.int8, device=raw.device)
    scales = torch.empty(nblocks, dtype=torch.float16 if scales_f16 else torch.float32, device=raw.device)
    rc = native.lib().asm_gguf_split_async(fmt, _ptr(raw), _ptr(qs), _ptr(scales), 1 if scales_f16 else 0,
                                           nblocks, _stream_handle(stream))
    native.check(rc)
    return qs, scales


__all__ = [
    "AsmError", "FMT_Q4_0", "FMT_Q8_0",
    "matmul_q4", "matmul_q4_mt", "matmul_q4_avx512", "matmul_q4_f32", "matmul_q8", "matmul_q8_mt",
    "matmul_q8q8", "quantize_q8_0", "register_weights", "unregister_weights", "threadpool_init",
    "threadpool_shutdown", "threadpool_get_num_threads", "max_k", "matvec", "quantize_q8_0_dev",
    "block_sums_dev", "gguf_split_dev", "act_image_bytes", "act_image_dev", "matvec_image",
    "mark_static", "unmark_static", "device_error", "set_option",
    "rope_append", "attention_prompt", "attention_paged", "attention_paged_workspace", "rows_sample",
    "rope_append_q8", "cache_read_q8", "attention_paged_q8", "attention_paged_q8_workspace", "attention_shared",
    "attention_shared_workspace", "rows_adjust",
]


def fused_matvec(fmt: int, qweights, scales, epilogue: int, *, y, x=None, image=None, norm_w=None,
                 eps: float = 1e-5, embed=None, x_copy=None, h=None, image_out=None, counters=None,
                 best=None, done=None, tokens=None, pos=None, vocab: int = 0, max_tokens: int = 0,
                 n_prompt: int = 0, stream=None):
    """One decode-step matvec with its prologue / epilogue fusion (asm_fused_matvec_async).

    epilogue: native.EPI_STORE, EPI_RESIDUAL (y += W x), EPI_SWIGLU (rows
    interleaved gate/up -> h and its Q8_0 image) or EPI_ARGMAX (y = logits,
    tokens[*pos + 1] = argmax, *pos += 1).  Scales must be fp16."""
    torch = _torch()
    _check_dev(scales, (torch.float16,), "scales")
    M, K = scales.shape[0], scales.shape[1] * 32
    d = native.FusedMatvec()
    d.fmt, d.epilogue, d.M, d.K, d.eps = fmt, epilogue, M, K, eps
    d.vocab, d.max_tokens, d.n_prompt = vocab, max_tokens, n_prompt
    for name, t in (("qweights", qweights), ("scales", scales), ("x", x), ("image", image), ("norm_w", norm_w),
                    ("embed", embed), ("x_copy", x_copy), ("y", y), ("h", h), ("image_out", image_out),
                    ("counters", counters), ("best", best), ("done", done), ("tokens", tokens), ("pos", pos)):
        if t is not None:
            setattr(d, name, t.data_ptr())
    native.check(native.lib().asm_fused_matvec_async(ctypes.byref(d), _stream_handle(stream)))
    return y


def attention_decode(qkv, k_cache, v_cache, rope_cs, pos, image_out, n_heads: int, n_kv_heads: int,
                     ctx: int, sqrt_head_dim: float, stream=None):
    """RoPE + fp16 KV append + attention at position *pos (asm_attention_decode_async)."""
    L = native.lib()
    rc = L.asm_attention_decode_async(_ptr(qkv), _ptr(k_cache), _ptr(v_cache), _ptr(rope_cs), _ptr(pos),
                                      _ptr(image_out), n_heads, n_kv_heads, 128, ctx, sqrt_head_dim,
                                      _stream_handle(stream))
    native.check(rc)
    return image_out


def gemm_image(fmt: int, qweights, scales, images, K: int, out=None, stream=None):
    """Y [N, M] = the matvec of every activation-image row (uint8 [N, bytes]), on the
    tensor cores (asm_gemm_image_async).  Scales fp16 [M, K/32]."""
    torch = _torch()
    wdt = torch.uint8 if fmt == FMT_Q4_0 else torch.int8
    _check_dev(qweights, (wdt,), "qweights")
    _check_dev(scales, (torch.float16,), "scales")
    _check_dev(images, (torch.uint8,), "images")
    M = scales.shape[0]
    N = images.shape[0]
    if out is None:
        out = torch.empty((N, M), dtype=torch.float32, device=images.device)
    rc = native.lib().asm_gemm_image_async(fmt, _ptr(qweights), _ptr(scales), _ptr(images), images.stride(0),
                                           _ptr(out), M, N, K, _stream_handle(stream))
    native.check(rc)
    return out


def gemm_narrow(fmt: int, qweights, scales, images, K: int, out=None, stream=None):
    """Y [N, M] for N <= 8 activation-image rows (uint8 [N, bytes]) on the CUDA cores,
    every weight byte read once for all N rows (asm_gemm_narrow_async); row n equals
    the warp-ring matvec of row n bit for bit.  Scales fp16 [M, K/32]."""
    torch = _torch()
    wdt = torch.uint8 if fmt == FMT_Q4_0 else torch.int8
    _check_dev(qweights, (wdt,), "qweights")
    _check_dev(scales, (torch.float16,), "scales")
    _check_dev(images, (torch.uint8,), "images")
    M = scales.shape[0]
    N = images.shape[0]
    if out is None:
        out = torch.empty((N, M), dtype=torch.float32, device=images.device)
    rc = native.lib().asm_gemm_narrow_async(fmt, _ptr(qweights), _ptr(scales), _ptr(images), images.stride(0),
                                            _ptr(out), M, N, K, _stream_handle(stream))
    native.check(rc)
    return out


def gemm(fmt: int, qweights, scales, X, out=None, stream=None, tiles=None):
    """Y [N, M] = W x_n for the N rows of X fp32 [N, K]: quantize every row to Q8_0
    into activation tiles (asm_rows_norm_tiles_async without a norm), then the
    tensor-core product (asm_gemm_tiles_async)."""
    torch = _torch()
    N, K = X.shape
    if tiles is None:
        tiles = torch.empty(act_tiles_bytes(N, K), dtype=torch.uint8, device=X.device)
    rows_norm_tiles(X, tiles, stream=stream)
    return gemm_tiles(fmt, qweights, scales, tiles, N, out=out, stream=stream)


def act_tiles_bytes(N: int, K: int) -> int:
    """Bytes of the activation tiles of N rows of K values (asm_act_tiles_bytes)."""
    n = int(native.lib().asm_act_tiles_bytes(N, K))
    if n <= 0:
        raise ValueError(f"no activation tiles for N={N}, K={K}")
    return n


def act_tiles_from_image(images, K: int, out=None, stream=None):
    """Activation tiles (uint8) of the N activation-image rows (asm_act_tiles_from_image_async)."""
    torch = _torch()
    _check_dev(images, (torch.uint8,), "images")
    N = images.shape[0]
    if out is None:
        out = torch.empty(act_tiles_bytes(N, K), dtype=torch.uint8, device=images.device)
    native.check(native.lib().asm_act_tiles_from_image_async(_ptr(images), images.stride(0), N, K, _ptr(out),
                                                             _stream_handle(stream)))
    return out


def gemm_tiles(fmt: int, qweights, scales, tiles, N: int, out=None, stream=None):
    """Y [N, M] from N rows of activation tiles on the tensor cores (asm_gemm_tiles_async)."""
    torch = _torch()
    wdt = torch.uint8 if fmt == FMT_Q4_0 else torch.int8
    _check_dev(qweights, (wdt,), "qweights")
    _check_dev(scales, (torch.float16,), "scales")
    _check_dev(tiles, (torch.uint8,), "tiles")
    M, K = scales.shape[0], scales.shape[1] * 32
    if tiles.numel() < act_tiles_bytes(N, K):
        raise ValueError("tiles buffer too small")
    if out is None:
        out = torch.empty((N, M), dtype=torch.float32, device=tiles.device)
    native.check(native.lib().asm_gemm_tiles_async(fmt, _ptr(qweights), _ptr(scales), _ptr(tiles), _ptr(out), M, N,
                                                   K, _stream_handle(stream)))
    return out


def rows_norm_tiles(x, tiles, norm_w=None, eps: float = 1e-5, delta=None, embed=None, tokens=None, pos=None,
                    stream=None):
    """asm_rows_norm_tiles_async on x fp32 [B, dim] (updated in place when embed or delta is given)."""
    d = native.Rows()
    d.rows, d.dim = x.shape[0], x.shape[1]
    d.eps = eps
    for name, t in (("x", x), ("delta", delta), ("embed", embed), ("tokens", tokens), ("pos", pos),
                    ("norm_w", norm_w), ("tiles", tiles)):
        if t is not None:
            setattr(d, name, t.data_ptr())
    if embed is not None:
        d.vocab, d.max_tokens = embed.shape[0], tokens.shape[1]
    native.check(native.lib().asm_rows_norm_tiles_async(ctypes.byref(d), _stream_handle(stream)))
    return tiles


def rows_swiglu_tiles(gu, tiles, stream=None):
    """asm_rows_swiglu_tiles_async: gu fp32 [B, 2*ffn] (gate/up pairs) -> tiles of h [B, ffn]."""
    native.check(native.lib().asm_rows_swiglu_tiles_async(_ptr(gu), gu.shape[0], gu.shape[1] // 2, _ptr(tiles),
                                                          _stream_handle(stream)))
    return tiles


def attention_batch(qkv, k_cache, v_cache, rope_cs, pos, tiles, n_heads: int, n_kv_heads: int, ctx: int,
                    sqrt_head_dim: float, stream=None):
    """asm_attention_batch_async: qkv fp32 [B, (nh + 2 nkv) * 128], caches fp16 [B, ctx, nkv, 128]."""
    rows = qkv.shape[0]
    native.check(native.lib().asm_attention_batch_async(
        _ptr(qkv), qkv.stride(0), _ptr(k_cache), _ptr(v_cache), k_cache.stride(0), _ptr(rope_cs), _ptr(pos),
        _ptr(tiles), rows, n_heads, n_kv_heads, 128, ctx, sqrt_head_dim, _stream_handle(stream)))
    return tiles


def rows_argmax(logits, keys, offset: int = 0, stream=None):
    """asm_rows_argmax_async: keys int64 [B] = signed-orderable (value, offset + index) maxima."""
    native.check(native.lib().asm_rows_argmax_async(_ptr(logits), logits.shape[0], logits.shape[1],
                                                    logits.stride(0), offset, _ptr(keys), _stream_handle(stream)))
    return keys


def rows_advance(keys, tokens, pos, n_prompt: int, stream=None):
    """asm_rows_advance_async: tokens[r][pos + 1] = argmax index of keys[r] after the prompt; pos += 1."""
    native.check(native.lib().asm_rows_advance_async(_ptr(keys), keys.shape[0], _ptr(tokens), tokens.shape[1],
                                                     _ptr(pos), n_prompt, _stream_handle(stream)))


def key_index(keys):
    """Index part of signed-orderable argmax keys (host or device int64 tensor)."""
    return ((keys ^ (-(1 << 63))) & 0xFFFFFFFF).neg().add(0xFFFFFFFF)


# --------------------------------------------------------------------------
# Serving operators: prompts of different lengths, a paged cache, sampling
#
# A decode step makes hundreds of these calls and the kernels take a few
# microseconds, so the checks are written for the case that passes: one
# expression over what the tensors say, and the long way (which names the
# fault) only where it fails.
# --------------------------------------------------------------------------

_DT: dict = {}   # torch dtype -> ASM_DT_*
_H16: dict = {}  # the 16-bit ones alone
_KV_PACK = struct.Struct("QQqqqQqQQiiiiiiii").pack  # asm_kv_t (native.Kv), field for field
_KV_Q8_PACK = struct.Struct("QQQQqqqqqQqQiiiiii").pack  # asm_kv_q8_t (native.KvQ8)
_ADJUST_PACK = struct.Struct("QQqqiiiiQqQQQQQQQQqii").pack  # asm_adjust_t (native.Adjust)
_F32 = _F16 = _I32 = _I8 = _U8 = _current_stream = None  # torch's, once it is imported


def _dtypes():
    global _F32, _F16, _I32, _I8, _U8, _current_stream
    torch = _torch()
    _F32, _F16, _I32, _I8, _U8 = torch.float32, torch.float16, torch.int32, torch.int8, torch.uint8
    _current_stream = torch._C._cuda_getCurrentRawStream
    _H16.update({torch.float16: native.DT_F16, torch.bfloat16: native.DT_BF16})
    _DT.update({torch.float32: native.DT_F32, **_H16})
    return _DT


def _empty(like, shape, dtype, stream):
    """A new output beside `like` that belongs to the stream the kernel runs on."""
    if stream is None:
        return like.new_empty(shape, dtype=dtype)
    with _torch().cuda.stream(stream):
        return like.new_empty(shape, dtype=dtype)


def _call(rc: int) -> None:
    if rc:
        native.check(rc)


def _dense(t, name, ndim, dtypes):
    """A CUDA tensor of `ndim` axes whose last one is dense (the others may be strided)."""
    torch = _torch()
    if not isinstance(t, torch.Tensor) or not t.is_cuda:
        raise TypeError(f"{name}: expected a CUDA tensor")
    if t.dtype not in dtypes:
        raise TypeError(f"{name}: dtype {t.dtype} not in {tuple(dtypes)}")
    if t.dim() != ndim or (t.shape[-1] > 1 and t.stride(-1) != 1):
        raise ValueError(f"{name}: expected {ndim} axes, the last one dense; got {tuple(t.shape)} "
                         f"with strides {t.stride()}")


def _strides(t):
    """Strides, those of axes with a single entry replaced by the dense ones (they mean nothing)."""
    st = t.stride()
    if 1 in t.shape:
        st, dense = list(st), 1
        for i in range(len(st) - 1, -1, -1):
            if t.shape[i] == 1:
                st[i] = dense
            dense = max(dense, st[i] * t.shape[i])
        st = tuple(st)
    return st


def _vector(t, name, n, device):
    """int32 [n], contiguous, on the device."""
    if t.dtype is _I32 and t.shape == (n,) and t.get_device() == device and (n < 2 or t.stride(0) == 1):
        return
    _check_dev(t, (_I32,), name)
    if t.shape != (n,):
        raise ValueError(f"{name} has shape {tuple(t.shape)}, expected ({n},)")
    raise ValueError(f"{name} is on another device")


def _kv_view(k, v, device, kv_len=None, page_table=None, cu_k=None):
    """asm_kv_t of paged k, v [pages, page_size, heads, head_dim] or packed k, v [rows, heads, head_dim]."""
    if not _DT:
        _dtypes()
    paged = page_table is not None
    shape, st = k.shape, _strides(k)
    if (k.dtype not in _H16 or v.dtype != k.dtype or shape != v.shape or st != _strides(v) or st[-1] != 1
            or len(st) != (4 if paged else 3) or not k.get_device() == v.get_device() == device >= 0):
        for t, name in ((k, "k"), (v, "v")):
            _dense(t, name, 4 if paged else 3, _H16)
        if shape != v.shape or k.dtype != v.dtype or st != _strides(v):
            raise ValueError(f"k and v must agree in shape, strides and type: {tuple(k.shape)} {k.stride()} {k.dtype}, "
                             f"{tuple(v.shape)} {v.stride()} {v.dtype}")
        raise ValueError("k, v and the rows are on different devices")
    if paged:
        batch, width = page_table.shape
        if (page_table.dtype is not _I32 or page_table.get_device() != device
                or (width > 1 and page_table.stride(1) != 1)):
            _dense(page_table, "page_table", 2, (_I32,))
            raise ValueError("page_table is on another device")
        _vector(kv_len, "kv_len", batch, device)
        return (_KV_PACK(k.data_ptr(), v.data_ptr(), st[0], st[1], st[2], page_table.data_ptr(),
                         page_table.stride(0) if batch > 1 else width, kv_len.data_ptr(), 0, batch, shape[0], shape[1],
                         width, shape[2], shape[3], _H16[k.dtype], 0), batch)
    batch = cu_k.shape[0] - 1
    _vector(cu_k, "cu_k", batch + 1, device)
    return (_KV_PACK(k.data_ptr(), v.data_ptr(), max(st[0], 8), st[0], st[1], 0, 0, 0, cu_k.data_ptr(), batch, 1,
                     shape[0], 0, shape[1], shape[2], _H16[k.dtype], 0), batch)


def _no_keys(k, stream):
    """One row in place of none: no sequence has a key, but a tensor without elements has no address."""
    if stream is None:
        return k.new_zeros((1, *k.shape[1:]))
    with _torch().cuda.stream(stream):
        return k.new_zeros((1, *k.shape[1:]))


def _query(q, k, out, out_dtype, stream):
    """Checks q [rows, heads, head_dim] against k and returns (strides, out)."""
    if not _DT:
        _dtypes()
    shape, st = q.shape, _strides(q)
    if q.dtype not in _H16 or not q.is_cuda or len(shape) != 3 or st[2] != 1:
        _dense(q, "q", 3, _H16)
    heads = k.shape[-2]
    if q.dtype != k.dtype or shape[2] != k.shape[-1]:
        raise ValueError(f"q {q.dtype} of head_dim {shape[2]} against keys {k.dtype} of {k.shape[-1]}")
    if heads == 0 or shape[1] == 0 or shape[1] % heads:
        raise ValueError(f"{shape[1]} query heads are not a multiple of {heads} KV heads")
    if out is None:
        dt = out_dtype or q.dtype
        if dt != q.dtype and dt != _F32:
            raise TypeError(f"out_dtype {dt}: fp32 or q's type")
        return st, _empty(q, shape, dt, stream)
    _check_dev(out, (q.dtype, _F32), "out")
    if out.data_ptr() == q.data_ptr() and q.numel():
        raise ValueError("out must not be q: queries are read again after rows have been written")
    if out.shape != shape or (out_dtype is not None and out.dtype != out_dtype):
        raise ValueError(f"out: {tuple(out.shape)} {out.dtype}, expected {tuple(shape)} {out_dtype or q.dtype}")
    return st, out


def rope_append(qkv, rope_cs, kv_len, page_table, k_pages, v_pages, n_heads: int, *, cu_q=None, q_out=None,
                stream=None):
    """Rotary positions on the query and key heads of qkv [T, (nh + 2 nkv) * hd] (fp32 or the cache's
    type) and append of keys and values to their pages (asm_rope_append_async).

    Row t of sequence s (cu_q int32 [B + 1]; without it row s is sequence s) is the position
    kv_len[s] - (rows of s) + (t - cu_q[s]): kv_len counts the new rows already.  k_pages, v_pages
    [pages, page_size, nkv, hd] fp16 or bf16 (any strides, hd dense), page_table int32 [B, n], rope_cs fp32
    [positions, hd/2, 2] (decode.rope_table).  Returns the rotated queries [T, nh, hd] in the cache's
    type; rows at or past cu_q[B] are not written."""
    if page_table is None:
        raise ValueError("page_table is required")
    device = qkv.get_device()
    if device < 0:
        raise TypeError("qkv: expected a CUDA tensor")
    kv, batch = _kv_view(k_pages, v_pages, device, kv_len, page_table)
    dt = k_pages.dtype
    nkv, hd = k_pages.shape[2:]
    if (qkv.dtype is not _F32 and qkv.dtype is not dt) or qkv.dim() != 2 or qkv.stride(1) != 1:
        _dense(qkv, "qkv", 2, (_F32, dt))
    T = qkv.shape[0]
    if qkv.shape[1] != (n_heads + 2 * nkv) * hd:
        raise ValueError(f"qkv has {qkv.shape[1]} columns, expected ({n_heads} + 2 * {nkv}) * {hd}")
    if rope_cs.dtype is not _F32 or not rope_cs.is_cuda or not rope_cs.is_contiguous():
        _check_dev(rope_cs, (_F32,), "rope_cs")
    if rope_cs.shape[1:] != (hd // 2, 2):
        raise ValueError(f"rope_cs {tuple(rope_cs.shape)}: expected [positions, {hd // 2}, 2]")
    if cu_q is not None:
        _vector(cu_q, "cu_q", batch + 1, device)
    elif T != batch:
        raise ValueError(f"{T} rows for {batch} sequences: pass cu_q")
    if q_out is None:
        q_out = _empty(qkv, (T, n_heads, hd), dt, stream)
    else:
        _check_dev(q_out, (dt,), "q_out")
        if q_out.shape != (T, n_heads, hd):
            raise ValueError(f"q_out {tuple(q_out.shape)}: expected {(T, n_heads, hd)}")
    if T == 0 or batch == 0:
        return q_out
    _call((native._lib or native.lib()).asm_rope_append_async(
        qkv.data_ptr(), _DT[qkv.dtype], qkv.stride(0) if T > 1 else qkv.shape[1], rope_cs.data_ptr(),
        rope_cs.shape[0], None if cu_q is None else cu_q.data_ptr(), T, n_heads, q_out.data_ptr(), kv,
        _current_stream(device) if stream is None else stream.cuda_stream))
    return q_out


def attention_prompt(q, k, v, cu_q, *, cu_k=None, kv_len=None, page_table=None, scale: float | None = None, out=None,
                     out_dtype=None, stream=None):
    """Causal attention of packed prompts q [T, nh, hd], fp16 or bf16 (asm_attention_prompt_async).

    Sequence s owns rows cu_q[s] .. cu_q[s + 1] - 1 (int32 [B + 1]).  Keys and values are packed
    [Tk, nkv, hd] with offsets cu_k (cu_q where they are the prompt's own), or the pages of a cache
    [pages, page_size, nkv, hd] with page_table int32 [B, n] and kv_len int32 [B].  The last row of a
    sequence sees all its keys; earlier rows one less each; a row without keys gives zeros.  scale
    (positive) defaults to hd ** -0.5.  out [T, nh, hd] in q's type or fp32 (whose weights have two 16-bit
    parts: about a third more time); rows at or past cu_q[B] are not written."""
    if (page_table is None) != (kv_len is None) or (page_table is not None and cu_k is not None):
        raise ValueError("pass page_table and kv_len (paged) or cu_k (packed)")
    device = q.get_device()
    if page_table is None and device >= 0 and k.dim() == 3 and k.shape[0] == 0 == v.shape[0]:
        k = v = _no_keys(k, stream)
    kv, batch = _kv_view(k, v, device, kv_len, page_table, cu_q if cu_k is None else cu_k)
    _vector(cu_q, "cu_q", batch + 1, device)
    st, out = _query(q, k, out, out_dtype, stream)
    T, nh, hd = q.shape
    if T == 0 or batch == 0:
        return out
    _call((native._lib or native.lib()).asm_attention_prompt_async(
        q.data_ptr(), st[0], st[1], cu_q.data_ptr(), T, nh, hd ** -0.5 if scale is None else scale, out.data_ptr(),
        _DT[out.dtype], kv, _current_stream(device) if stream is None else stream.cuda_stream))
    return out


def attention_paged_workspace(batch: int, n_heads: int, n_kv_heads: int, head_dim: int) -> int:
    """Bytes of scratch one attention_paged call needs (asm_attention_paged_workspace)."""
    n = int(native.lib().asm_attention_paged_workspace(batch, n_heads, n_kv_heads, head_dim))
    if n < 0:
        native.check()
    return n


def attention_paged(q, k_pages, v_pages, page_table, kv_len, *, scale: float | None = None, out=None, out_dtype=None,
                    workspace=None, stream=None):
    """Attention of one new token per sequence, q [B, nh, hd] fp16 or bf16, over a paged cache
    (asm_attention_paged_async): k_pages, v_pages [pages, page_size, nkv, hd], page_table int32 [B, n],
    kv_len int32 [B] (the new token counted).  kv_len 0 gives zeros.  scale (positive) defaults to
    hd ** -0.5.  out [B, nh, hd] in q's type or fp32.  workspace: uint8 of attention_paged_workspace bytes,
    one per call that may overlap another (a call without one takes it from torch's allocator)."""
    if page_table is None:
        raise ValueError("page_table is required")
    device = q.get_device()
    kv, batch = _kv_view(k_pages, v_pages, device, kv_len, page_table)
    st, out = _query(q, k_pages, out, out_dtype, stream)
    B, nh, hd = q.shape
    if B != batch:
        raise ValueError(f"q has {B} rows for {batch} sequences")
    lib = native._lib or native.lib()
    if B == 0:
        return out
    if workspace is None:
        need = lib.asm_attention_paged_workspace(B, nh, k_pages.shape[2], hd)
        if need < 0:
            native.check()
        workspace = _empty(q, (need,), _U8, stream)
    else:
        _check_dev(workspace, (_U8,), "workspace")
    _call(lib.asm_attention_paged_async(
        q.data_ptr(), st[0], st[1], nh, hd ** -0.5 if scale is None else scale, out.data_ptr(), _DT[out.dtype], kv,
        workspace.data_ptr(), workspace.numel(), _current_stream(device) if stream is None else stream.cuda_stream))
    return out


def rows_sample(logits, u, *, temperature=None, top_k=None, top_p=None, min_p=None, tokens=None, stream=None):
    """The next token of each row of logits [B, V] (fp32, fp16 or bf16; V <= 262144) from the given
    numbers u fp32 [B] in [0, 1) (asm_rows_sample_async).

    temperature, top_p, min_p fp32 [B] and top_k int32 [B], each optional (1, 1, 0, off).  top_k first,
    then top_p of what is left, then min_p of the largest probability; ties go to the lower index; the
    word is the first, in index order, whose cumulative probability exceeds u.  temperature 0: the first
    maximum.  NaN is never chosen; a row of NaN and -inf gives -1.  Returns int32 [B]."""
    if not _DT:
        _dtypes()
    if logits.dtype not in _DT or not logits.is_cuda or logits.dim() != 2 or logits.stride(1) != 1:
        _dense(logits, "logits", 2, _DT)
    B, V = shape = logits.shape
    device = logits.get_device()
    if tokens is None:
        tokens = _empty(logits, shape[:1], _I32, stream)
    ptr, rows = [], shape[:1]
    for t, name, dt in ((u, "u", _F32), (temperature, "temperature", _F32), (top_k, "top_k", _I32),
                        (top_p, "top_p", _F32), (min_p, "min_p", _F32), (tokens, "tokens", _I32)):
        if t is None and name != "u":
            ptr.append(None)
            continue
        if t.dtype is not dt or t.get_device() != device or t.shape != rows or (B > 1 and t.stride(0) != 1):
            _check_dev(t, (dt,), name)
            raise ValueError(f"{name}: shape {tuple(t.shape)} on device {t.get_device()}, expected ({B},) on {device}")
        ptr.append(t.data_ptr())
    _call((native._lib or native.lib()).asm_rows_sample_async(logits.data_ptr(), _DT[logits.dtype], B, V,
                                             logits.stride(0) if B > 1 else V, *ptr, _current_stream(device) if stream is None else stream.cuda_stream))
    return tokens


# --------------------------------------------------------------------------
# Serving operators around an 8-bit cache, shared prefixes and logits
#
# Where a tensor is (which device, or none) is looked at by the library, once
# a pointer; when it refuses a call, the tensors are gone through for the one
# at fault.  Types, shapes and strides are only known here.
# --------------------------------------------------------------------------

_SPACE: dict = {}  # (function, sizes) -> bytes of workspace
_cuda_empty = None
_ready = False


def _setup():
    """_dtypes, and torch's quickest way to an uninitialised tensor (0.9 us, new_empty takes 2) where it has it.

    The name is not a public one: it is used where it does what is expected of it, once a process."""
    global _cuda_empty, _ready
    _dtypes()
    _ready = True
    try:
        from torch._C._dynamo.guards import _empty_strided_cuda as quick
        t = quick((2, 3), (3, 1), _I8)
        if t.is_cuda and t.dtype is _I8 and tuple(t.shape) == (2, 3) and t.stride() == (3, 1):
            _cuda_empty = quick
    except Exception:  # whatever another release of torch does there: new_empty then
        pass


def _fresh(like, shape, dtype, stream):
    """_empty on the current device (where the library wants its tensors), dense."""
    if stream is not None or _cuda_empty is None:
        return _empty(like, shape, dtype, stream)
    if len(shape) == 3:
        return _cuda_empty(shape, (shape[1] * shape[2], shape[2], 1), dtype)
    return _cuda_empty(shape, (shape[1], 1) if len(shape) == 2 else (1,), dtype)


def _place(t, name):
    device = t.get_device()
    if device < 0:
        raise TypeError(f"{name}: expected a CUDA tensor")
    return device


def _ran(rc, tensors):
    """Raises what the library refused: a TypeError or ValueError that names the tensor where it is one's place."""
    if not rc:
        return
    code, message = native.last_error()
    where = None
    for t, name in tensors:
        if t is None or not t.numel():
            continue
        if not t.is_cuda:
            raise TypeError(f"{name}: expected a CUDA tensor")
        where = t.get_device() if where is None else where
        if t.get_device() != where:
            raise ValueError(f"{name} is on device {t.get_device()}, {tensors[0][1]} on {where}")
    raise AsmError(code or rc, message or "call failed")


def _column(t, name, n, dtype):
    """[n] of dtype, dense."""
    if t.dtype is dtype and t.dim() == 1 and t.shape[0] == n and (n < 2 or t.is_contiguous()):
        return t.data_ptr()
    if t.dtype is not dtype:
        raise TypeError(f"{name}: dtype {t.dtype}, expected {dtype}")
    raise ValueError(f"{name}: shape {tuple(t.shape)} with strides {t.stride()}, expected ({n},), dense")


def _table(page_table):
    """Checked int32 [batch, width]: (address, row stride, batch, width)."""
    if page_table is None:
        raise ValueError("page_table is required")
    if page_table.dtype is not _I32 or page_table.dim() != 2:
        raise TypeError(f"page_table: expected int32 with 2 axes, got {page_table.dtype} {tuple(page_table.shape)}")
    batch, width = page_table.shape
    row, col = page_table.stride()
    if width > 1 and col != 1:
        raise ValueError(f"page_table: rows must be dense, got strides {page_table.stride()}")
    return page_table.data_ptr(), row if batch > 1 else width, batch, width


def _kv_q8_view(k, v, k_scales, v_scales, kv_len, page_table):
    """asm_kv_q8_t of codes k, v int8 [pages, page_size, heads, head_dim] and scales fp16
    [pages, heads, page_size, head_dim / 32]."""
    shape, st, ss = k.shape, k.stride(), k_scales.stride()
    if not (k.dtype is v.dtype is _I8 and k_scales.dtype is v_scales.dtype is _F16 and len(st) == 4 == len(ss)
            and v.shape == shape and (v.stride() == st or _strides(v) == _strides(k)) and v_scales.shape == k_scales.shape
            and (v_scales.stride() == ss or _strides(v_scales) == _strides(k_scales))):
        for t, name, dt in ((k, "k", _I8), (v, "v", _I8), (k_scales, "k_scales", _F16), (v_scales, "v_scales", _F16)):
            if t.dtype is not dt:
                raise TypeError(f"{name}: dtype {t.dtype}, expected {dt}")
        raise ValueError(f"k and v, and their scales, must have 4 axes and agree in shape and strides: {tuple(k.shape)} "
                         f"{k.stride()}, {tuple(v.shape)} {v.stride()}; {tuple(k_scales.shape)} {k_scales.stride()}, "
                         f"{tuple(v_scales.shape)} {v_scales.stride()}")
    pages, size, heads, hd = shape
    per = hd // 32
    if k_scales.shape != (pages, heads, size, per) or hd % 32:
        raise ValueError(f"k_scales {tuple(k_scales.shape)}: expected [pages, heads, page_size, head_dim / 32] of "
                         f"k {tuple(shape)}")
    page, token, head, one = st
    if one != 1 or (per > 1 and ss[3] != 1) or (size > 1 and ss[2] != per):
        raise ValueError(f"head_dim, and a head's scales of a page, must be dense: k {k.stride()}, k_scales "
                         f"{k_scales.stride()}")
    spage, shead = ss[0], ss[1]
    if heads == 1:  # the stride of an axis with one entry means nothing
        head, shead = hd, size * per
    if pages == 1:
        page, spage = token * size, heads * size * per
    table, row, batch, width = _table(page_table)
    return _KV_Q8_PACK(k.data_ptr(), v.data_ptr(), k_scales.data_ptr(), v_scales.data_ptr(), page, token, head,
                       spage, shead, table, row, _column(kv_len, "kv_len", batch, _I32), batch, pages, size, width,
                       heads, hd), batch, heads, hd


def rope_append_q8(qkv, rope_cs, kv_len, page_table, k_pages, v_pages, k_scales, v_scales, n_heads: int, *, cu_q=None,
                   q_dtype=None, q_out=None, stream=None):
    """rope_append into a Q8_0 cache (asm_rope_append_q8_async): codes k_pages, v_pages int8
    [pages, page_size, nkv, hd] (any strides, hd dense), scales fp16 [pages, nkv, page_size, hd / 32] (the
    last two axes dense).

    Keys are rotated in fp32, and keys and values quantized in blocks of 32 as quantize_q8_0 does it, the
    scale rounded to fp16.  qkv fp32, or fp16 or bf16 (the queries' type then).  Returns the rotated queries
    [T, nh, hd] in q_dtype (qkv's type; fp16 for fp32)."""
    device = _place(qkv, "qkv")
    if not _ready:
        _setup()
    kv, batch, nkv, hd = _kv_q8_view(k_pages, v_pages, k_scales, v_scales, kv_len, page_table)
    src = qkv.dtype
    if src not in _DT:
        raise TypeError(f"qkv: dtype {src} not in {tuple(_DT)}")
    T, cols = qkv.shape
    row, col = qkv.stride()
    if cols != (n_heads + 2 * nkv) * hd or col != 1:
        raise ValueError(f"qkv {tuple(qkv.shape)} with strides {qkv.stride()}, expected dense rows of ({n_heads} + "
                         f"2 * {nkv}) * {hd}")
    if rope_cs.dtype is not _F32 or rope_cs.shape[1:] != (hd // 2, 2) or not rope_cs.is_contiguous():
        if rope_cs.dtype is not _F32:
            raise TypeError(f"rope_cs: dtype {rope_cs.dtype}, expected fp32")
        raise ValueError(f"rope_cs {tuple(rope_cs.shape)}: expected [positions, {hd // 2}, 2], dense")
    cu = None
    if cu_q is not None:
        cu = _column(cu_q, "cu_q", batch + 1, _I32)
    elif T != batch:
        raise ValueError(f"{T} rows for {batch} sequences: pass cu_q")
    dt = q_dtype or (q_out.dtype if q_out is not None else _F16 if src is _F32 else src)
    if dt not in _H16 or (src is not _F32 and src is not dt):
        raise TypeError(f"queries of {dt} from qkv of {src}: fp16 or bf16, from fp32 or the same type")
    if q_out is None:
        q_out = _fresh(qkv, (T, n_heads, hd), dt, stream)
    elif q_out.dtype is not dt or q_out.shape != (T, n_heads, hd) or not q_out.is_contiguous():
        if q_out.dtype is not dt:
            raise TypeError(f"q_out: dtype {q_out.dtype}, expected {dt}")
        raise ValueError(f"q_out {tuple(q_out.shape)}: expected {(T, n_heads, hd)}, dense")
    if T == 0 or batch == 0:
        return q_out
    rc = (native._lib or native.lib()).asm_rope_append_q8_async(
        qkv.data_ptr(), _DT[src], row if T > 1 else cols, rope_cs.data_ptr(), rope_cs.shape[0], cu, T, n_heads,
        q_out.data_ptr(), _H16[dt], kv,
        _current_stream(device) if stream is None else stream.cuda_stream)
    if rc:
        _ran(rc, ((qkv, "qkv"), (rope_cs, "rope_cs"), (kv_len, "kv_len"), (page_table, "page_table"), (k_pages, "k_pages"),
                  (v_pages, "v_pages"), (k_scales, "k_scales"), (v_scales, "v_scales"), (cu_q, "cu_q"), (q_out, "q_out")))
    return q_out


def cache_read_q8(k_pages, v_pages, k_scales, v_scales, page_table, kv_len, cu, rows: int, *, dtype=None, out=None,
                  stream=None):
    """Keys and values of a Q8_0 cache as packed 16-bit rows (asm_cache_read_q8_async), for attention_prompt
    with cu_k=cu.

    Sequence s gets rows cu[s] .. cu[s + 1] - 1 (int32 [B + 1]) of `rows` in all: its last positions, as many
    as it has rows (cu of the sums of kv_len reads everything, cu_q what a call has just appended).  Returns
    (k, v) [rows, nkv, hd] in dtype (fp16 unless given) or in out=(k, v); rows before a sequence's first
    position are zeros, rows at or past cu[B] are not written."""
    device = _place(k_pages, "k_pages")
    if not _ready:
        _setup()
    kv, batch, nkv, hd = _kv_q8_view(k_pages, v_pages, k_scales, v_scales, kv_len, page_table)
    at = _column(cu, "cu", batch + 1, _I32)
    shape = (rows, nkv, hd)
    if rows < 0:
        raise ValueError(f"rows {rows}")
    dt = dtype or (_F16 if out is None else out[0].dtype)
    if dt not in _H16:
        raise TypeError(f"dtype {dt}: fp16 or bf16")
    if out is None:
        k, v = _fresh(k_pages, shape, dt, stream), _fresh(k_pages, shape, dt, stream)
    else:
        k, v = out
        for t, name in ((k, "out[0]"), (v, "out[1]")):
            if t.dtype is not dt:
                raise TypeError(f"{name}: dtype {t.dtype}, expected {dt}")
            if t.shape != shape or not t.is_contiguous():
                raise ValueError(f"{name} {tuple(t.shape)}: expected {shape}, dense")
    if rows == 0 or batch == 0:
        return k, v
    rc = (native._lib or native.lib()).asm_cache_read_q8_async(
        kv, at, rows, k.data_ptr(), v.data_ptr(), _H16[dt],
        _current_stream(device) if stream is None else stream.cuda_stream)
    if rc:
        _ran(rc, ((k_pages, "k_pages"), (v_pages, "v_pages"), (k_scales, "k_scales"), (v_scales, "v_scales"),
                  (page_table, "page_table"), (kv_len, "kv_len"), (cu, "cu"), (k, "out[0]"), (v, "out[1]")))
    return k, v


def _decode_query(q, batch, nkv, hd, out, out_dtype, stream):
    """Checks q [B, heads, head_dim] against the cache; (row stride, head stride, heads, out)."""
    shape, st = q.shape, q.stride()
    if q.dtype not in _H16 or len(st) != 3:
        raise TypeError(f"q: expected fp16 or bf16 with 3 axes, got {q.dtype} {tuple(shape)}")
    B, nh, d = shape
    row, head, one = st
    if B == 1:  # the stride of an axis with one entry means nothing
        row = nh * hd
    if nh == 1:
        head = hd
    if d != hd or one != 1 or B != batch:
        raise ValueError(f"q {tuple(shape)} with strides {q.stride()}: expected {batch} sequences and head_dim {hd}, dense")
    if nkv == 0 or nh == 0 or nh % nkv:
        raise ValueError(f"{nh} query heads are not a multiple of {nkv} KV heads")
    if out is None:
        dt = out_dtype or q.dtype
        if dt is not q.dtype and dt is not _F32:
            raise TypeError(f"out_dtype {dt}: fp32 or q's type")
        return row, head, nh, _fresh(q, (B, nh, hd), dt, stream)
    if (out.dtype is not q.dtype and out.dtype is not _F32) or (out_dtype is not None and out.dtype is not out_dtype):
        raise TypeError(f"out: dtype {out.dtype}, expected {out_dtype or q.dtype}")
    if out.shape != shape or not out.is_contiguous():
        raise ValueError(f"out {tuple(out.shape)}: expected {tuple(shape)}, dense")
    return row, head, nh, out


def _scratch(q, workspace, function, sizes, stream):
    """The given workspace, or a new one of the bytes function(*sizes) asks for."""
    if workspace is not None:
        if workspace.dtype is not _U8 or not workspace.is_contiguous():
            raise TypeError(f"workspace: expected dense uint8, got {workspace.dtype}")
        return workspace
    need = _SPACE.get((function, sizes))
    if need is None:
        need = int(getattr(native.lib(), function)(*sizes))
        if need < 0:
            native.check()
        if len(_SPACE) > 4096:
            _SPACE.clear()
        _SPACE[function, sizes] = need
    return _fresh(q, (need,), _U8, stream)


def attention_paged_q8_workspace(batch: int, n_heads: int, n_kv_heads: int, head_dim: int) -> int:
    """Bytes of scratch one attention_paged_q8 call needs (asm_attention_paged_q8_workspace)."""
    n = int(native.lib().asm_attention_paged_q8_workspace(batch, n_heads, n_kv_heads, head_dim))
    if n < 0:
        native.check()
    return n


def attention_paged_q8(q, k_pages, v_pages, k_scales, v_scales, page_table, kv_len, *, scale: float | None = None,
                       out=None, out_dtype=None, workspace=None, stream=None):
    """attention_paged over a Q8_0 cache (asm_attention_paged_q8_async): q [B, nh, hd] fp16 or bf16, the cache
    as rope_append_q8 fills it, page_table int32 [B, n], kv_len int32 [B].  out [B, nh, hd] in q's type or
    fp32.  workspace: uint8 of attention_paged_q8_workspace bytes, one per call that may overlap another."""
    device = _place(q, "q")
    if not _ready:
        _setup()
    kv, batch, nkv, hd = _kv_q8_view(k_pages, v_pages, k_scales, v_scales, kv_len, page_table)
    row, head, nh, out = _decode_query(q, batch, nkv, hd, out, out_dtype, stream)
    if batch == 0:
        return out
    workspace = _scratch(q, workspace, "asm_attention_paged_q8_workspace", (batch, nh, nkv, hd), stream)
    rc = (native._lib or native.lib()).asm_attention_paged_q8_async(
        q.data_ptr(), _H16[q.dtype], row, head, nh, hd ** -0.5 if scale is None else scale, out.data_ptr(),
        _DT[out.dtype], kv, workspace.data_ptr(), workspace.shape[0],
        _current_stream(device) if stream is None else stream.cuda_stream)
    if rc:
        _ran(rc, ((q, "q"), (k_pages, "k_pages"), (v_pages, "v_pages"), (k_scales, "k_scales"), (v_scales, "v_scales"),
                  (page_table, "page_table"), (kv_len, "kv_len"), (out, "out"), (workspace, "workspace")))
    return out


def attention_shared_workspace(batch: int, groups: int, n_heads: int, n_kv_heads: int, head_dim: int) -> int:
    """Bytes of scratch one attention_shared call needs (asm_attention_shared_workspace)."""
    n = int(native.lib().asm_attention_shared_workspace(batch, groups, n_heads, n_kv_heads, head_dim))
    if n < 0:
        native.check()
    return n


def attention_shared(q, k_pages, v_pages, page_table, kv_len, cu_group, shared_len, *, scale: float | None = None,
                     out=None, out_dtype=None, workspace=None, stream=None):
    """attention_paged where groups of sequences begin with the same pages, which are read once for the whole
    group (asm_attention_shared_async).

    Sequences cu_group[i] .. cu_group[i + 1] - 1 (int32 [G + 1]) have their first shared_len[i] positions
    (int32 [G], rounded down to whole pages) in common: their rows of page_table begin alike, kv_len counts
    all positions.  A sequence in no group, or shorter than what its group shares, is on its own.  The rest is
    attention_paged's, but for one rounding: with 16-bit outputs the weights over shared positions are rounded once
    to 16 bits, as attention_prompt's are (attention_paged and out_dtype=torch.float32 have two parts of them).
    workspace: uint8 of attention_shared_workspace bytes, one per call that may overlap another."""
    device = _place(q, "q")
    if not _ready:
        _setup()
    shape, st = k_pages.shape, k_pages.stride()
    if not (k_pages.dtype is v_pages.dtype is q.dtype in _H16 and len(st) == 4 and v_pages.shape == shape
            and (v_pages.stride() == st or _strides(v_pages) == _strides(k_pages)) and st[3] == 1):
        if not k_pages.dtype is v_pages.dtype is q.dtype in _H16:
            raise TypeError(f"q {q.dtype}, k_pages {k_pages.dtype}, v_pages {v_pages.dtype}: fp16 or bf16, all the same")
        raise ValueError(f"k_pages and v_pages must have 4 axes, the last one dense, and agree in shape and strides: "
                         f"{tuple(shape)} {k_pages.stride()}, {tuple(v_pages.shape)} {v_pages.stride()}")
    pages, size, nkv, hd = shape
    page, token, khead, _ = st
    if nkv == 1:  # the stride of an axis with one entry means nothing
        khead = hd
    if pages == 1:
        page = token * size
    table, trow, batch, width = _table(page_table)
    row, head, nh, out = _decode_query(q, batch, nkv, hd, out, out_dtype, stream)
    if shared_len.dim() != 1:
        raise ValueError(f"shared_len {tuple(shared_len.shape)}: expected one axis")
    groups = shared_len.shape[0]
    shared, cu = _column(shared_len, "shared_len", groups, _I32), _column(cu_group, "cu_group", groups + 1, _I32)
    lens = _column(kv_len, "kv_len", batch, _I32)
    if batch == 0:
        return out
    workspace = _scratch(q, workspace, "asm_attention_shared_workspace", (batch, groups, nh, nkv, hd), stream)
    rc = (native._lib or native.lib()).asm_attention_shared_async(
        q.data_ptr(), row, head, nh, hd ** -0.5 if scale is None else scale, out.data_ptr(), _DT[out.dtype],
        _KV_PACK(k_pages.data_ptr(), v_pages.data_ptr(), page, token, khead, table, trow, lens, 0, batch, pages, size,
                 width, nkv, hd, _H16[q.dtype], 0),
        cu, shared, groups, workspace.data_ptr(), workspace.shape[0],
        _current_stream(device) if stream is None else stream.cuda_stream)
    if rc:
        _ran(rc, ((q, "q"), (k_pages, "k_pages"), (v_pages, "v_pages"), (page_table, "page_table"), (kv_len, "kv_len"),
                  (cu_group, "cu_group"), (shared_len, "shared_len"), (out, "out"), (workspace, "workspace")))
    return out


def _rows2(t, name, rows, dtype):
    """[rows, n] of dtype with dense rows: (address, n, row stride)."""
    if t.dtype is not dtype:
        raise TypeError(f"{name}: dtype {t.dtype}, expected {dtype}")
    shape = t.shape
    if len(shape) != 2 or shape[0] != rows:
        raise ValueError(f"{name}: shape {tuple(shape)}, expected {rows} rows")
    row, col = t.stride()
    n = shape[1]
    if n > 1 and col != 1:
        raise ValueError(f"{name}: rows must be dense, got strides {t.stride()}")
    return t.data_ptr(), n, row if rows > 1 else n


def rows_adjust(logits, *, tokens=None, n_tokens=None, n_prompt=None, repetition=None, frequency=None, presence=None,
                bias_tokens=None, bias=None, allowed=None, out=None, stream=None):
    """Logits [B, V] (fp32, fp16 or bf16; V <= 262144) with penalties, biases and a mask, for rows_sample
    (asm_rows_adjust_async).

    In fp32: words among tokens [B, L] int32 (the first n_tokens[r] of a row) are multiplied by 1 / repetition
    where they are above 0 and by repetition elsewhere; words that come c > 0 times from n_prompt[r] on lose
    frequency * c + presence; words among bias_tokens int32 [B, N] (-1: unused; N <= 1024) gain their bias
    fp32 [B, N], those of equal entries added up; words whose bit is 0 in allowed int32 [B, ceil(V / 32)] (bit
    w % 32 of w / 32) become -inf.  n_tokens, n_prompt int32 [B] (L, 0) and repetition, frequency, presence
    fp32 [B] (1, 0, 0) are optional.  Returns a new tensor, or out, which may be logits."""
    device = _place(logits, "logits")
    if not _ready:
        _setup()
    dt = logits.dtype
    if dt not in _DT or logits.dim() != 2:
        raise TypeError(f"logits: expected fp32, fp16 or bf16 with 2 axes, got {dt} {tuple(logits.shape)}")
    B, V = logits.shape
    at, _, row = _rows2(logits, "logits", B, dt)
    if out is None:
        out = _fresh(logits, (B, V), dt, stream)
        to, n, to_row = out.data_ptr(), V, V
    else:
        to, n, to_row = _rows2(out, "out", B, dt)
    if n != V:
        raise ValueError(f"out {tuple(out.shape)}: expected {(B, V)}")
    token = held = token_row = 0
    n1 = n2 = rep = freq = pres = words = biases = bits = bits_row = n_bias = 0
    if tokens is not None:
        token, held, token_row = _rows2(tokens, "tokens", B, _I32)
        if n_tokens is not None:
            n1 = _column(n_tokens, "n_tokens", B, _I32)
        if n_prompt is not None:
            n2 = _column(n_prompt, "n_prompt", B, _I32)
        if repetition is not None:
            rep = _column(repetition, "repetition", B, _F32)
        if frequency is not None:
            freq = _column(frequency, "frequency", B, _F32)
        if presence is not None:
            pres = _column(presence, "presence", B, _F32)
        if held == 0:  # nothing is read, and an array without elements has no address
            token = n1 = n2 = rep = freq = pres = 0
    elif not (n_tokens is n_prompt is repetition is frequency is presence is None):
        raise ValueError("penalties without tokens")
    if bias_tokens is not None and bias is not None:
        words, n_bias, row1 = _rows2(bias_tokens, "bias_tokens", B, _I32)
        biases, m, row2 = _rows2(bias, "bias", B, _F32)
        if m != n_bias or m and (row1 != m or row2 != m):
            raise ValueError(f"bias_tokens {tuple(bias_tokens.shape)} and bias {tuple(bias.shape)}: expected equal, dense ones")
        if m == 0:
            words = biases = 0
    elif not (bias_tokens is bias is None):
        raise ValueError("pass bias_tokens and bias together")
    if allowed is not None:
        bits, n, bits_row = _rows2(allowed, "allowed", B, _I32)
        if n < (V + 31) // 32:
            raise ValueError(f"allowed has {n} words of 32 bits a row, {(V + 31) // 32} are needed")
    if B == 0 or V == 0:
        return out
    rc = (native._lib or native.lib()).asm_rows_adjust_async(
        _ADJUST_PACK(at, to, row, to_row, _DT[dt], B, V, held, token, token_row, n1, n2, rep, freq, pres, words, biases,
                     bits, bits_row, n_bias, 0),
        _current_stream(device) if stream is None else stream.cuda_stream)
    if rc:
        _ran(rc, ((logits, "logits"), (out, "out"), (tokens, "tokens"), (n_tokens, "n_tokens"), (n_prompt, "n_prompt"),
                  (repetition, "repetition"), (frequency, "frequency"), (presence, "presence"),
                  (bias_tokens, "bias_tokens"), (bias, "bias"), (allowed, "allowed")))
    return out
