"""Refusals of the operators around the Q8_0 cache, shared prefixes and logits that need no GPU: the C entries reject
bad descriptors before touching the device, and the Python layer rejects what is not a CUDA tensor."""
from __future__ import annotations

import ctypes
import struct

import pytest

from asmllm_b200 import native, ops


@pytest.fixture(scope="module")
def L():
    return native.try_load_native_library()


def kv8(**over):
    d = native.KvQ8()
    base = dict(k=4096, v=8192, k_scales=256, v_scales=512, page_stride=2048, token_stride=128, head_stride=128,
                scale_page_stride=64, scale_head_stride=64, table=64, table_stride=4, len=64, batch=2, n_pages=8,
                page_size=16, table_width=4, n_kv_heads=1, head_dim=128)
    for name, value in {**base, **over}.items():
        setattr(d, name, value)
    return d


def kv16(**over):
    d = native.Kv()
    base = dict(k=4096, v=8192, page_stride=2048, token_stride=128, head_stride=128, table=64, table_stride=4, len=64,
                batch=2, n_pages=8, page_size=16, table_width=4, n_kv_heads=1, head_dim=128, dtype=native.DT_F16)
    for name, value in {**base, **over}.items():
        setattr(d, name, value)
    return d


def adjust(**over):
    d = native.Adjust()
    base = dict(logits=64, out=4096, stride=10, out_stride=10, dtype=native.DT_F32, rows=2, n=10)
    for name, value in {**base, **over}.items():
        setattr(d, name, value)
    return d


def calls(L, d):
    p = ctypes.byref(d)
    yield L.asm_rope_append_q8_async(64, native.DT_F32, 384, 64, 32, None, 2, 1, 64, native.DT_F16, p, None)
    yield L.asm_cache_read_q8_async(p, 64, 2, 64, 128, native.DT_F16, None)
    yield L.asm_attention_paged_q8_async(64, native.DT_F16, 128, 128, 1, 1.0, 64, native.DT_F16, p, 64, 1 << 30, None)


@pytest.mark.parametrize("over,code,text", [
    (dict(head_dim=96), 2, "head_dim"), (dict(batch=-1), 1, "batch"), (dict(n_kv_heads=0), 1, "n_kv_heads"),
    (dict(n_pages=0), 1, "n_pages"), (dict(page_size=8), 2, "page_size"), (dict(page_size=48), 2, "page_size"),
    (dict(page_size=512), 2, "page_size"), (dict(table=None), 1, "page table"), (dict(table_width=0), 1, "table_width"),
    (dict(table_stride=3), 1, "table_stride"), (dict(token_stride=120), 1, "strides"), (dict(head_stride=0), 1, "strides"),
    (dict(page_stride=-2048), 1, "strides"), (dict(scale_page_stride=4), 1, "scale strides"),
    (dict(scale_head_stride=-8), 1, "scale strides"), (dict(k=4100), 1, "aligned"), (dict(v_scales=520), 1, "aligned"),
])
def test_bad_cache_descriptors(L, over, code, text):
    for rc in calls(L, kv8(**over)):
        assert rc == code
        got, msg = native.last_error()
        assert got == code and text in msg


def test_null_descriptors(L):
    for call in (lambda: L.asm_rope_append_q8_async(64, 0, 384, 64, 32, None, 2, 1, 64, 1, None, None),
                 lambda: L.asm_cache_read_q8_async(None, 64, 2, 64, 128, 1, None),
                 lambda: L.asm_attention_paged_q8_async(64, 1, 128, 128, 1, 1.0, 64, 1, None, 64, 1 << 30, None),
                 lambda: L.asm_attention_shared_async(64, 128, 128, 1, 1.0, 64, 1, None, 64, 64, 1, 64, 1 << 30, None),
                 lambda: L.asm_rows_adjust_async(None, None)):
        assert call() == 1
        assert "null" in native.last_error()[1]


def test_bad_arguments(L):
    p = ctypes.byref(kv8())
    for call, code, text in [
        (lambda: L.asm_rope_append_q8_async(64, 0, 384, 64, 32, None, 2, 0, 64, 1, p, None), 1, "n_heads"),
        (lambda: L.asm_rope_append_q8_async(64, 0, 384, 64, 32, None, 3, 1, 64, 1, p, None), 1, "rows"),
        (lambda: L.asm_rope_append_q8_async(64, 0, 384, 64, 0, None, 2, 1, 64, 1, p, None), 1, "rope_len"),
        (lambda: L.asm_rope_append_q8_async(64, 0, 384, 64, 32, None, 2, 1, 64, 0, p, None), 2, "q_out"),
        (lambda: L.asm_rope_append_q8_async(64, 2, 384, 64, 32, None, 2, 1, 64, 1, p, None), 2, "qkv"),
        (lambda: L.asm_rope_append_q8_async(64, 0, 376, 64, 32, None, 2, 1, 64, 1, p, None), 1, "qkv_stride"),
        (lambda: L.asm_rope_append_q8_async(68, 0, 384, 64, 32, None, 2, 1, 64, 1, p, None), 1, "misaligned"),
        (lambda: L.asm_cache_read_q8_async(p, 64, -1, 64, 128, 1, None), 1, "rows"),
        (lambda: L.asm_cache_read_q8_async(p, 64, 2, 64, 128, 0, None), 2, "fp16 or bf16"),
        (lambda: L.asm_cache_read_q8_async(p, 64, 2, 72, 128, 1, None), 1, "misaligned"),
        (lambda: L.asm_attention_paged_q8_async(64, 0, 128, 128, 1, 1.0, 64, 0, p, 64, 1 << 30, None), 2, "q is"),
        (lambda: L.asm_attention_paged_q8_async(64, 1, 128, 128, 1, 0.0, 64, 1, p, 64, 1 << 30, None), 1, "scale"),
        (lambda: L.asm_attention_paged_q8_async(64, 1, 100, 128, 1, 1.0, 64, 1, p, 64, 1 << 30, None), 1, "strides"),
        (lambda: L.asm_attention_paged_q8_async(64, 1, 128, 128, 1, 1.0, 64, 2, p, 64, 1 << 30, None), 2, "out"),
        (lambda: L.asm_attention_paged_q8_async(64, 1, 128, 128, 1, 1.0, 64, 1, p, 64, 100, None), 1, "workspace"),
        (lambda: L.asm_attention_paged_q8_async(64, 1, 128, 128, 1, 1.0, 64, 1, ctypes.byref(kv8(batch=40000)), 64, 1 << 40, None), 2, "batch"),
    ]:
        rc = call()
        got, msg = native.last_error()
        assert rc == code == got and text in msg, msg
    p = ctypes.byref(kv16())
    for call, code, text in [
        (lambda: L.asm_attention_shared_async(64, 128, 128, 1, 1.0, 64, 1, p, 64, 64, -1, 64, 1 << 30, None), 1, "groups"),
        (lambda: L.asm_attention_shared_async(64, 128, 128, 1, 1.0, 64, 1, p, 64, 64, 1, 64, 100, None), 1, "workspace"),
        (lambda: L.asm_attention_shared_async(64, 128, 128, 1, -1.0, 64, 1, p, 64, 64, 1, 64, 1 << 30, None), 1, "scale"),
        (lambda: L.asm_attention_shared_async(64, 128, 128, 1, 1.0, 64, 2, p, 64, 64, 1, 64, 1 << 30, None), 2, "out"),
        (lambda: L.asm_attention_shared_async(64, 128, 128, 1, 1.0, 64, 1, p, 64, 64, 40000, 64, 1 << 30, None), 2, "at most"),
        (lambda: L.asm_attention_shared_async(64, 1 << 13, 128, 1 << 9, 1.0, 64, 1, ctypes.byref(kv16(batch=1 << 14)), 64, 64, 1, 64,
                                      1 << 40, None), 2, "2^22"),
        (lambda: L.asm_attention_shared_async(64, 128, 128, 1, 1.0, 64, 1, ctypes.byref(kv16(table=None)), 64, 64, 1, 64, 1 << 30,
                                      None), 1, "page table"),
    ]:
        rc = call()
        got, msg = native.last_error()
        assert rc == code == got and text in msg, msg
    for args in ((-1, 4, 2, 128), (1, 3, 2, 128), (1, 4, 2, 96)):
        with pytest.raises(ops.AsmError):
            ops.attention_paged_q8_workspace(*args)
        with pytest.raises(ops.AsmError):
            ops.attention_shared_workspace(args[0], 1, *args[1:])
    with pytest.raises(ops.AsmError):
        ops.attention_shared_workspace(1, -1, 4, 2, 128)
    assert ops.attention_paged_q8_workspace(0, 4, 2, 128) == 0 == ops.attention_shared_workspace(0, 3, 4, 2, 128)


@pytest.mark.parametrize("over,code,text", [
    (dict(rows=-1), 1, "rows"), (dict(n=0), 1, "n > 0"), (dict(stride=9), 1, "strides"), (dict(out_stride=9), 1, "strides"),
    (dict(rows=70000), 2, "65535"), (dict(n=(1 << 18) + 1, stride=1 << 19, out_stride=1 << 19), 2, "at most"),
    (dict(dtype=3), 2, "logits type"), (dict(logits=66), 1, "misaligned"), (dict(out=65, dtype=1), 1, "misaligned"),
    (dict(tokens=64, held=-1), 1, "held"), (dict(tokens=64, held=5, token_stride=4), 1, "held"),
    (dict(repetition=64), 1, "without tokens"), (dict(n_tokens=64), 1, "without tokens"),
    (dict(n_bias=3, bias=64), 1, "biases"), (dict(n_bias=-1), 1, "n_bias"),
    (dict(n_bias=1025, bias=64, bias_tokens=64), 2, "1025"), (dict(allowed=64, allowed_stride=0), 1, "allowed_stride"),
    (dict(tokens=64, held=(1 << 28) + 1, token_stride=1 << 29), 2, "2^28"),
])
def test_bad_adjustments(L, over, code, text):
    assert L.asm_rows_adjust_async(ctypes.byref(adjust(**over)), None) == code
    got, msg = native.last_error()
    assert got == code and text in msg


def test_nothing_to_do_is_no_call(L):
    p = ctypes.byref(kv8(batch=0))
    assert L.asm_rope_append_q8_async(64, 0, 384, 64, 32, None, 0, 1, 64, 1, p, None) == 0
    assert L.asm_cache_read_q8_async(p, 64, 0, 64, 128, 1, None) == 0
    assert L.asm_attention_paged_q8_async(64, 1, 128, 128, 1, 1.0, 64, 1, p, 64, 1 << 30, None) == 0
    assert L.asm_attention_shared_async(64, 128, 128, 1, 1.0, 64, 1, ctypes.byref(kv16(batch=0)), 64, 64, 1, 64, 1 << 30, None) == 0
    assert L.asm_rows_adjust_async(ctypes.byref(adjust(rows=0)), None) == 0


def test_host_memory_is_refused(L):
    import numpy as np

    buf = np.zeros(1 << 16, dtype=np.uint8)
    at = (buf.ctypes.data + 255) & ~255
    for rc in calls(L, kv8(k=at, v=at, k_scales=at, v_scales=at, table=at, len=at)):
        assert rc == native.ASM_E_NOT_DEVICE
        assert "device pointer" in native.last_error()[1]
    d = kv16(k=at, v=at, table=at, len=at)
    assert L.asm_attention_shared_async(at, 128, 128, 1, 1.0, at, 1, ctypes.byref(d), at, at, 1, at, 1 << 30,
                                        None) == native.ASM_E_NOT_DEVICE
    native.last_error()
    assert L.asm_rows_adjust_async(ctypes.byref(adjust(logits=at, out=at)), None) == native.ASM_E_NOT_DEVICE
    native.last_error()


def test_descriptors_are_packed_as_declared():
    assert struct.calcsize("QQQQqqqqqQqQiiiiii") == ctypes.sizeof(native.KvQ8)
    assert struct.calcsize("QQqqiiiiQqQQQQQQQQqii") == ctypes.sizeof(native.Adjust)


def test_python_layer_refuses_host_tensors():
    torch = pytest.importorskip("torch")
    x, h, s = torch.zeros(2, 4, 128), torch.zeros(2, 16, 1, 128, dtype=torch.int8), torch.zeros(2, 1, 16, 4).half()
    t, n = torch.zeros(2, 2, dtype=torch.int32), torch.zeros(2, dtype=torch.int32)
    for call in (lambda: ops.rope_append_q8(x.view(2, -1), x, n, t, h, h, s, s, 2),
                 lambda: ops.cache_read_q8(h, h, s, s, t, n, n, 2),
                 lambda: ops.attention_paged_q8(x.half(), h, h, s, s, t, n),
                 lambda: ops.attention_shared(x.half(), h.half(), h.half(), t, n, n, n[:1]),
                 lambda: ops.rows_adjust(x[:, 0])):
        with pytest.raises(TypeError):
            call()
