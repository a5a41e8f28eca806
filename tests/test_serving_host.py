"""Refusals of the serving operators that need no GPU: the C entries reject bad descriptors before touching the
device, and the Python layer rejects what is not a CUDA tensor."""
from __future__ import annotations

import ctypes

import pytest

from asmllm_b200 import native, ops


@pytest.fixture(scope="module")
def L():
    return native.try_load_native_library()


def kv(**over):
    d = native.Kv()
    base = dict(k=4096, v=8192, page_stride=2048, token_stride=128, head_stride=128, table=64, table_stride=4, len=64,
                batch=2, n_pages=8, page_size=16, table_width=4, n_kv_heads=1, head_dim=128, dtype=native.DT_F16)
    for name, value in {**base, **over}.items():
        setattr(d, name, value)
    return d


BAD_KV = [
    (dict(dtype=native.DT_F32), 2, "cache type"), (dict(head_dim=96), 2, "head_dim"), (dict(batch=-1), 1, "batch"),
    (dict(n_kv_heads=0), 1, "n_kv_heads"), (dict(n_pages=0), 1, "n_pages"), (dict(page_size=8), 2, "page_size"),
    (dict(page_size=48), 2, "page_size"), (dict(page_size=512), 2, "page_size"),
    (dict(table_width=0), 1, "table_width"), (dict(table_stride=3), 1, "table_stride"),
    (dict(token_stride=100), 1, "strides"), (dict(head_stride=0), 1, "strides"),
    (dict(page_stride=-2048), 1, "strides"), (dict(k=4100), 1, "aligned"), (dict(v=8196), 1, "aligned"),
]


def calls(L, d):
    p = ctypes.byref(d)
    yield L.asm_rope_append_async(64, native.DT_F32, 384, 64, 32, None, 2, 1, 64, p, None)
    yield L.asm_attention_prompt_async(64, 128, 128, 64, 2, 1, 1.0, 64, native.DT_F16, p, None)
    yield L.asm_attention_paged_async(64, 128, 128, 1, 1.0, 64, native.DT_F16, p, 64, 1 << 30, None)


@pytest.mark.parametrize("over,code,text", BAD_KV)
def test_bad_cache_descriptors(L, over, code, text):
    for rc in calls(L, kv(**over)):
        assert rc == code
        got, msg = native.last_error()
        assert got == code and text in msg


def test_null_descriptors_and_missing_table(L):
    assert L.asm_rope_append_async(64, 0, 384, 64, 32, None, 2, 1, 64, None, None) == 1
    assert "null" in native.last_error()[1]
    d = kv(table=None)
    assert L.asm_rope_append_async(64, 0, 384, 64, 32, None, 2, 1, 64, ctypes.byref(d), None) == 1
    assert "page table" in native.last_error()[1]
    assert L.asm_attention_paged_async(64, 128, 128, 1, 1.0, 64, 1, ctypes.byref(d), 64, 1 << 30, None) == 1
    assert "page table" in native.last_error()[1]
    assert L.asm_attention_prompt_async(64, 128, 128, 64, 2, 1, 1.0, 64, 1, ctypes.byref(d), None) == 1
    assert "one page" in native.last_error()[1]  # packed keys are a single page


def test_bad_queries(L):
    p = ctypes.byref(kv())
    for args, code, text in [
        ((64, 0, 384, 64, 32, None, 2, 0, 64), 1, "n_heads"),
        ((64, 0, 384, 64, 32, None, 3, 1, 64), 1, "rows"),           # three rows, two sequences, no offsets
        ((64, 0, 384, 64, 0, None, 2, 1, 64), 1, "rope_len"),
        ((64, native.DT_BF16, 384, 64, 32, None, 2, 1, 64), 2, "qkv"),
        ((64, 0, 376, 64, 32, None, 2, 1, 64), 1, "qkv_stride"),
        ((68, 0, 384, 64, 32, None, 2, 1, 64), 1, "misaligned"),
    ]:
        assert L.asm_rope_append_async(*args, p, None) == code
        assert text in native.last_error()[1]
    for args, code, text in [
        ((64, 100, 128, 64, 2, 1, 1.0, 64, 1), 1, "strides"),
        ((64, 128, 0, 64, 2, 1, 1.0, 64, 1), 1, "strides"),
        ((66, 128, 128, 64, 2, 1, 1.0, 64, 1), 1, "aligned"),
        ((64, 128, 128, 64, 2, 1, 1.0, 64, native.DT_BF16), 2, "out"),
        ((64, 128, 128, 64, -1, 1, 1.0, 64, 1), 1, "rows"),
        ((64, 128, 128, 64, (1 << 22) + 1, 1, 1.0, 64, 1), 2, "rows"),
    ]:
        assert L.asm_attention_prompt_async(*args, p, None) == code
        assert text in native.last_error()[1]
    d = kv(n_kv_heads=2)
    assert L.asm_attention_paged_async(64, 384, 128, 3, 1.0, 64, 1, ctypes.byref(d), 64, 1 << 30, None) == 1
    assert "multiple" in native.last_error()[1]
    assert L.asm_attention_paged_async(64, 128, 128, 1, 1.0, 64, 1, p, 64, -1, None) == 1
    assert "workspace" in native.last_error()[1]
    assert L.asm_attention_paged_async(64, 128, 128, 1, 1.0, 64, 1, p, 72, 1 << 30, None) == 1
    assert "workspace" in native.last_error()[1]
    assert L.asm_attention_paged_workspace(1, 3, 2, 128) == -1
    native.last_error()
    assert L.asm_attention_paged_workspace(1, 4, 2, 96) == -1
    native.last_error()
    with pytest.raises(ops.AsmError):
        ops.attention_paged_workspace(-1, 4, 2, 128)


def test_bad_samples(L):
    for args, code, text in [
        ((64, 0, -1, 10, 10), 1, "rows"), ((64, 0, 1, 0, 10), 1, "n > 0"), ((64, 0, 1, 10, 9), 1, "stride"),
        ((64, 0, 1, (1 << 18) + 1, 1 << 19), 2, "at most"), ((64, 3, 1, 10, 10), 2, "logits type"),
        ((66, 0, 1, 10, 10), 1, "misaligned"), ((65, 1, 1, 10, 10), 1, "misaligned"),
    ]:
        assert L.asm_rows_sample_async(*args, 64, None, None, None, None, 64, None) == code
        assert text in native.last_error()[1]


def test_nothing_to_do_is_no_call(L):
    d = kv(batch=0)
    for rc in calls_empty(L, d):
        assert rc == 0
    assert L.asm_rows_sample_async(64, 0, 0, 10, 10, 64, None, None, None, None, 64, None) == 0


def calls_empty(L, d):
    p = ctypes.byref(d)
    yield L.asm_rope_append_async(64, native.DT_F32, 384, 64, 32, None, 0, 1, 64, p, None)
    yield L.asm_attention_prompt_async(64, 128, 128, 64, 0, 1, 1.0, 64, native.DT_F16, p, None)
    yield L.asm_attention_paged_async(64, 128, 128, 1, 1.0, 64, native.DT_F16, p, 64, 1 << 30, None)


def test_host_memory_is_refused(L):
    import numpy as np

    buf = np.zeros(1 << 16, dtype=np.uint8)
    at = (buf.ctypes.data + 255) & ~255
    d = kv(k=at, v=at, table=at, len=at)
    for rc in calls(L, d):
        assert rc == native.ASM_E_NOT_DEVICE
        assert "device pointer" in native.last_error()[1]
    assert L.asm_rows_sample_async(at, 0, 1, 10, 10, at, None, None, None, None, at, None) == native.ASM_E_NOT_DEVICE
    native.last_error()


def test_python_layer_refuses_host_tensors():
    torch = pytest.importorskip("torch")
    x, h = torch.zeros(2, 4, 128), torch.zeros(2, 16, 1, 128, dtype=torch.float16)
    t, n = torch.zeros(2, 2, dtype=torch.int32), torch.zeros(2, dtype=torch.int32)
    with pytest.raises(TypeError):
        ops.rope_append(x.view(2, -1), x, n, t, h, h, 2)
    with pytest.raises(TypeError):
        ops.attention_prompt(x.half(), h, h, n, kv_len=n, page_table=t)
    with pytest.raises(TypeError):
        ops.attention_paged(x.half(), h, h, t, n)
    with pytest.raises(TypeError):
        ops.rows_sample(x[:, 0], n)


# ------------------------------------------------------------------ a bound that one 16-bit rounding of a weight exceeds
# Scores that come out exactly (one value of q and of each key is not zero, both short) leave the weights' own errors:
# the scaled score and maximum, at most 1.4427 each, are off by 1.5 * 2^-24 of themselves and their difference by half
# a step, under 2^-21 in all, and the exponential by 2^-22; the two 16-bit parts by u^2 (and 2^-38 of the largest weight
# where fp16 runs out of exponent); sums of n terms by n * 2^-23.  Twice, for the weighted sum and the sum of weights.
WEIGHT_CASES = [1, 2, 3, 5, 9, 17, 33]  # keys


def one_value_case(torch, dt, n, nkv, hd, device, seed):
    """q [1, nkv, hd], k, v [n, nkv, hd]: scores k[:, :, 0] in eighths from -1 to 1, values of both signs."""
    g = torch.Generator().manual_seed(seed)
    q = torch.zeros(1, nkv, hd, dtype=dt)
    q[..., 0] = 1.0
    k = torch.zeros(n, nkv, hd, dtype=dt)
    k[..., 0] = (torch.randint(-8, 9, (n, nkv), generator=g) / 8).to(dt)
    v = torch.randn(n, nkv, hd, generator=g).to(dt)
    return [t.to(device) for t in (q, k, v)]


def one_value_exact(torch, k, v):
    """Outputs [1, nkv, hd] in 64 bits and the bound above."""
    p = torch.softmax(k[..., 0].double(), 0)
    want, pv = (torch.einsum("nh,nhd->hd", p, x)[None] for x in (v.double(), v.double().abs()))
    u = torch.finfo(v.dtype).eps / 2
    part = u * u + (len(v) * 2.0 ** -38 if v.dtype == torch.float16 else 0.0)
    return want, 2 * (2.0 ** -21 + 2.0 ** -22 + part + len(v) * 2.0 ** -23) * pv + 2.0 ** -24 * want.abs()


@pytest.mark.parametrize("dtype", ["float16", "bfloat16"])
def test_the_bound_on_two_part_weights_shows_a_missing_part(dtype):
    torch = pytest.importorskip("torch")
    dt = getattr(torch, dtype)
    once = []
    for n in WEIGHT_CASES:
        _, k, v = one_value_case(torch, dt, n, 4, 128, "cpu", n)
        want, tol = one_value_exact(torch, k, v)
        w = 2.0 ** 14 * torch.exp(k[..., 0].double() - k[..., 0].double().amax(0))
        hi = w.to(dt).double()
        both = hi + (w - hi).to(dt).double()
        got = [torch.einsum("nh,nhd->hd", x, v.double())[None] / w.sum(0)[None, :, None] for x in (both, hi)]
        assert ((got[0] - want).abs() <= tol).all()
        once.append(float(((got[1] - want).abs() / tol).max()))
    assert min(once[1:]) > 5  # the second part left out: far outside at every length (a single weight is exact)
