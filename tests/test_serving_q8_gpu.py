"""The operators around the Q8_0 cache (ops.rope_append_q8, cache_read_q8, attention_paged_q8), attention over shared
prefixes (ops.attention_shared) and the changes to logits (ops.rows_adjust) on the GPU, against plain implementations.

Append and read back are compared bit for bit: the rotary products and sums and the quantizer's steps are single fp32
operations.  Tolerances of the attentions count roundings, as in test_serving_gpu.py (exact_attention, close); what is
different here:
  * Q8_0: a block's product of 32 codes and queries is exact in its terms and added up in fp32, the blocks' scales and
    sums take hd / 32 more roundings: the bound of hd truncated steps holds with 8 more.  bf16 queries are scaled to
    fp16: those below 2^-31 of the row's largest round by 2^-39 of it, which the same 8 steps of 2^-23 cover.
    The weights and their products with a scale are two fp16 parts each: 2 * 2^-22, and 2^-34 of the largest
    weight a position where fp16 runs out of exponent.
  * Shared prefix: the weights of the shared positions are rounded once to 16 bits (fp32 outputs: two parts)."""
from __future__ import annotations

import math

import numpy as np
import pytest

from asmllm_b200 import decode as D
from asmllm_b200 import native, ops
from test_serving_gpu import close, exact_attention, half_step, make_pages, prompt_weight, rand

pytestmark = pytest.mark.gpu


@pytest.fixture(autouse=True)
def clean_error_word(cuda):
    ops.device_error()
    yield
    assert ops.device_error() == 0


# ------------------------------------------------------------------ helpers
def blocks(x):
    """numpy Q8_0 of x fp32 [..., n] in the library's steps: codes int8 [..., n], scales fp16 [..., n / 32]."""
    with np.errstate(all="ignore"):
        b = x.astype(np.float32).reshape(*x.shape[:-1], -1, 32)
        a = np.abs(b).max(-1, keepdims=True)
        inv = np.where(a == 0, np.float32(0), np.float32(127) / a).astype(np.float32)
        t = (b * inv).astype(np.float32)
        codes = np.where(np.isnan(t), 0, np.rint(np.clip(t, -128, 127)))
        return codes.astype(np.int8).reshape(x.shape), (a[..., 0] / np.float32(127)).astype(np.float16)


def make_pages8(torch, dense, page, layout="token", extra=3, seed=0, fill=True):
    """Pages of per-sequence (k codes, k scales, v codes, v scales), NaN scales wherever no position lives."""
    nkv, hd = dense[0][0].shape[1:]
    need = [-(-d[0].shape[0] // page) for d in dense]
    total = sum(need) + extra
    perm = torch.randperm(total, generator=torch.Generator().manual_seed(seed)).tolist()
    if layout == "token":
        mk = lambda: torch.full((total, page, nkv, hd), 77, dtype=torch.int8, device="cuda")  # noqa: E731
        ms = lambda: torch.full((total, nkv, page, hd // 32), float("nan"), dtype=torch.float16, device="cuda")  # noqa: E731
    elif layout == "head":
        mk = lambda: torch.full((total, nkv, page, hd), 77, dtype=torch.int8, device="cuda").transpose(1, 2)  # noqa: E731
        ms = lambda: torch.full((nkv, total, page, hd // 32), float("nan"), dtype=torch.float16,  # noqa: E731
                                device="cuda").transpose(0, 1)
    else:  # rows and heads padded
        mk = lambda: torch.full((total, page, nkv, hd + 16), 77, dtype=torch.int8, device="cuda")[..., :hd]  # noqa: E731
        ms = lambda: torch.full((total, nkv, page * (hd // 32) + 8), float("nan"), dtype=torch.float16,  # noqa: E731
                                device="cuda")[..., :page * (hd // 32)].unflatten(-1, (page, hd // 32))
    k, v, ks, vs = mk(), mk(), ms(), ms()
    table = torch.full((len(need), max(need + [1]) + 2), -7, dtype=torch.int32)
    at = 0
    for s, n in enumerate(need):
        for i in range(n):
            pg = perm[at]
            at += 1
            table[s, i] = pg
            if not fill:
                continue
            for pages, scales, codes, d in ((k, ks, dense[s][0], dense[s][1]), (v, vs, dense[s][2], dense[s][3])):
                rows = codes[i * page:(i + 1) * page]
                pages[pg, :rows.shape[0]] = rows
                scales[pg, :, :rows.shape[0]] = d[i * page:(i + 1) * page].transpose(0, 1)
    return k, v, ks, vs, table.cuda()


def random8(torch, n, nkv, hd, seed, spread=0.0):
    """(k codes, k scales, v codes, v scales) of n positions; scales of very different sizes with spread."""
    g = torch.Generator(device="cuda").manual_seed(seed)
    code = lambda: torch.randint(-128, 128, (n, nkv, hd), generator=g, device="cuda").to(torch.int8)  # noqa: E731
    scale = lambda: (0.01 * torch.exp2(spread * torch.randn(n, nkv, hd // 32, generator=g, device="cuda"))).half()  # noqa: E731
    return code(), scale(), code(), scale()


def values(codes, scales):
    return codes.double() * scales.double().repeat_interleave(32, -1)


def rope_steps(x, cs):
    """numpy: pairs of x [T, heads, hd] rotated by cs [T, hd / 2, 2], each product and sum rounded to fp32."""
    x0, x1, c, s = x[..., 0::2], x[..., 1::2], cs[:, None, :, 0], cs[:, None, :, 1]
    out = np.empty_like(x)
    out[..., 0::2] = x0 * c - x1 * s
    out[..., 1::2] = x0 * s + x1 * c
    return out


def ints(torch, *x):
    return torch.tensor(x, dtype=torch.int32, device="cuda")


# ------------------------------------------------------------------ append and read back
@pytest.mark.parametrize("src,dtype", [("float32", "float16"), ("float32", "bfloat16"), ("float16", "float16"),
                                       ("bfloat16", "bfloat16")])
@pytest.mark.parametrize("nh,nkv,hd", [(4, 2, 128), (5, 1, 64), (32, 32, 128)])
@pytest.mark.parametrize("page,layout", [(16, "token"), (64, "head"), (256, "padded")])
def test_rope_append_q8(cuda, src, dtype, nh, nkv, hd, page, layout):
    torch = cuda
    dt, q_len, kv_len, tail = getattr(torch, dtype), [3, 1, 0, 40, 5], [3, 17, 9, 300, 2], 4
    T = sum(q_len)  # the last sequence has more rows than positions
    x = rand(torch, T + tail, (nh + 2 * nkv) * hd, dt=getattr(torch, src), seed=1)
    x[1, -hd:] = 0.0  # a block of zeros
    rope = D.rope_table(512, hd, 10000.0)
    dense = [random8(torch, n, nkv, hd, n) for n in kv_len]
    k, v, ks, vs, table = make_pages8(torch, dense, page, layout)
    before = [t.clone() for t in (k, v, ks, vs)]
    cu = ints(torch, *np.concatenate([[0], np.cumsum(q_len)]).tolist())
    q_out = torch.full((T + tail, nh, hd), 77.0, dtype=dt, device="cuda")
    got = ops.rope_append_q8(x, torch.from_numpy(rope).cuda(), ints(torch, *kv_len), table, k, v, ks, vs, nh, cu_q=cu,
                             q_out=q_out)
    assert got is q_out
    host, at = x.float().cpu().numpy().reshape(T + tail, nh + 2 * nkv, hd), 0
    for s, (n, m) in enumerate(zip(q_len, kv_len)):
        for i in range(n):
            p, row = m - n + i, host[at]
            at += 1
            if p < 0:
                assert (q_out[at - 1] == 0).all()
                continue
            qk = rope_steps(row[None, :nh + nkv], rope[p][None])[0]
            assert torch.equal(q_out[at - 1], torch.from_numpy(qk[:nh]).cuda().to(dt))
            pg = int(table[s, p // page])
            for pages, scales, old, old_d, new in ((k, ks, before[0], before[2], qk[nh:]),
                                                   (v, vs, before[1], before[3], row[nh + nkv:])):
                codes, d = blocks(new)
                assert np.array_equal(pages[pg, p % page].cpu().numpy(), codes)
                assert np.array_equal(scales[pg, :, p % page].cpu().numpy().view(np.uint16), d.view(np.uint16))
                old[pg, p % page], old_d[pg, :, p % page] = torch.from_numpy(codes).cuda(), torch.from_numpy(d).cuda()
    assert (q_out[T:] == 77).all()
    assert torch.equal(before[0], k) and torch.equal(before[1], v)  # and nothing else was written
    for a, b in ((before[2], ks), (before[3], vs)):
        assert torch.equal(a.contiguous().view(torch.int16), b.contiguous().view(torch.int16))


def test_rope_append_q8_codes_are_quantize_q8_0s_and_one_row_per_sequence(cuda):
    torch = cuda
    nh, nkv, hd, B = 6, 3, 128, 7
    wide = rand(torch, B, 8 + (nh + 2 * nkv) * hd, dt=torch.float32, seed=2, scale=30.0)
    x = wide[:, 8:]  # strided rows
    rope = torch.zeros(64, hd // 2, 2, device="cuda")
    rope[..., 0] = 1.0  # no rotation: keys are the rows themselves
    k, v, ks, vs, table = make_pages8(torch, [random8(torch, 33 + s, nkv, hd, s) for s in range(B)], 16)
    kv = ints(torch, *[33 + s for s in range(B)])
    q = ops.rope_append_q8(x, rope, kv, table, k, v, ks, vs, nh)
    assert q.dtype == torch.float16 and torch.equal(q, x[:, :nh * hd].view(B, nh, hd).half())
    codes, d = ops.quantize_q8_0_dev(x[:, nh * hd:].contiguous())
    for s in range(B):
        pg, at = int(table[s, (32 + s) // 16]), (32 + s) % 16
        got = torch.cat([k[pg, at].flatten(), v[pg, at].flatten()])
        assert torch.equal(got, codes[s])
        assert torch.equal(torch.cat([ks[pg, :, at].flatten(), vs[pg, :, at].flatten()]), d[s].half())


def test_rope_append_q8_infinities_and_nan_mark_their_block(cuda):
    torch = cuda
    nh = nkv = 1
    x = rand(torch, 1, 3 * 64, dt=torch.float32, seed=3)
    x[0, 128 + 5], x[0, 128 + 40] = float("inf"), float("nan")  # both blocks of the value
    rope = torch.zeros(4, 32, 2, device="cuda")
    rope[..., 0] = 1.0
    k, v, ks, vs, table = make_pages8(torch, [random8(torch, 1, 1, 64, 0)], 16)
    ops.rope_append_q8(x, rope, ints(torch, 1), table, k, v, ks, vs, nh)
    kr, vr = ops.cache_read_q8(k, v, ks, vs, table, ints(torch, 1), ints(torch, 0, 1), 1)
    assert torch.isfinite(kr).all() and torch.isnan(vr).all()


def test_rope_append_q8_refuses_positions_and_pages_on_the_device(cuda):
    torch = cuda
    nkv, hd = 1, 128
    rope = torch.from_numpy(D.rope_table(40, hd, 10000.0)).cuda()
    x = rand(torch, 1, 3 * hd, dt=torch.float32, seed=4)
    for length, width, page_no, bad in ((41, 4, None, True), (65, 4, None, True), (33, 4, 9, True), (33, 4, -1, True),
                                        (40, 4, None, False)):
        k, v, ks, vs, table = make_pages8(torch, [random8(torch, 64, nkv, hd, 0)], 16, extra=0)
        table = table[:, :width].contiguous()
        if page_no is not None:
            table[0, 2] = page_no
        before = [t.clone() for t in (k, v, ks, vs)]
        q = ops.rope_append_q8(x, rope, ints(torch, length), table, k, v, ks, vs, 1)
        assert ops.device_error() == (native.DEVERR_DECODE_RANGE if bad else 0)
        assert bool((q == 0).all()) == bad
        assert all(torch.equal(a, b) for a, b in zip(before, (k, v, ks, vs))) == bad
    # a length that no row meets, an offset beyond the rows
    cu = ints(torch, 0, 1, 1)
    k, v, ks, vs, table = make_pages8(torch, [random8(torch, 16, nkv, hd, s) for s in range(2)], 16)
    ops.rope_append_q8(x, rope, ints(torch, 3, -4), table, k, v, ks, vs, 1, cu_q=cu)
    assert ops.device_error() == native.DEVERR_DECODE_RANGE
    ops.rope_append_q8(x, rope, ints(torch, 3, 4), table, k, v, ks, vs, 1, cu_q=ints(torch, 0, 1, 2))
    assert ops.device_error() == native.DEVERR_DECODE_RANGE


@pytest.mark.parametrize("dtype", ["float16", "bfloat16"])
@pytest.mark.parametrize("nkv,hd,page,layout", [(2, 128, 16, "token"), (1, 64, 32, "head"), (32, 128, 128, "padded"),
                                                (3, 64, 256, "token")])
def test_cache_read_q8(cuda, dtype, nkv, hd, page, layout):
    torch = cuda
    dt, kv_len, read = getattr(torch, dtype), [37, 0, 1, 300, 64, 5], [37, 0, 1, 17, 64, 9]  # the last: more than it has
    dense = [random8(torch, n, nkv, hd, 7 + n, spread=4.0) for n in kv_len]
    k, v, ks, vs, table = make_pages8(torch, dense, page, layout)
    cu, tail = np.concatenate([[0], np.cumsum(read)]).tolist(), 3
    out = [torch.full((cu[-1] + tail, nkv, hd), 7.0, dtype=dt, device="cuda") for _ in "kv"]
    got = ops.cache_read_q8(k, v, ks, vs, table, ints(torch, *kv_len), ints(torch, *cu), cu[-1] + tail, out=out)
    assert got[0] is out[0] and got[1] is out[1]
    for s, (n, m) in enumerate(zip(read, kv_len)):
        for y, codes, scales in ((out[0], dense[s][0], dense[s][1]), (out[1], dense[s][2], dense[s][3])):
            want = torch.zeros(n, nkv, hd, dtype=dt, device="cuda")
            have = min(n, m)
            want[n - have:] = values(codes, scales)[m - have:].to(dt)
            assert torch.equal(y[cu[s]:cu[s + 1]], want)
    assert (out[0][cu[-1]:] == 7).all() and (out[1][cu[-1]:] == 7).all()


def test_cache_read_q8_reports_pages_and_offsets(cuda):
    torch = cuda
    k, v, ks, vs, table = make_pages8(torch, [random8(torch, 40, 1, 64, 0)], 16)
    table[0, 1] = 1000
    a, b = ops.cache_read_q8(k, v, ks, vs, table, ints(torch, 40), ints(torch, 0, 40), 40)
    assert ops.device_error() == native.DEVERR_DECODE_RANGE
    assert (a[16:32] == 0).all() and (b[16:32] == 0).all() and (a[:16] != 0).any() and (a[32:] != 0).any()
    ops.cache_read_q8(k, v, ks, vs, table, ints(torch, 40), ints(torch, 0, 41), 40)
    assert ops.device_error() == native.DEVERR_DECODE_RANGE


# ------------------------------------------------------------------ decode attention over the Q8_0 cache
def close8(torch, got, want, pv, serr, n, what=""):
    # 8 more steps of the scores' sums (of hd, at least 64), and two roundings of two fp16 parts
    close(torch, got, want, pv, serr * (1 + 8 / 64), n, 2 * 2.0 ** -22 + n * 2.0 ** -34, torch.float16, what)


@pytest.mark.parametrize("dtype,out", [("float16", "float32"), ("float16", "float16"), ("bfloat16", "bfloat16"),
                                       ("bfloat16", "float32")])
@pytest.mark.parametrize("nh,nkv,hd,page,layout,lens", [
    (1, 1, 128, 16, "token", [1, 0, 15, 16, 17, 33]),
    (32, 32, 128, 16, "head", [63, 64, 65, 1]),
    (64, 8, 128, 32, "token", [200, 0, 7, 640, 1000, 129]),
    (10, 2, 64, 64, "padded", [127, 128, 3, 900]),
    (40, 2, 64, 16, "token", [77, 300]),
    (12, 1, 128, 128, "head", [500, 1, 255]),
    (48, 1, 128, 256, "token", [2000, 31]),
])
def test_attention_paged_q8(cuda, dtype, out, nh, nkv, hd, page, layout, lens):
    torch = cuda
    dt, odt = getattr(torch, dtype), getattr(torch, out)
    dense = [random8(torch, n, nkv, hd, 3 + n, spread=1.0) for n in lens]
    k, v, ks, vs, table = make_pages8(torch, dense, page, layout)
    q = rand(torch, len(lens), nh, hd, dt=dt, seed=5, scale=0.3)
    kv = ints(torch, *lens)
    got = ops.attention_paged_q8(q, k, v, ks, vs, table, kv, out_dtype=odt)
    assert got.dtype == odt
    for s, n in enumerate(lens):
        want, pv, serr = exact_attention(torch, q[s:s + 1], values(*dense[s][:2]), values(*dense[s][2:]), hd ** -0.5, n - 1)
        close8(torch, got[s:s + 1], want, pv, serr, n, f"sequence {s}")
    again = ops.attention_paged_q8(q, k, v, ks, vs, table, kv, out_dtype=odt)
    assert torch.equal(got.view(torch.uint8), again.view(torch.uint8))  # the same bits every time


@pytest.mark.parametrize("spread", [4.0, 8.0])
def test_attention_paged_q8_scales_of_every_size(cuda, spread):
    """Scales from fp16's smallest to its largest: a block's output keeps its own precision."""
    torch = cuda
    n, nh, nkv, hd = 700, 16, 2, 128
    kc, kd, vc, vd = random8(torch, n, nkv, hd, 1)
    g = torch.Generator(device="cuda").manual_seed(2)
    vd = (0.01 * torch.exp2(spread * torch.randn(n, nkv, hd // 32, generator=g, device="cuda"))).clamp_max(60000.0).half()
    vd[100:200], vd[300] = 0.0, 2.0 ** -24
    dense = [(kc, kd, vc, vd)]
    k, v, ks, vs, table = make_pages8(torch, dense, 16)
    q = rand(torch, 1, nh, hd, dt=torch.float16, seed=5, scale=0.2)
    got = ops.attention_paged_q8(q, k, v, ks, vs, table, ints(torch, n), out_dtype=torch.float32)
    want, pv, serr = exact_attention(torch, q, values(kc, kd), values(vc, vd), hd ** -0.5, n - 1)
    # what runs out of exponent does so next to the largest weight and the block's largest scale
    worst = values(torch.full_like(vc, 127), vd).amax(0).repeat_interleave(nh // nkv, 0)[None]
    close8(torch, got, want, pv + n * 2.0 ** -33 * worst, serr, n)


def test_attention_paged_q8_queries_of_every_size_scale_and_strides(cuda):
    torch = cuda
    n, nh, nkv, hd = 90, 8, 2, 128
    dense = [random8(torch, n, nkv, hd, s) for s in range(5)]
    k, v, ks, vs, table = make_pages8(torch, dense, 16)
    q = rand(torch, 5, 2 * nh + 3, hd + 8, dt=torch.bfloat16, seed=6)[:, 3:nh + 3, :hd]  # strided rows and heads
    q[1] *= 1e-30
    q[2] *= 2.0 ** 30
    q[3, :, ::2] *= 2.0 ** -20  # some values far below the row's largest
    q[4] = 0.0
    ws = torch.empty(ops.attention_paged_q8_workspace(5, nh, nkv, hd), dtype=torch.uint8, device="cuda").fill_(255)
    out = torch.empty(5, nh, hd, dtype=torch.float32, device="cuda")
    for scale in (0.02, 3e-11):
        got = ops.attention_paged_q8(q, k, v, ks, vs, table, ints(torch, *[n] * 5), scale=scale, out=out, workspace=ws)
        assert got is out
        for s in range(5):
            if s == 2 and scale == 0.02:
                continue  # scores of 2^30: one key has all the weight or the difference of two is below their steps
            want, pv, serr = exact_attention(torch, q[s:s + 1], values(*dense[s][:2]), values(*dense[s][2:]), scale, n - 1)
            close8(torch, got[s:s + 1], want, pv, serr, n, f"sequence {s}, scale {scale}")


def test_attention_paged_q8_a_scale_that_is_not_finite_shows_in_its_block_alone(cuda):
    torch = cuda
    n, nh, nkv, hd = 100, 8, 2, 128
    for bad in (float("inf"), float("nan")):
        dense = [list(random8(torch, n, nkv, hd, s)) for s in range(3)]
        clean = ops.attention_paged_q8
        q = rand(torch, 3, nh, hd, dt=torch.float16, seed=5, scale=0.3)
        args = make_pages8(torch, dense, 16)
        lens = ints(torch, *[n] * 3)
        want = clean(q, *args[:4], args[4], lens, out_dtype=torch.float32)
        dense[1][3][50, 1, 2] = bad
        args = make_pages8(torch, dense, 16)
        got = clean(q, *args[:4], args[4], lens, out_dtype=torch.float32)
        hit = torch.zeros_like(got, dtype=torch.bool)
        hit[1, nh // 2:, 64:96] = True
        assert torch.isnan(got[hit]).all()
        # the other blocks: the same sums, another moment of rescaling
        assert float((got - want)[~hit].abs().max()) <= 2.0 ** -20 * float(want.abs().max())


def test_attention_paged_q8_bad_pages_and_lengths_are_reported(cuda):
    torch = cuda
    n, nkv, hd = 64, 1, 64
    kc, kd, vc, vd = random8(torch, n, nkv, hd, 0)
    k, v, ks, vs, table = make_pages8(torch, [(kc, kd, vc, vd)], 16, extra=0)
    table = table[:, :4].contiguous()
    q = rand(torch, 1, 4, hd, dt=torch.float16, seed=5, scale=0.3)
    table[0, 1] = 4
    got = ops.attention_paged_q8(q, k, v, ks, vs, table, ints(torch, n), out_dtype=torch.float32)
    assert ops.device_error() == native.DEVERR_DECODE_RANGE
    kk, vv = values(kc, kd), values(vc, vd)
    kk[16:32] = vv[16:32] = 0.0  # zero keys and values
    want, pv, serr = exact_attention(torch, q, kk, vv, hd ** -0.5, n - 1)
    close8(torch, got, want, pv, serr, n)
    table[0, 1] = table[0, 0]
    for length in (65, -1):
        ops.attention_paged_q8(q, k, v, ks, vs, table, ints(torch, length))
        assert ops.device_error() == native.DEVERR_DECODE_RANGE


def test_attention_paged_q8_many_and_long_sequences(cuda):
    torch = cuda
    nh, nkv, hd = 8, 1, 128
    lens = [(i * 37) % 90 for i in range(700)] + [60000]
    big = random8(torch, 60000, nkv, hd, 1)
    dense = [tuple(t[:n] if n < 60000 else t for t in big) for n in lens]
    k, v, ks, vs, table = make_pages8(torch, dense, 64, fill=False)
    for s, n in enumerate(lens):  # whole pages at a time
        for pages, scales, c, d in ((k, ks, 0, 1), (v, vs, 2, 3)):
            for i in range(0, n, 64):
                pg = int(table[s, i // 64]) if n < 60000 else None
                if pg is None:
                    break
                m = min(64, n - i)
                pages[pg, :m], scales[pg, :, :m] = big[c][i:i + m], big[d][i:i + m].transpose(0, 1)
            if n == 60000:
                pg, full = table[s, :60000 // 64].long(), 60000 // 64 * 64
                pages[pg] = big[c][:full].view(-1, 64, nkv, hd)
                scales[pg] = big[d][:full].view(-1, 64, nkv, hd // 32).transpose(1, 2)
                last = int(table[s, full // 64])
                pages[last, :60000 - full], scales[last, :, :60000 - full] = big[c][full:], big[d][full:].transpose(0, 1)
    q = rand(torch, len(lens), nh, hd, dt=torch.float16, seed=5, scale=0.3)
    got = ops.attention_paged_q8(q, k, v, ks, vs, table, ints(torch, *lens), out_dtype=torch.float32)
    for s in [0, 1, 2, 350, 699, 700]:
        n = lens[s]
        want, pv, serr = exact_attention(torch, q[s:s + 1], values(*dense[s][:2]), values(*dense[s][2:]), hd ** -0.5, n - 1)
        # sums of n terms lie in parts: no chain is longer than a CTA's share
        close8(torch, got[s:s + 1], want, pv, serr, min(n, 4096), f"sequence {s}")


# ------------------------------------------------------------------ attention over shared prefixes
def shared_case(torch, groups, alone, nkv, hd, dt, page, layout="token", seed=0):
    """groups: (rows, shared positions) of each; alone: positions of each sequence of its own.  (dense k, v, pages, table)"""
    dense_k, dense_v, heads = [], [], []
    at = 0
    for gi, (rows, shared) in enumerate(groups):
        pk, pv = rand(torch, shared, nkv, hd, dt=dt, seed=seed + 100 + gi), rand(torch, shared, nkv, hd, dt=dt, seed=seed + 200 + gi)
        for _ in range(rows):
            n = alone[at]
            dense_k.append(torch.cat([pk, rand(torch, n, nkv, hd, dt=dt, seed=seed + 300 + at)]))
            dense_v.append(torch.cat([pv, rand(torch, n, nkv, hd, dt=dt, seed=seed + 900 + at)]))
            heads.append(gi)
            at += 1
    kp, vp, table = make_pages(torch, dense_k, dense_v, page, layout)
    for s in range(1, len(heads)):  # the group's first pages, whole ones, are the first sequence's
        if heads[s] == heads[s - 1]:
            whole = groups[heads[s]][1] // page
            table[s, :whole] = table[s - 1, :whole]
    return dense_k, dense_v, kp, vp, table


def check_shared(torch, got, q, dense_k, dense_v, scale, dt, what=""):
    for s, (k, v) in enumerate(zip(dense_k, dense_v)):
        n = k.shape[0]
        want, pv, serr = exact_attention(torch, q[s:s + 1], k, v, scale, n - 1)
        u = half_step(torch, dt)
        w = 2 * u * u + (n * 2.0 ** -32 if dt == torch.float16 else 0.0) if got.dtype == torch.float32 else prompt_weight(torch, dt, n)
        close(torch, got[s:s + 1], want, pv, serr, min(n, 4096), w, dt, f"{what} sequence {s}")


@pytest.mark.parametrize("dtype,out", [("float16", "float32"), ("float16", "float16"), ("bfloat16", "bfloat16"),
                                       ("bfloat16", "float32")])
@pytest.mark.parametrize("nh,nkv,hd,page,layout,groups,alone", [
    (8, 1, 128, 16, "token", [(8, 64)], [1, 5, 64, 70, 0, 3, 16, 17]),              # one tile, one row without its own
    (8, 1, 128, 16, "token", [(5, 1024)], [1, 2, 3, 4, 5]),                            # split over many CTAs
    (64, 8, 128, 64, "head", [(40, 256)], [1 + i % 9 for i in range(40)]),             # 320 rows a head: two blocks
    (32, 32, 128, 16, "token", [(3, 48), (1, 16), (2, 400)], [9, 1, 30, 2, 100, 0]),   # groups; a row a head
    (10, 2, 64, 32, "padded", [(4, 96), (60, 320)], [i % 50 for i in range(64)]),      # blocks that split a sequence's heads
    (40, 2, 64, 16, "token", [(3, 160)], [3, 0, 40]),                                  # 20 heads a KV head
    (48, 1, 128, 256, "token", [(7, 512)], [0, 1, 2, 300, 4, 5, 6]),
    (6, 3, 128, 128, "head", [(2, 0), (3, 384)], [5, 0, 7, 8, 130]),                   # nothing shared: one's own alone
])
def test_attention_shared(cuda, dtype, out, nh, nkv, hd, page, layout, groups, alone):
    torch = cuda
    dt, odt = getattr(torch, dtype), getattr(torch, out)
    dense_k, dense_v, kp, vp, table = shared_case(torch, groups, alone, nkv, hd, dt, page, layout)
    B = len(alone)
    q = rand(torch, B, nh, hd, dt=dt, seed=5, scale=2.0)
    kv = ints(torch, *[k.shape[0] for k in dense_k])
    cu = ints(torch, *np.concatenate([[0], np.cumsum([r for r, _ in groups])]).tolist())
    shared = ints(torch, *[p for _, p in groups])
    got = ops.attention_shared(q, kp, vp, table, kv, cu, shared, out_dtype=odt)
    assert got.dtype == odt
    check_shared(torch, got, q, dense_k, dense_v, hd ** -0.5, dt)
    again = ops.attention_shared(q, kp, vp, table, kv, cu, shared, out_dtype=odt)
    assert torch.equal(got.view(torch.uint8), again.view(torch.uint8))
    # no groups: attention_paged's result
    none = ops.attention_shared(q, kp, vp, table, kv, cu[:1], shared[:0], out_dtype=odt)
    check_shared(torch, none, q, dense_k, dense_v, hd ** -0.5, dt, "no groups,")


def test_attention_shared_rows_that_do_not_share(cuda):
    """Sequences in no group, padded ones, shorter ones than their group shares, lengths inside a page."""
    torch = cuda
    nh, nkv, hd, page, dt = 8, 2, 128, 16, torch.float16
    dense_k, dense_v, kp, vp, table = shared_case(torch, [(1, 30), (6, 100), (1, 20)], [3, 40, 20, 60, 5, 1, 9, 7], nkv, hd, dt, page)
    q = rand(torch, 8, nh, hd, dt=dt, seed=5, scale=2.0)
    lens = [k.shape[0] for k in dense_k]
    lens[2], lens[3], lens[4] = 95, 0, 96  # 96 positions are shared: sequence 2 has fewer, 3 none, 4 exactly those
    for s in (2, 3, 4):
        dense_k[s], dense_v[s] = dense_k[s][:lens[s]], dense_v[s][:lens[s]]
    for odt in (torch.float16, torch.float32):
        got = ops.attention_shared(q, kp, vp, table, ints(torch, *lens), ints(torch, 1, 7), ints(torch, 100), out_dtype=odt)
        assert (got[3] == 0).all()
        check_shared(torch, got, q, dense_k, dense_v, hd ** -0.5, dt)
        # an empty group between two, and what a group says of rows it does not have
        got = ops.attention_shared(q, kp, vp, table, ints(torch, *lens), ints(torch, 0, 0, 1, 7, 7), ints(torch, 16, 16, 96, 48),
                                   out_dtype=odt)
        check_shared(torch, got, q, dense_k, dense_v, hd ** -0.5, dt)


@pytest.mark.parametrize("dtype", ["float16", "bfloat16"])
def test_attention_shared_long_prefix_keeps_fp32(cuda, dtype):
    """The tensor core truncates its sums: 16384 positions in one chain come out 1e-5 too small."""
    torch = cuda
    dt, nh, nkv, hd, page, P, B = getattr(torch, dtype), 64, 2, 128, 64, 16384, 6
    dense_k, dense_v, kp, vp, table = shared_case(torch, [(B, P)], [3] * B, nkv, hd, dt, page)
    for x in dense_v:
        x.add_(1.0)  # outputs near 1: a bias of the sums is one of the result
    vp.add_(1.0)
    q = rand(torch, B, nh, hd, dt=dt, seed=5)
    got = ops.attention_shared(q, kp, vp, table, ints(torch, *[P + 3] * B), ints(torch, 0, B), ints(torch, P),
                               out_dtype=torch.float32)
    for s in range(B):
        k, v = kp[table[s].clamp_min(0).long()].flatten(0, 1)[:P + 3], vp[table[s].clamp_min(0).long()].flatten(0, 1)[:P + 3]
        want, pv, serr = exact_attention(torch, q[s:s + 1], k, v, hd ** -0.5, P + 2)
        rel = float((got[s:s + 1].double() - want).norm() / want.norm())
        assert rel <= 3e-6, rel  # scores 2^-23 sqrt(hd) of 4 or so, weights 2^-16 of bf16, both averaged over thousands


def test_attention_shared_scores_that_rise_and_strided_queries(cuda):
    torch = cuda
    nh, nkv, hd, page, dt, P, B = 4, 1, 128, 16, torch.float16, 700 // 16 * 16, 40
    dense_k, dense_v, kp, vp, table = shared_case(torch, [(B, P)], [i % 4 for i in range(B)], nkv, hd, dt, page)
    ramp = torch.linspace(0.05, 2.0, P, device="cuda").to(dt)[:, None, None]  # each tile's maximum above the last one's
    for x in dense_k:
        x[:P] = ramp
    kp[table[0, :P // page].long()] = ramp.view(-1, page, 1, 1).expand(-1, -1, nkv, hd)
    wide = rand(torch, B, 3 * nh, hd + 8, dt=dt, seed=5).abs()
    q = wide[:, nh:2 * nh, :hd]
    kv = ints(torch, *[x.shape[0] for x in dense_k])
    for odt in (torch.float16, torch.float32):
        out = torch.empty(B, nh, hd, dtype=odt, device="cuda")
        ws = torch.full((ops.attention_shared_workspace(B, 1, nh, nkv, hd),), 255, dtype=torch.uint8, device="cuda")
        got = ops.attention_shared(q, kp, vp, table, kv, ints(torch, 0, B), ints(torch, P), scale=0.07, out=out, workspace=ws)
        assert got is out
        check_shared(torch, got, q, dense_k, dense_v, 0.07, dt)


def test_attention_shared_nan_elsewhere_does_not_reach_a_row(cuda):
    """NaN in the rest of a shared tile's pages, in another group, in what a shorter sequence does not have."""
    torch = cuda
    nh, nkv, hd, page, dt = 8, 1, 128, 16, torch.float16
    dense_k, dense_v, kp, vp, table = shared_case(torch, [(2, 80), (2, 32)], [3, 4, 5, 6], nkv, hd, dt, page)
    q = rand(torch, 4, nh, hd, dt=dt, seed=5, scale=2.0)
    kv, cu, shared = ints(torch, 83, 84, 37, 38), ints(torch, 0, 2, 4), ints(torch, 80, 32)
    nan_v = vp.clone()
    nan_v[table[0, 1].long()] = float("nan")  # a value that the first group attends to
    for odt in (dt, torch.float32):
        want = ops.attention_shared(q, kp, vp, table, kv, cu, shared, out_dtype=odt)
        got = ops.attention_shared(q, kp, nan_v, table, kv, cu, shared, out_dtype=odt)
        assert not torch.isfinite(got[:2]).any() and torch.equal(got[2:], want[2:])
        # sequences of the first group that have fewer positions than it shares stay clean of what they do not have
        short = ints(torch, 10, 84, 37, 38)
        got = ops.attention_shared(q, kp, nan_v, table, short, cu, shared, out_dtype=odt)
        check_shared(torch, got[:1], q[:1], [dense_k[0][:10]], [dense_v[0][:10]], hd ** -0.5, dt)


def test_attention_shared_reports_what_is_out_of_range(cuda):
    torch = cuda
    nh, nkv, hd, page, dt = 4, 1, 64, 16, torch.float16
    dense_k, dense_v, kp, vp, table = shared_case(torch, [(3, 64)], [3, 4, 5], nkv, hd, dt, page)
    q = rand(torch, 3, nh, hd, dt=dt, seed=5, scale=2.0)
    kv, cu, shared = ints(torch, 67, 68, 69), ints(torch, 0, 3), ints(torch, 64)
    for bad_cu in (ints(torch, 0, 4), ints(torch, -1, 3), ints(torch, 2, 1)):  # the group shares nothing
        got = ops.attention_shared(q, kp, vp, table, kv, bad_cu, shared)
        assert ops.device_error() == native.DEVERR_DECODE_RANGE
        check_shared(torch, got, q, dense_k, dense_v, hd ** -0.5, dt)
    for n in (-5, 10000):  # clipped: nothing, or more than any sequence has
        got = ops.attention_shared(q, kp, vp, table, kv, cu, ints(torch, n))
        assert ops.device_error() == native.DEVERR_DECODE_RANGE
        check_shared(torch, got, q, dense_k, dense_v, hd ** -0.5, dt)
    bad = table.clone()
    bad[:, 1] = 999
    got = ops.attention_shared(q, kp, vp, bad, kv, cu, shared)
    assert ops.device_error() == native.DEVERR_DECODE_RANGE
    for x in dense_k + dense_v:
        x[16:32] = 0.0
    check_shared(torch, got, q, dense_k, dense_v, hd ** -0.5, dt)
    ops.attention_shared(q, kp, vp, table, ints(torch, 67, -1, 69), cu, shared)
    assert ops.device_error() == native.DEVERR_DECODE_RANGE


# ------------------------------------------------------------------ logits
def exact_adjust(torch, x, tokens, n_tokens, n_prompt, rep, freq, pres, bias_tokens, bias, allowed):
    """64 bits, and the size of what was added up (for the roundings)."""
    y, size = x.double().clone(), x.double().abs()
    V = x.shape[1]
    for r in range(x.shape[0]):
        if tokens is not None:
            t = tokens[r, :n_tokens[r]].tolist()
            seen = sorted({w for w in t if 0 <= w < V})
            late = [w for w in t[max(0, n_prompt[r]):] if 0 <= w < V]
            if seen:
                v = y[r, seen]
                y[r, seen] = torch.where(v > 0, v / rep[r].double(), v * rep[r].double())
                size[r, seen] = torch.maximum(size[r, seen], y[r, seen].abs())
            for w in sorted(set(late)):
                c = late.count(w)
                y[r, w] -= freq[r].double() * c + pres[r].double()
                size[r, w] += freq[r].double().abs() * c + pres[r].double().abs()
        if bias is not None:
            for w, b in zip(bias_tokens[r].tolist(), bias[r].double().tolist()):
                if 0 <= w < V:
                    y[r, w] += b
                    size[r, w] += abs(b)
        if allowed is not None:
            bits = (allowed[r][:, None] >> torch.arange(32, device="cuda")) & 1
            y[r][bits.flatten()[:V] == 0] = -math.inf
    return y, size


def check_adjust(torch, got, want, size):
    inf = torch.isinf(want)
    assert torch.equal(torch.isinf(got), inf) and torch.equal(got[inf].double(), want[inf])
    # at most seven fp32 steps (the reciprocal, its product, frequency * c, two differences, the biases' sum and its
    # addition), and the output's own rounding
    tol = 7 * 2.0 ** -24 * size + half_step(torch, got.dtype) * (want.abs() + 7 * 2.0 ** -24 * size) + 2.0 ** -24
    bad = ~((got.double() - want).abs() <= tol) & ~inf
    assert not bad.any(), f"{int(bad.sum())} of {bad.numel()}"


def adjust_case(torch, B, V, L, N, dtype, seed, mask=True):
    g = torch.Generator(device="cuda").manual_seed(seed)
    r = lambda *s: torch.rand(*s, generator=g, device="cuda")  # noqa: E731
    x = (torch.randn(B, V, generator=g, device="cuda") * 3).to(dtype)
    tokens = (r(B, L) ** 2 * (V + 2)).int() - 1  # -1, V and V + 1 among them
    n_tokens = (r(B) * (L + 1)).int().clamp_max(L)
    n_prompt = (r(B) * (n_tokens + 3)).int() - 1
    rep, freq, pres = 0.5 + r(B) * 1.5, r(B) - 0.3, r(B) - 0.3
    words = (r(B, N) ** 2 * (V + 1)).int() - 1 if N else None  # equal entries among them
    bias = torch.randn(B, N, generator=g, device="cuda") * 4 if N else None
    allowed = torch.randint(-2 ** 31, 2 ** 31, (B, (V + 31) // 32 + 1), generator=g, device="cuda").int() if mask else None
    return x, tokens, n_tokens, n_prompt, rep, freq, pres, words, bias, allowed


@pytest.mark.parametrize("dtype", ["float32", "float16", "bfloat16"])
@pytest.mark.parametrize("B,V,L,N", [(1, 1, 1, 0), (3, 100, 50, 7), (2, 2049, 5000, 300), (5, 4096, 3, 1024), (1, 32000, 512, 8),
                                     (9, 130000, 700, 65), (40, 50004, 33, 5), (6, 262144, 1000, 100)])
def test_rows_adjust(cuda, dtype, B, V, L, N):
    torch = cuda
    for seed, mask in ((1, True), (2, False)):
        x, tokens, n_tokens, n_prompt, rep, freq, pres, words, bias, allowed = adjust_case(torch, B, V, L, N, getattr(torch, dtype),
                                                                                         seed, mask)
        before = x.clone()
        kw = dict(tokens=tokens, n_tokens=n_tokens, n_prompt=n_prompt, repetition=rep, frequency=freq, presence=pres,
                  bias_tokens=words, bias=bias, allowed=allowed)
        got = ops.rows_adjust(x, **kw)
        assert torch.equal(x, before) and got.dtype == x.dtype and got.is_contiguous()
        want, size = exact_adjust(torch, x, tokens, n_tokens, n_prompt, rep, freq, pres, words, bias, allowed)
        check_adjust(torch, got, want, size)
        assert ops.rows_adjust(x, out=x, **kw) is x  # in place: the same bits
        assert torch.equal(x, got)


@pytest.mark.parametrize("B,V", [(2, 1000), (60, 20003), (33, 40000), (90, 12289)])
def test_rows_adjust_parts_alone_strides_and_untouched_words(cuda, B, V):
    torch = cuda
    W = V // 4 * 4 + 16
    wide = torch.randn(B, W, device="cuda")
    for x, at in ((wide[:, 3:V + 3], 2), (wide[:, 8:V + 8], 4)):  # rows that are not aligned, and some that are
        out = torch.full((B, W), 7.0, device="cuda")
        assert torch.equal(ops.rows_adjust(x, out=out[:, at:V + at]), x)
        tokens = torch.randint(0, V, (B, 20), device="cuda").int()
        got = ops.rows_adjust(x, tokens=tokens, out=out[:, at:V + at])  # no penalty given: the words stay
        assert torch.equal(got, x) and (out[:, :at] == 7).all() and (out[:, V + at:] == 7).all()
        adjusted = lambda x=x, at=at, out=out, **kw: ops.rows_adjust(x, out=out[:, at:V + at], **kw)  # noqa: E731
        got = adjusted(tokens=tokens[:, :0], repetition=torch.full((B,), 2.0, device="cuda"))
        assert torch.equal(got, x)
        rep = torch.full((B,), 2.0, device="cuda")
        hit = torch.zeros(B, V, dtype=torch.bool, device="cuda").scatter_(1, tokens.long(), True)
        got = adjusted(tokens=tokens, repetition=rep)
        assert torch.equal(got, torch.where(hit, torch.where(x > 0, x / 2, x * 2), x))
        freq = torch.full((B,), 0.5, device="cuda")
        same = tokens[:, :1].expand(B, 20).contiguous()
        got = adjusted(tokens=same, frequency=freq, n_prompt=ints(torch, *[8] * B))
        want = x.clone().scatter_add_(1, same[:, :1].long(), torch.full((B, 1), -6.0, device="cuda"))
        assert torch.equal(got, want)
        bits = torch.zeros(B, (V + 31) // 32, dtype=torch.int32, device="cuda")
        assert torch.isneginf(adjusted(allowed=bits)).all()
        bits[:, 0] = 2
        got = adjusted(allowed=bits, bias_tokens=ints(torch, 1, 0).expand(B, 2).contiguous(),
                       bias=torch.ones(B, 2, device="cuda"))
        assert torch.equal(got[:, 1], x[:, 1] + 1) and torch.isneginf(got[:, 0]).all() and torch.isneginf(got[:, 2:]).all()


def test_rows_adjust_nan_infinities_and_long_counts(cuda):
    torch = cuda
    V = 5000
    x = torch.zeros(2, V, device="cuda")
    x[:, 0], x[:, 1], x[:, 2] = float("nan"), float("inf"), -float("inf")
    tokens = torch.zeros(2, 40000, dtype=torch.int32, device="cuda")
    tokens[:, 1:3] = torch.tensor([1, 2], device="cuda").int()
    tokens[:, 3:] = 4
    got = ops.rows_adjust(x, tokens=tokens, repetition=torch.full((2,), 1.5, device="cuda"),
                          frequency=torch.full((2,), 0.25, device="cuda"))
    assert torch.isnan(got[:, 0]).all() and torch.isposinf(got[:, 1]).all() and torch.isneginf(got[:, 2]).all()
    assert (got[:, 4] == -0.25 * 39997).all() and (got[:, 3] == 0).all() and (got[:, 5:] == 0).all()
    ops.rows_adjust(x, tokens=tokens, n_tokens=ints(torch, 40001, 5))
    assert ops.device_error() == native.DEVERR_DECODE_RANGE
    big = torch.zeros(300, V, device="cuda")
    many = torch.zeros(300, 4, dtype=torch.int32, device="cuda")
    n = torch.full((300,), 4, dtype=torch.int32, device="cuda")
    n[299] = -1
    ops.rows_adjust(big, tokens=many, n_tokens=n)
    assert ops.device_error() == native.DEVERR_DECODE_RANGE


# ------------------------------------------------------------------ refusals, streams, graphs
def test_refusals_of_the_python_layer(cuda):
    torch = cuda
    nh, nkv, hd = 4, 2, 128
    k, v, ks, vs, table = make_pages8(torch, [random8(torch, 40, nkv, hd, 0)], 16)
    n, cu = ints(torch, 40), ints(torch, 0, 1)
    x, rope = torch.zeros(1, (nh + 2 * nkv) * hd, device="cuda"), torch.zeros(64, hd // 2, 2, device="cuda")
    q = torch.zeros(1, nh, hd, dtype=torch.float16, device="cuda")
    kp, vp, t16 = make_pages(torch, [torch.zeros(40, nkv, hd).half()], [torch.zeros(40, nkv, hd).half()], 16)
    app = lambda **kw: ops.rope_append_q8(**{**dict(qkv=x, rope_cs=rope, kv_len=n, page_table=table, k_pages=k, v_pages=v,  # noqa: E731
                                                  k_scales=ks, v_scales=vs, n_heads=nh), **kw})
    rd = lambda **kw: ops.cache_read_q8(**{**dict(k_pages=k, v_pages=v, k_scales=ks, v_scales=vs, page_table=table, kv_len=n,  # noqa: E731
                                                cu=cu, rows=1), **kw})
    att = lambda **kw: ops.attention_paged_q8(**{**dict(q=q, k_pages=k, v_pages=v, k_scales=ks, v_scales=vs,  # noqa: E731
                                                      page_table=table, kv_len=n), **kw})
    sh = lambda **kw: ops.attention_shared(**{**dict(q=q, k_pages=kp, v_pages=vp, page_table=t16, kv_len=n, cu_group=cu,  # noqa: E731
                                                   shared_len=n), **kw})
    adj = lambda **kw: ops.rows_adjust(**{**dict(logits=torch.zeros(3, 50, device="cuda")), **kw})  # noqa: E731
    three = lambda d: torch.zeros(3, dtype=d, device="cuda")  # noqa: E731
    for err, call in [
        (TypeError, lambda: app(k_pages=k.float())), (TypeError, lambda: app(k_scales=ks.float())),
        (ValueError, lambda: app(v_pages=v[:1])), (ValueError, lambda: app(k_scales=ks.transpose(1, 2))),
        (ValueError, lambda: app(page_table=None)), (TypeError, lambda: app(page_table=table.long())),
        (TypeError, lambda: app(kv_len=n.long())), (ValueError, lambda: app(kv_len=ints(torch, 1, 2))),
        (ValueError, lambda: app(qkv=x[:, :-8])), (TypeError, lambda: app(qkv=x.double())),
        (TypeError, lambda: app(qkv=x.half(), q_dtype=torch.bfloat16)), (TypeError, lambda: app(q_dtype=torch.float32)),
        (ValueError, lambda: app(rope_cs=rope[:, :3])), (TypeError, lambda: app(rope_cs=rope.half())),
        (ValueError, lambda: app(q_out=q[:, :2].contiguous())), (TypeError, lambda: app(q_out=q, q_dtype=torch.bfloat16)),
        (ValueError, lambda: app(qkv=torch.zeros(2, x.shape[1], device="cuda"))),
        (TypeError, lambda: app(k_pages=k.cpu(), v_pages=v.cpu())), (TypeError, lambda: app(kv_len=n.cpu())),
        (ops.AsmError, lambda: app(v_pages=k, v_scales=ks)),
        (TypeError, lambda: rd(dtype=torch.float32)), (ValueError, lambda: rd(rows=-1)), (ValueError, lambda: rd(cu=n)),
        (ValueError, lambda: rd(out=(q, q))), (TypeError, lambda: rd(out=(x, x), dtype=torch.float16)),
        (ops.AsmError, lambda: rd(out=[torch.zeros(1, nkv, hd, dtype=torch.float16, device="cuda")] * 2)),
        (TypeError, lambda: att(q=q.float())), (ValueError, lambda: att(q=q[:, :3])), (ValueError, lambda: att(q=q[..., :64])),
        (TypeError, lambda: att(out_dtype=torch.bfloat16)), (ValueError, lambda: att(out=q[:, :2])),
        (ops.AsmError, lambda: att(scale=-1.0)), (ops.AsmError, lambda: att(workspace=torch.zeros(16, dtype=torch.uint8, device="cuda"))),
        (TypeError, lambda: att(workspace=x)), (ops.AsmError, lambda: att(out=q)),
        (TypeError, lambda: sh(q=q.bfloat16())), (ValueError, lambda: sh(cu_group=ints(torch, 0, 1, 1))),
        (TypeError, lambda: sh(shared_len=n.long())), (ValueError, lambda: sh(shared_len=n.view(1, 1))),
        (ValueError, lambda: sh(q=torch.cat([q, q]))), (ValueError, lambda: sh(v_pages=vp[:1])), (ops.AsmError, lambda: sh(out=q)),
        (ops.AsmError, lambda: sh(workspace=torch.zeros(16, dtype=torch.uint8, device="cuda"))),
        (TypeError, lambda: sh(kv_len=n.cpu())),
        (TypeError, lambda: adj(logits=torch.zeros(3, 50, device="cuda").double())),
        (TypeError, lambda: adj(tokens=torch.zeros(3, 4, device="cuda"))), (ValueError, lambda: adj(repetition=three(torch.float32))),
        (TypeError, lambda: adj(tokens=torch.zeros(3, 4, device="cuda").int(), repetition=three(torch.float64))),
        (ValueError, lambda: adj(tokens=torch.zeros(2, 4, device="cuda").int())),
        (ValueError, lambda: adj(bias=torch.zeros(3, 2, device="cuda"))),
        (ValueError, lambda: adj(bias=torch.zeros(3, 2, device="cuda"), bias_tokens=torch.zeros(3, 3, device="cuda").int())),
        (ValueError, lambda: adj(allowed=torch.zeros(3, 1, device="cuda").int())), (ValueError, lambda: adj(out=torch.zeros(3, 49, device="cuda"))),
        (TypeError, lambda: adj(out=torch.zeros(3, 50, device="cuda").half())),
        (ops.AsmError, lambda: adj(bias=torch.zeros(3, 1025, device="cuda"), bias_tokens=torch.zeros(3, 1025, device="cuda").int())),
        (TypeError, lambda: adj(allowed=torch.zeros(3, 2).int())),
    ]:
        with pytest.raises(err):
            call()
    # outputs over inputs
    both = torch.zeros(3, 100, device="cuda")
    with pytest.raises(ops.AsmError, match="overlaps"):
        ops.rows_adjust(both[:, :50], out=both[:, 25:75])
    assert ops.rows_adjust(both[:, :50], out=both[:, 50:]).shape == (3, 50)
    bits = torch.zeros(3, 50, device="cuda")
    with pytest.raises(ops.AsmError, match="overlaps"):
        ops.rows_adjust(torch.zeros(3, 50, device="cuda"), allowed=bits.view(torch.int32)[:, :2], out=bits)
    for need, call in ((ops.attention_paged_q8_workspace(1, nh, nkv, hd), att), (ops.attention_shared_workspace(1, 1, nh, nkv, hd), sh)):
        buf = torch.zeros(need + 1024, dtype=torch.uint8, device="cuda")
        inside = buf[need - 256:need - 256 + q.numel() * 2].view(torch.float16).view(q.shape)  # begins in the workspace
        with pytest.raises(ops.AsmError, match="overlaps"):
            call(q=inside, workspace=buf[:need])
    # without rows
    assert ops.rows_adjust(torch.zeros(0, 50, device="cuda")).shape == (0, 50)
    assert att(q=q[:0], page_table=table[:0], kv_len=n[:0]).shape == (0, nh, hd)
    assert sh(q=q[:0], page_table=t16[:0], kv_len=n[:0], cu_group=cu[:1], shared_len=n[:0]).shape == (0, nh, hd)
    assert app(qkv=x[:0], page_table=table[:0], kv_len=n[:0]).shape == (0, nh, hd)
    assert rd(rows=0, cu=ints(torch, 0, 0))[0].shape == (0, nkv, hd)


def serving_state(torch, seed):
    nh, nkv, hd, B = 8, 2, 128, 3
    dense = [random8(torch, n, nkv, hd, seed + n) for n in (40, 70, 200)]
    k, v, ks, vs, table = make_pages8(torch, dense, 16)
    dk, dv, kp, vp, t16 = shared_case(torch, [(B, 96)], [5, 9, 30], nkv, hd, torch.float16, 16, seed=seed)
    return dict(q=rand(torch, B, nh, hd, dt=torch.float16, seed=seed), q8=(k, v, ks, vs), table=table, lens=ints(torch, 40, 70, 200),
                kp=kp, vp=vp, t16=t16, kv=ints(torch, 101, 105, 126), cu=ints(torch, 0, B), shared=ints(torch, 96),
                qkv=rand(torch, B, (nh + 2 * nkv) * hd, dt=torch.float32, seed=seed + 1), nh=nh,
                rope=torch.from_numpy(D.rope_table(256, hd, 10000.0)).cuda(),
                logits=torch.randn(B, 9000, generator=torch.Generator(device="cuda").manual_seed(seed), device="cuda"),
                tokens=torch.randint(0, 9000, (B, 60), generator=torch.Generator(device="cuda").manual_seed(seed), device="cuda").int(),
                rep=torch.full((B,), 1.3, device="cuda"))


def serving_step(st, stream=None):
    q = ops.rope_append_q8(st["qkv"], st["rope"], st["lens"], st["table"], *st["q8"], st["nh"], stream=stream)
    a = ops.attention_paged_q8(q, *st["q8"], st["table"], st["lens"], out_dtype=None, stream=stream)
    k, v = ops.cache_read_q8(*st["q8"], st["table"], st["lens"], st["cu_read"], 310, stream=stream)
    b = ops.attention_shared(st["q"], st["kp"], st["vp"], st["t16"], st["kv"], st["cu"], st["shared"], stream=stream)
    c = ops.rows_adjust(st["logits"], tokens=st["tokens"], repetition=st["rep"], stream=stream)
    return q, a, k, v, b, c


def test_two_streams_and_graph_replay_with_other_contents(cuda):
    torch = cuda
    states = [serving_state(torch, s) for s in (10, 20)]
    for st in states:
        st["cu_read"] = ints(torch, 0, 40, 110, 310)
    want = [[t.clone() for t in serving_step(st)] for st in states]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in states]
    for _ in range(10):
        got = [serving_step(st, stream) for st, stream in zip(states, streams)]
        torch.cuda.synchronize()
        for w, g in zip(want, got):
            assert all(torch.equal(a, b) for a, b in zip(w, g))
    # captured on the first state's tensors, replayed with the second's contents and shorter lengths
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = serving_step(states[0])
    graph.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(out, want[0]))
    states[1]["shared"].fill_(32)
    states[1]["kv"].copy_(ints(torch, 101, 0, 40))
    states[1]["lens"].copy_(ints(torch, 1, 70, 33))
    states[1]["cu_read"].copy_(ints(torch, 0, 1, 71, 104))
    want = [t.clone() for t in serving_step(states[1])]
    for name, t in states[1].items():
        if name == "q8":
            for a, b in zip(states[0]["q8"], t):
                a.copy_(b)
        elif torch.is_tensor(t):
            states[0][name].copy_(t)
    graph.replay()
    torch.cuda.synchronize()
    for i, (a, b) in enumerate(zip(out, want)):
        if i in (2, 3):
            a, b = a[:104], b[:104]
        assert torch.equal(a, b)


# ------------------------------------------------------------------ together
def test_prompts_then_decode_on_a_q8_cache_with_a_shared_prefix(cuda):
    """Two chunks of prompts into a Q8_0 cache (read back for their attention), then decode steps over it; the same
    sequences, sharing their first pages, over a 16-bit cache; logits adjusted and sampled.  Against 64 bits on what the
    caches hold."""
    torch = cuda
    nh, nkv, hd, page, P = 8, 2, 128, 16, 64
    rope = torch.from_numpy(D.rope_table(256, hd, 10000.0)).cuda()
    chunks = [[40, 64, 3], [24, 9, 70]]
    B, total = 3, [64, 73, 73]
    k, v, ks, vs, table = make_pages8(torch, [random8(torch, 120, nkv, hd, s) for s in range(B)], page, fill=False)
    lens = [0] * B
    for c, rows in enumerate(chunks):
        lens = [a + b for a, b in zip(lens, rows)]
        cu, kv = ints(torch, *np.concatenate([[0], np.cumsum(rows)]).tolist()), ints(torch, *lens)
        cu_k = ints(torch, *np.concatenate([[0], np.cumsum(lens)]).tolist())
        qkv = rand(torch, sum(rows), (nh + 2 * nkv) * hd, dt=torch.float32, seed=c)
        q = ops.rope_append_q8(qkv, rope, kv, table, k, v, ks, vs, nh, cu_q=cu)
        kr, vr = ops.cache_read_q8(k, v, ks, vs, table, kv, cu_k, sum(lens))
        a = ops.attention_prompt(q, kr, vr, cu, cu_k=cu_k, out_dtype=torch.float32)
        for s in range(B):
            lo, hi = int(cu_k[s]), int(cu_k[s + 1])
            qs = q[int(cu[s]):int(cu[s + 1])]
            want, pv, serr = exact_attention(torch, qs, kr[lo:hi], vr[lo:hi], hd ** -0.5, lens[s] - rows[s])
            close(torch, a[int(cu[s]):int(cu[s + 1])], want, pv, serr, lens[s], 2 * 2.0 ** -22 + lens[s] * 2.0 ** -32, torch.float16)
    assert lens == total
    logits = rand(torch, B, 5000, dt=torch.float32, seed=9, scale=3.0)
    history = torch.full((B, 8), -1, dtype=torch.int32, device="cuda")
    for step in range(3):
        lens = [n + 1 for n in lens]
        kv = ints(torch, *lens)
        q = ops.rope_append_q8(rand(torch, B, (nh + 2 * nkv) * hd, dt=torch.float32, seed=50 + step), rope, kv, table, k, v, ks, vs, nh)
        a = ops.attention_paged_q8(q, k, v, ks, vs, table, kv, out_dtype=torch.float32)
        cu_k = ints(torch, *np.concatenate([[0], np.cumsum(lens)]).tolist())
        codes = [(pages[table[s].clamp_min(0).long()].flatten(0, 1)[:lens[s]],
                  scales[table[s].clamp_min(0).long()].transpose(1, 2).flatten(0, 1)[:lens[s]])
                 for s in range(B) for pages, scales in ((k, ks), (v, vs))]
        for s in range(B):
            want, pv, serr = exact_attention(torch, q[s:s + 1], values(*codes[2 * s]), values(*codes[2 * s + 1]), hd ** -0.5,
                                             lens[s] - 1)
            close8(torch, a[s:s + 1], want, pv, serr, lens[s])
        # a word that has been chosen is never chosen again
        y = ops.rows_adjust(logits, tokens=history, presence=torch.full((B,), 1e4, device="cuda"))
        word = ops.rows_sample(y, torch.full((B,), 0.5, device="cuda"), top_k=ints(torch, *[1] * B))
        assert torch.equal(word.long(), y.argmax(-1)) and not (history == word[:, None]).any()
        history[:, step] = word
    # the same decode over a 16-bit cache whose first pages are shared
    dense_k, dense_v, kp, vp, t16 = shared_case(torch, [(B, P)], [5, 9, 40], nkv, hd, torch.float16, page)
    kv = ints(torch, *[x.shape[0] for x in dense_k])
    q = rand(torch, B, nh, hd, dt=torch.float16, seed=3)
    one = ops.attention_shared(q, kp, vp, t16, kv, ints(torch, 0, B), ints(torch, P), out_dtype=torch.float32)
    two = ops.attention_paged(q, kp, vp, t16, kv, out_dtype=torch.float32)
    assert float((one - two).abs().max()) <= 1e-5 * float(two.abs().max())
    check_shared(torch, one, q, dense_k, dense_v, hd ** -0.5, torch.float16)
