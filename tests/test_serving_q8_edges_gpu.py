"""The serving operators around the Q8_0 cache where their kernels' layouts have edges: several rows to a CTA, blocks of
every size, outputs on 16 bytes, strides past 32 bits.  Helpers and tolerances are test_serving_q8_gpu.py's."""
from __future__ import annotations

import numpy as np
import pytest

from asmllm_b200 import decode as D
from asmllm_b200 import native, ops
from test_serving_gpu import rand
from test_serving_q8_gpu import (blocks, check_adjust, check_shared, clean_error_word, close8, exact_adjust,  # noqa: F401
                                 exact_attention, ints, make_pages8, random8, values)

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("nh,nkv,hd", [(6, 2, 64), (7, 1, 128), (32, 32, 128)])
def test_append_of_thousands_of_rows_and_read_back(cuda, nh, nkv, hd):
    torch = cuda
    q_len, kv_len, tail, page = [2001, 0, 1, 400, 99], [2100, 7, 1, 390, 99], 7, 16  # the fourth: ten rows before its start
    T = sum(q_len)
    cu = np.concatenate([[0], np.cumsum(q_len)]).tolist()
    x = rand(torch, T + tail, (nh + 2 * nkv) * hd, dt=torch.float32, seed=1)
    rope = torch.from_numpy(D.rope_table(2200, hd, 10000.0)).cuda()
    dense = [random8(torch, n, nkv, hd, n) for n in kv_len]
    k, v, ks, vs, table = make_pages8(torch, dense, page)
    bad = int(table[0, 100])  # positions 1600 .. 1615 of the first sequence
    table[0, 100] = 10 ** 6
    before = [t.clone() for t in (k, v, ks, vs)]
    q_out = torch.full((T + tail, nh, hd), 77.0, dtype=torch.float16, device="cuda")
    ops.rope_append_q8(x, rope, ints(torch, *kv_len), table, k, v, ks, vs, nh, cu_q=ints(torch, *cu), q_out=q_out)
    assert ops.device_error() == native.DEVERR_DECODE_RANGE

    pos = torch.cat([torch.arange(n) + m - n for n, m in zip(q_len, kv_len)]).cuda()
    seq = torch.repeat_interleave(torch.arange(5), torch.tensor(q_len)).cuda()
    live = (pos >= 0) & ~((seq == 0) & (pos // page == 100))
    cs = rope.view(2200, hd // 2, 2)[pos.clamp_min(0)][:, None]
    h = x[:T].view(T, nh + 2 * nkv, hd // 2, 2)
    a, b, c, s = h[:, :nh + nkv, :, 0], h[:, :nh + nkv, :, 1], cs[..., 0], cs[..., 1]
    turned = torch.stack([a * c - b * s, a * s + b * c], -1).flatten(-2)  # torch rounds each step
    want_q = torch.where(live[:, None, None], turned[:, :nh], 0.0).half()
    assert torch.equal(q_out[:T], want_q) and (q_out[T:] == 77).all()
    codes, d = ops.quantize_q8_0_dev(torch.cat([turned[:, nh:], h[:, nh + nkv:].flatten(-2)], 1).reshape(T, -1).contiguous())
    codes, d = codes.view(T, 2, nkv, hd)[live], d.half().view(T, 2, nkv, hd // 32)[live]
    pg, at = table[seq[live], (pos[live] // page)].long(), pos[live] % page
    for i, (pages, scales, old, old_d) in enumerate(((k, ks, before[0], before[2]), (v, vs, before[1], before[3]))):
        old[pg, at], old_d[pg, :, at] = codes[:, i], d[:, i]
        assert torch.equal(pages, old) and torch.equal(scales.view(torch.int16), old_d.view(torch.int16))

    table[0, 100] = bad
    for dt in (torch.float16, torch.bfloat16):
        read = ops.cache_read_q8(k, v, ks, vs, table, ints(torch, *kv_len), ints(torch, *cu), T, dtype=dt)
        for i, y in enumerate(read):
            assert torch.equal(y[live], values(codes[:, i], d[:, i]).to(dt))
            assert (y[pos < 0] == 0).all()


def test_append_blocks_of_every_size(cuda):
    torch = cuda
    nkv, hd, B = 2, 64, 130
    g = torch.Generator().manual_seed(3)
    size = torch.exp2(torch.linspace(-149, 127.9, B * 2 * nkv * 2).double())[torch.randperm(B * 2 * nkv * 2, generator=g)]
    x = (torch.rand(B, 2 * nkv * 2, 32, generator=g).double() * 2 - 1) * size.view(B, -1, 1)
    x[::7, 0, 3:] = 0.0  # one value other than zero, or none
    x[::9, 2] = 0.0
    kv = x.float().flatten(1).cuda()
    kv[3, 40], kv[4, 70], kv[5, 100] = float("inf"), float("-inf"), float("nan")
    rope = torch.zeros(64, hd // 2, 2, device="cuda")
    rope[..., 0] = 1.0
    k, v, ks, vs, table = make_pages8(torch, [random8(torch, 20, nkv, hd, s) for s in range(B)], 16)
    row = torch.cat([torch.ones(B, nkv * hd, device="cuda"), kv], 1)
    ops.rope_append_q8(row, rope, ints(torch, *[20] * B), table, k, v, ks, vs, nkv)
    with np.errstate(all="ignore"):  # the rotation by nothing: x0 - 0 x1, 0 x0 + x1
        h = kv.cpu().numpy().reshape(B, 2 * nkv, hd)
        turned = h.copy()
        turned[:, :nkv, 0::2] = h[:, :nkv, 0::2] - h[:, :nkv, 1::2] * np.float32(0)
        turned[:, :nkv, 1::2] = h[:, :nkv, 0::2] * np.float32(0) + h[:, :nkv, 1::2]
        codes, d = blocks(turned)
    pg = table[:, 1].long()
    got = torch.cat([k[pg, 3], v[pg, 3]], 1).cpu().numpy()
    scale = torch.cat([ks[pg, :, 3], vs[pg, :, 3]], 1).cpu().numpy()
    assert np.array_equal(got, codes)
    nan = np.isnan(d)
    assert nan.any() and np.array_equal(np.isnan(scale), nan)
    assert np.array_equal(scale[~nan].view(np.uint16), d[~nan].view(np.uint16))


@pytest.mark.parametrize("dtype", ["float16", "bfloat16"])
@pytest.mark.parametrize("nkv,hd", [(1, 64), (3, 128), (5, 64)])
def test_cache_read_outputs_on_16_bytes(cuda, dtype, nkv, hd):
    torch = cuda
    dt, n = getattr(torch, dtype), 61
    dense = random8(torch, n, nkv, hd, 3, spread=3.0)
    dense[0][7, 0, :4] = ints(torch, -128, 127, 0, -1).to(torch.int8)
    dense[1][7, 0, 0] = 6e-8  # the smallest scale: products that are not normal numbers
    k, v, ks, vs, table = make_pages8(torch, [dense], 16)
    out = [torch.full((n * nkv * hd + 16,), 7.0, dtype=dt, device="cuda") for _ in "kv"]
    y = [t[8:-8].view(n, nkv, hd) for t in out]
    ops.cache_read_q8(k, v, ks, vs, table, ints(torch, n), ints(torch, 0, n), n, out=y)
    for i in (0, 1):
        assert torch.equal(y[i], values(*dense[2 * i:2 * i + 2]).to(dt))
        assert (out[i][:8] == 7).all() and (out[i][-8:] == 7).all()


def far(torch, shape, stride, dtype):
    """A view whose first axis has a stride past 2^31 elements (not filled)."""
    size = sum((n - 1) * s for n, s in zip(shape, stride)) + 1
    return torch.empty(size, dtype=dtype, device="cuda").as_strided(shape, stride)


def test_q8_pages_more_than_2_31_apart(cuda):
    torch = cuda
    nh, nkv, hd, page, n = 4, 2, 128, 16, 29
    step, scale_step = 2 ** 31 + 4096, 2 ** 31 + 64
    k, v = (far(torch, (2, page, nkv, hd), (step, nkv * hd, hd, 1), torch.int8) for _ in "kv")
    ks, vs = (far(torch, (2, nkv, page, hd // 32), (scale_step, page * 4, 4, 1), torch.float16) for _ in "kv")
    table = ints(torch, 1, 0).view(1, 2)  # the first positions in the far page
    x = rand(torch, n, (nh + 2 * nkv) * hd, dt=torch.float16, seed=1)
    rope = torch.zeros(64, hd // 2, 2, device="cuda")
    rope[..., 0] = 1.0
    q = ops.rope_append_q8(x, rope, ints(torch, n), table, k, v, ks, vs, nh, cu_q=ints(torch, 0, n))
    codes, d = ops.quantize_q8_0_dev(x[:, nh * hd:].float().contiguous())
    codes, d = codes.view(n, 2, nkv, hd), d.half().view(n, 2, nkv, hd // 32)
    read = ops.cache_read_q8(k, v, ks, vs, table, ints(torch, n), ints(torch, 0, n), n)
    for i in (0, 1):
        assert torch.equal(read[i], values(codes[:, i], d[:, i]).to(read[i].dtype))
    got = ops.attention_paged_q8(q[-1:], k, v, ks, vs, table, ints(torch, n), out_dtype=torch.float32)
    want, pv, serr = exact_attention(torch, q[-1:], values(codes[:, 0], d[:, 0]), values(codes[:, 1], d[:, 1]), hd ** -0.5, n - 1)
    close8(torch, got, want, pv, serr, n)


def test_shared_pages_more_than_2_31_apart(cuda):
    torch = cuda
    nh, nkv, hd, page = 8, 1, 128, 16
    k, v = (far(torch, (3, page, nkv, hd), (2 ** 30 + 64, nkv * hd, hd, 1), torch.float16) for _ in "kv")
    own = rand(torch, 3, page, nkv, hd, dt=torch.float16, seed=2), rand(torch, 3, page, nkv, hd, dt=torch.float16, seed=3)
    k.copy_(own[0])
    v.copy_(own[1])
    table = ints(torch, 2, 0, 2, 1).view(2, 2)  # the shared page lies past 2^31 elements
    q = rand(torch, 2, nh, hd, dt=torch.float16, seed=4)
    got = ops.attention_shared(q, k, v, table, ints(torch, 20, 31), ints(torch, 0, 2), ints(torch, 16), out_dtype=torch.float32)
    dense = [[torch.cat([t[2], t[0, :4]]), torch.cat([t[2], t[1, :15]])] for t in own]
    check_shared(torch, got, q, dense[0], dense[1], hd ** -0.5, torch.float16)


@pytest.mark.parametrize("B,V", [(2, 5000), (40, 32768)])
def test_logits_rows_more_than_2_31_apart(cuda, B, V):
    torch = cuda
    step = (2 ** 31 // (B - 1) + 64) // 8 * 8
    x = far(torch, (B, V), (step, 1), torch.float16)
    x.copy_(rand(torch, B, V, dt=torch.float16, seed=5))
    tokens = ((torch.rand(B, 50, generator=torch.Generator().manual_seed(6)) * V).int()).cuda()
    ones = torch.ones(B, device="cuda")
    want, size = exact_adjust(torch, x, tokens, [50] * B, [10] * B, 1.5 * ones, 0.5 * ones, 0.25 * ones, None, None, None)
    ops.rows_adjust(x, tokens=tokens, n_prompt=ints(torch, *[10] * B), repetition=1.5 * ones, frequency=0.5 * ones,
                    presence=0.25 * ones, out=x)
    check_adjust(torch, x, want, size)


def test_shared_groups_that_begin_with_padding(cuda):
    """Slots without a sequence, and short ones, before those that hold the prefix: their tables are not read for it."""
    torch = cuda
    nh, nkv, hd, page = 8, 2, 128, 16
    k, v = (rand(torch, 40, page, nkv, hd, dt=torch.float16, seed=s) for s in (2, 3))
    for empty in (1, 31, 32, 40, 70):
        B = empty + 3
        table = torch.full((B + 2, 6), -7, dtype=torch.int32)
        table[empty:B, :4] = torch.tensor([30, 4, 17, 9])
        table[empty:B, 4] = torch.tensor([5, 6, 7])
        table[0, 0] = 39
        table[B:, :2] = torch.tensor([[1, 2], [3, 8]])
        lens = [9] + [0] * (empty - 1) + [64, 70, 80, 20, 32]  # the last two: a group whose prefix neither holds
        table = table.cuda()
        q = rand(torch, B + 2, nh, hd, dt=torch.float16, seed=4)
        for odt in (torch.float16, torch.float32):
            got = ops.attention_shared(q, k, v, table, ints(torch, *lens), ints(torch, 0, B, B + 2), ints(torch, 64, 48),
                                       out_dtype=odt)
            assert ops.device_error() == 0
            dense = [[t[table[s].clamp_min(0).long()].flatten(0, 1)[:lens[s]] for s in range(B + 2)] for t in (k, v)]
            some = [0, *range(empty, B + 2)]
            assert (got[1:empty] == 0).all()
            check_shared(torch, got[some], q[some], [dense[0][s] for s in some], [dense[1][s] for s in some], hd ** -0.5,
                         torch.float16)
