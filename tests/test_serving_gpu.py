"""The serving operators on the GPU (ops.rope_append, attention_prompt, attention_paged, rows_sample)
against plain implementations in 64 bits.

Tolerances count roundings.  u = eps/2 of the 16-bit type, u32 = 2^-24.
  * A score is a sum of hd exact products in fp32: off by at most hd * 2^-23 * sum|q||k| * scale (the
    tensor core truncates), and its scaled copy by 2^-22 of its size; the weight exp(s - m) follows
    with twice that (its own and the maximum's), and 2^-22 of the exponential itself.
  * Prompt: each weight is rounded once to 16 bits (u); paged: to twice 16 bits (2 u^2, and 2^-38 of the
    largest weight where fp16 runs out of exponent).
  * Sums of n terms in fp32, in chains of at most n: n * 2^-23 at most (it is far less).
  * The output is rounded once (u of its type).
So |out - exact| <= A * sum_j p_j |v_j| + u_out |exact|, A collecting the relative errors of the weights
(twice: in the weighted sum and in the sum of weights)."""
from __future__ import annotations

import math

import numpy as np
import pytest

from asmllm_b200 import decode as D
from asmllm_b200 import native, ops
from test_serving_host import WEIGHT_CASES, one_value_case, one_value_exact

pytestmark = pytest.mark.gpu

DTYPES = ["float16", "bfloat16"]


def half_step(torch, dt):
    return torch.finfo(dt).eps / 2


@pytest.fixture(autouse=True)
def clean_error_word(cuda):
    ops.device_error()
    yield
    assert ops.device_error() == 0


# ------------------------------------------------------------------ helpers
def make_pages(torch, dense_k, dense_v, page, layout="token", extra=3, seed=0, width_extra=2):
    """Pages (NaN wherever no position lives) of per-sequence keys and values [n, nkv, hd]."""
    nkv, hd, dt = dense_k[0].shape[1], dense_k[0].shape[2], dense_k[0].dtype
    need = [-(-k.shape[0] // page) for k in dense_k]
    total = sum(need) + extra
    g = torch.Generator().manual_seed(seed)
    perm = torch.randperm(total, generator=g).tolist()
    if layout == "token":  # [page][offset][head][hd]
        mk = lambda: torch.full((total, page, nkv, hd), float("nan"), dtype=dt, device="cuda")  # noqa: E731
    elif layout == "head":  # [page][head][offset][hd]
        mk = lambda: torch.full((total, nkv, page, hd), float("nan"), dtype=dt,  # noqa: E731
                                device="cuda").transpose(1, 2)
    else:  # keys and values side by side in one pool, heads padded
        mk = lambda: torch.full((total, page, nkv, hd + 16), float("nan"), dtype=dt,  # noqa: E731
                                device="cuda")[..., :hd]
    kp, vp = mk(), mk()
    table = torch.full((len(need), max(need + [1]) + width_extra), -7, dtype=torch.int32)  # not to be read
    at = 0
    for s, n in enumerate(need):
        for i in range(n):
            pg = perm[at]
            at += 1
            table[s, i] = pg
            rows = dense_k[s][i * page:(i + 1) * page]
            kp[pg, :rows.shape[0]] = rows
            vp[pg, :rows.shape[0]] = dense_v[s][i * page:(i + 1) * page]
    return kp, vp, table.cuda()


def exact_attention(torch, q, k, v, scale, first):
    """64-bit causal attention of q [n, nh, hd] whose row i sees keys 0 .. first + i; also sum p|v| and A's score part."""
    n, nh, hd = q.shape
    m, nkv = k.shape[0], k.shape[1]
    g = nh // nkv
    out = torch.zeros(n, nh, hd, dtype=torch.float64, device="cuda")
    pv = torch.zeros_like(out)
    serr = torch.zeros(n, nh, 1, dtype=torch.float64, device="cuda")
    if m == 0:
        return out, pv, serr
    keep = torch.arange(m, device="cuda")[None] <= (first + torch.arange(n, device="cuda"))[:, None]
    for h in range(nh):
        Q, K, V = q[:, h].double(), k[:, h // g].double(), v[:, h // g].double()
        s = (Q @ K.T * scale).masked_fill(~keep, -math.inf)
        mx = s.amax(-1, keepdim=True)
        mx = torch.where(torch.isinf(mx), torch.zeros_like(mx), mx)
        p = torch.exp(s - mx)
        l = p.sum(-1, keepdim=True)
        p = p / torch.where(l == 0, torch.ones_like(l), l)
        out[:, h] = p @ V
        pv[:, h] = p @ V.abs()
        mag = (Q.abs() @ K.abs().T * scale).masked_fill(~keep, 0)
        serr[:, h, 0] = (mag.amax(-1) * hd * 2.0 ** -23 + s.masked_fill(~keep, 0).abs().amax(-1) * 2.0 ** -22)
    return out, pv, serr


def close(torch, got, want, pv, serr, n, weight, dt, what=""):
    A = 2 * (2 * serr + 2.0 ** -22 + weight + n * 2.0 ** -23)
    u = half_step(torch, got.dtype)
    tiny = 2.0 ** -24 if got.dtype == torch.float16 else 0.0  # fp16 subnormal steps
    tol = A * pv + u * (want.abs() + A * pv) + tiny
    err = (got.double() - want).abs()
    bad = ~(err <= tol)
    assert not bad.any(), f"{what}: {int(bad.sum())} of {bad.numel()} outside, worst {float((err / tol).max()):.3g} of it"


def paged_weight(torch, dt, n):
    u = half_step(torch, dt)
    return 2 * u * u + (n * 2.0 ** -38 if dt == torch.float16 else 0.0)


def prompt_weight(torch, dt, n):
    return half_step(torch, dt) + (n * 2.0 ** -32 if dt == torch.float16 else 0.0)


def rand(torch, *shape, dt, seed, scale=1.0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return (torch.randn(*shape, generator=g, device="cuda") * scale).to(dt)


# ------------------------------------------------------------------ rotary and append
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("src", ["float32", "same"])
@pytest.mark.parametrize("nh,nkv,hd", [(4, 2, 128), (5, 1, 64), (32, 32, 128)])
@pytest.mark.parametrize("page,layout", [(16, "token"), (64, "head"), (256, "padded")])
def test_rope_append(cuda, dtype, src, nh, nkv, hd, page, layout):
    torch = cuda
    dt = getattr(torch, dtype)
    q_len, kv_len = [3, 1, 0, 40, 5], [3, 17, 9, 300, 2]  # the last has more rows than positions
    T, tail = sum(q_len), 4
    x = rand(torch, T + tail, (nh + 2 * nkv) * hd, dt=torch.float32 if src == "float32" else dt, seed=1)
    rope = torch.from_numpy(D.rope_table(512, hd, 10000.0)).cuda()
    empty = [torch.full((n, nkv, hd), float("nan"), dtype=dt, device="cuda") for n in kv_len]
    kp, vp, table = make_pages(torch, empty, empty, page, layout)
    cu = torch.tensor(np.concatenate([[0], np.cumsum(q_len)]), dtype=torch.int32, device="cuda")
    kv = torch.tensor(kv_len, dtype=torch.int32, device="cuda")
    q_out = torch.full((T + tail, nh, hd), 77.0, dtype=dt, device="cuda")
    before = (kp.clone(), vp.clone())
    ops.rope_append(x, rope, kv, table, kp, vp, nh, cu_q=cu, q_out=q_out)
    torch.cuda.synchronize()
    assert (q_out[T:] == 77.0).all()  # rows behind the last sequence
    xs = x.float().view(T + tail, nh + 2 * nkv, hd)
    want_k, want_v = before
    t = 0
    for s, (n, m) in enumerate(zip(q_len, kv_len)):
        for i in range(n):
            p = m - n + i
            if p < 0:
                assert (q_out[t] == 0).all()
            else:
                c, d = rope[p, :, 0], rope[p, :, 1]
                z = xs[t, :nh + nkv].unflatten(-1, (hd // 2, 2))
                # the same fp32 roundings, one by one; then one to 16 bits
                z = torch.stack([z[..., 0] * c - z[..., 1] * d, z[..., 0] * d + z[..., 1] * c], -1).flatten(-2).to(dt)
                assert torch.equal(q_out[t], z[:nh])
                pg = int(table[s, p // page])
                want_k[pg, p % page] = z[nh:]
                want_v[pg, p % page] = xs[t, nh + nkv:].to(dt)
            t += 1
    same = lambda a, b: torch.equal(torch.nan_to_num(a.float(), nan=123.0), torch.nan_to_num(b.float(), nan=123.0))  # noqa: E731
    assert same(kp, want_k) and same(vp, want_v)


def test_rope_append_one_row_per_sequence_and_strided_input(cuda):
    torch = cuda
    B, nh, nkv, hd = 7, 8, 2, 128
    big = rand(torch, B, (nh + 2 * nkv) * hd + 64, dt=torch.float32, seed=2)
    x = big[:, :(nh + 2 * nkv) * hd]
    rope = torch.from_numpy(D.rope_table(128, hd, 10000.0)).cuda()
    kv_len = [1, 16, 17, 100, 33, 0, 128]  # no position: nothing to write
    empty = [torch.zeros(n, nkv, hd, dtype=torch.float16, device="cuda") for n in kv_len]
    kp, vp, table = make_pages(torch, empty, empty, 16)
    kv = torch.tensor(kv_len, dtype=torch.int32, device="cuda")
    a = ops.rope_append(x, rope, kv, table, kp, vp, nh)
    b = ops.rope_append(x.contiguous(), rope, kv, table, kp.clone(), vp.clone(), nh,
                        cu_q=torch.arange(B + 1, dtype=torch.int32, device="cuda"))
    torch.cuda.synchronize()
    assert torch.equal(a, b)
    assert (a[5] == 0).all() and not (a[4] == 0).all()


def test_rope_append_refuses_positions_and_pages_on_the_device(cuda):
    torch = cuda
    nh, nkv, hd = 4, 2, 128
    x = rand(torch, 4, (nh + 2 * nkv) * hd, dt=torch.float32, seed=3)
    rope = torch.from_numpy(D.rope_table(32, hd, 10000.0)).cuda()
    kp = torch.zeros(4, 16, nkv, hd, dtype=torch.float16, device="cuda")
    vp = torch.zeros_like(kp)
    table = torch.tensor([[0, 1, 9], [9, 1, 2], [2, -1, 3], [3, 1, 2]], dtype=torch.int32, device="cuda")
    # past the rotary table; page 9 of 4; page -1; past the table's width
    kv = torch.tensor([40, 4, 20, 49], dtype=torch.int32, device="cuda")
    q = ops.rope_append(x, rope, kv, table, kp, vp, nh)
    assert ops.device_error() == native.DEVERR_DECODE_RANGE
    assert (q == 0).all() and (kp == 0).all() and (vp == 0).all()


def test_rope_append_reports_lengths_and_offsets_no_row_meets(cuda):
    torch = cuda
    nh, nkv, hd, B = 2, 1, 64, 300  # more sequences than a CTA has threads
    x = rand(torch, B, (nh + 2 * nkv) * hd, dt=torch.float32, seed=3)
    rope = torch.from_numpy(D.rope_table(32, hd, 10000.0)).cuda()
    kp = torch.zeros(B, 16, nkv, hd, dtype=torch.float16, device="cuda")
    vp = torch.zeros_like(kp)
    table = torch.arange(B, dtype=torch.int32, device="cuda")[:, None].contiguous()
    lens = lambda **kw: torch.tensor([kw.get(f"s{i}", 1) for i in range(B)], dtype=torch.int32, device="cuda")  # noqa: E731
    want = ops.rope_append(x, rope, lens(), table, kp, vp, nh)
    assert ops.device_error() == 0
    for bad in (dict(s0=-3), dict(s299=-1), dict(s280=17)):  # below zero; above the table's one page of 16
        got = ops.rope_append(x, rope, lens(**bad), table, kp, vp, nh)
        assert ops.device_error() == native.DEVERR_DECODE_RANGE
        assert torch.equal(got[100:200], want[100:200])
    cu = torch.arange(B + 1, dtype=torch.int32, device="cuda")
    one = cu.clone()
    one[B - 1:] = B + 5  # the last sequence begins and ends behind the rows
    got = ops.rope_append(x, rope, lens(), table, kp, vp, nh, cu_q=one)
    assert ops.device_error() == native.DEVERR_DECODE_RANGE
    assert torch.equal(got[100:200], want[100:200])
    none = lens(s7=40)  # a length past the table, without a new row
    cu[8:] -= 1
    ops.rope_append(x, rope, none, table, kp, vp, nh, cu_q=cu)
    assert ops.device_error() == native.DEVERR_DECODE_RANGE


# ------------------------------------------------------------------ paged attention
PAGED = [
    # nh, nkv, hd, page, lengths
    (32, 32, 128, 16, [1, 2, 15, 16, 17, 63, 64, 65]),
    (64, 8, 128, 16, [512, 0, 1, 700, 333, 1024, 64, 129]),
    (8, 1, 128, 64, [5000, 1, 0]),
    (8, 1, 64, 32, [4097, 31]),
    (12, 4, 64, 128, [129, 128, 127, 1, 0, 640]),
    (40, 2, 128, 256, [300, 256, 255, 1]),  # 20 query heads on one KV head
    (5, 5, 128, 16, [77]),
    (33, 1, 128, 32, [999, 40]),            # 33 on one
]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("nh,nkv,hd,page,lens", PAGED)
@pytest.mark.parametrize("out", ["same", "float32"])
def test_attention_paged(cuda, dtype, nh, nkv, hd, page, lens, out):
    torch = cuda
    dt = getattr(torch, dtype)
    k = [rand(torch, n, nkv, hd, dt=dt, seed=10 + i) for i, n in enumerate(lens)]
    v = [rand(torch, n, nkv, hd, dt=dt, seed=50 + i) for i, n in enumerate(lens)]
    layout = ["token", "head", "padded"][len(lens) % 3]
    kp, vp, table = make_pages(torch, k, v, page, layout)
    q = rand(torch, len(lens), nh, hd, dt=dt, seed=99, scale=2.0)
    kv = torch.tensor(lens, dtype=torch.int32, device="cuda")
    odt = dt if out == "same" else torch.float32
    ws = torch.empty(ops.attention_paged_workspace(len(lens), nh, nkv, hd), dtype=torch.uint8, device="cuda")
    got = ops.attention_paged(q, kp, vp, table, kv, out_dtype=odt, workspace=ws.fill_(255))  # NaN to begin with
    again = ops.attention_paged(q, kp, vp, table, kv, out_dtype=odt)
    torch.cuda.synchronize()
    assert got.dtype == odt and torch.equal(got, again)  # the same bits every time
    for i, n in enumerate(lens):
        want, pv, serr = exact_attention(torch, q[i:i + 1], k[i], v[i], hd ** -0.5, n - 1)
        close(torch, got[i:i + 1], want, pv, serr, max(1, n), paged_weight(torch, dt, n), dt, f"sequence {i} of {n}")


def test_attention_paged_long_tail_of_small_weights(cuda):
    # one key far above 60000 others whose weights are near 2^-25 of it: together they still count
    torch = cuda
    n, hd = 60001, 128
    q = torch.zeros(1, 1, hd, dtype=torch.float16, device="cuda")
    q[..., 0] = 1.0
    k = torch.zeros(n, 1, hd, dtype=torch.float16, device="cuda")
    k[1234, 0, 0] = 17.5
    v = torch.ones(n, 1, hd, dtype=torch.float16, device="cuda")
    v[1234] = 0.0
    kp, vp, table = make_pages(torch, [k], [v], 64)
    kv = torch.tensor([n], dtype=torch.int32, device="cuda")
    got = ops.attention_paged(q, kp, vp, table, kv, scale=1.0, out_dtype=torch.float32)
    want, pv, serr = exact_attention(torch, q, k, v, 1.0, n - 1)
    close(torch, got, want, pv, serr, n, paged_weight(torch, torch.float16, n), torch.float16)
    cu = torch.tensor([0, 1], dtype=torch.int32, device="cuda")
    got = ops.attention_prompt(q, kp, vp, cu, kv_len=kv, page_table=table, scale=1.0, out_dtype=torch.float32)
    # n weights of fp16 with 2^-32 of the largest as their step
    close(torch, got, want, pv, serr, n, prompt_weight(torch, torch.float16, n), torch.float16)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("n", WEIGHT_CASES)
@pytest.mark.parametrize("nkv,group,hd", [(4, 1, 128), (2, 12, 64)])
def test_fp32_outputs_have_weights_of_two_parts(cuda, dtype, n, nkv, group, hd):
    # exact scores, fp32 outputs, a bound that weights of one 16-bit rounding miss
    torch = cuda
    dt = getattr(torch, dtype)
    q, k, v = one_value_case(torch, dt, n, nkv, hd, "cuda", n)
    q = q.repeat_interleave(group, 1)
    want, tol = (x.repeat_interleave(group, 1) for x in one_value_exact(torch, k, v))
    kp, vp, table = make_pages(torch, [k], [v], 16)
    kv = torch.tensor([n], dtype=torch.int32, device="cuda")
    cu = torch.tensor([0, 1], dtype=torch.int32, device="cuda")
    wide = torch.zeros(1, 300, dtype=torch.int32, device="cuda")  # keys that may be many: dealt out by key tiles
    wide[:, :table.shape[1]] = table
    for got in (ops.attention_paged(q, kp, vp, table, kv, scale=1.0, out_dtype=torch.float32),
                ops.attention_prompt(q, kp, vp, cu, kv_len=kv, page_table=table, scale=1.0, out_dtype=torch.float32),
                ops.attention_prompt(q, kp, vp, cu, kv_len=kv, page_table=wide, scale=1.0, out_dtype=torch.float32)):
        err = (got.double() - want).abs()
        assert (err <= tol).all(), f"worst {float((err / tol).max()):.3g} of the bound"


def test_attention_paged_strided_query_scale_and_out(cuda):
    torch = cuda
    nh, nkv, hd, lens = 8, 2, 128, [100, 7]
    k = [rand(torch, n, nkv, hd, dt=torch.bfloat16, seed=i) for i, n in enumerate(lens)]
    v = [rand(torch, n, nkv, hd, dt=torch.bfloat16, seed=9 + i) for i, n in enumerate(lens)]
    kp, vp, table = make_pages(torch, k, v, 16)
    kv = torch.tensor(lens, dtype=torch.int32, device="cuda")
    rows = rand(torch, 2, nh + 5, hd + 8, dt=torch.bfloat16, seed=3)
    q = rows[:, 2:2 + nh, :hd]
    ws = torch.empty(ops.attention_paged_workspace(2, nh, nkv, hd), dtype=torch.uint8, device="cuda").fill_(255)
    out = torch.full((2, nh, hd), float("nan"), device="cuda")
    got = ops.attention_paged(q, kp, vp, table, kv, scale=0.3, out=out, workspace=ws)
    assert got is out
    for i, n in enumerate(lens):
        want, pv, serr = exact_attention(torch, q[i:i + 1], k[i], v[i], 0.3, n - 1)
        close(torch, got[i:i + 1], want, pv, serr, n, paged_weight(torch, torch.bfloat16, n), torch.bfloat16)


def test_attention_nonfinite_inputs_of_attended_positions_show(cuda):
    torch = cuda
    n, hd = 200, 128
    k, v = (rand(torch, n, 1, hd, dt=torch.float16, seed=i) for i in (1, 2))
    v[150, 0, 3] = float("inf")
    k[20, 0, 0] = float("nan")
    kp, vp, table = make_pages(torch, [k, v], [v, v], 16)
    q = rand(torch, 2, 2, hd, dt=torch.float16, seed=5)
    kv = torch.tensor([n, n], dtype=torch.int32, device="cuda")
    got = ops.attention_paged(q, kp, vp, table, kv)
    assert torch.isnan(got[0]).all()           # a NaN key reaches every value of its sequence
    got = ops.attention_paged(q[:1], kp, vp, table[:1], torch.tensor([20], dtype=torch.int32, device="cuda"))
    assert torch.isfinite(got).all()           # ... unless it is behind the sequence's end


def with_nonfinite(v, where):
    """v with values set: {(position, head, column): value}."""
    v = v.clone()
    for at, x in where.items():
        v[at] = x
    return v


def check_nonfinite(torch, got, q, k, v, scale, first, weight, dt, what):
    """got [n, nh, hd] against the definition where v holds infinities and NaN: a column whose attended values
    hold a NaN or infinities of both signs is NaN, one with an infinity is that infinity, the others are as ever."""
    n, nh, _ = got.shape
    m, g = k.shape[0], nh // k.shape[1]
    want, pv, serr = exact_attention(torch, q, k, torch.nan_to_num(v, nan=0.0, posinf=0.0, neginf=0.0), scale, first)
    keep = (torch.arange(m, device="cuda")[None] <= (first + torch.arange(n, device="cuda"))[:, None]).double()
    seen = lambda x: torch.einsum("nm,mhd->nhd", keep, x.double()).repeat_interleave(g, 1) > 0  # noqa: E731
    plus, minus, nan = seen(v == math.inf), seen(v == -math.inf), seen(v != v)
    nan |= plus & minus
    assert torch.isnan(got[nan]).all(), what
    assert (got[plus & ~nan] == math.inf).all() and (got[minus & ~nan] == -math.inf).all(), what
    rest = ~(plus | minus | nan)
    close(torch, torch.where(rest, got, 0), torch.where(rest, want, 0), pv, serr, max(1, m), weight, dt, what)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("out", ["same", "float32"])
@pytest.mark.parametrize("nh,nkv,hd,page", [(4, 4, 128, 16), (16, 2, 64, 64), (32, 2, 128, 32), (9, 1, 64, 16)])
def test_attention_paged_infinite_values(cuda, dtype, out, nh, nkv, hd, page):
    # an attended infinity comes out as itself whatever its weight's low part is
    torch = cuda
    dt = getattr(torch, dtype)
    inf, nan = math.inf, math.nan
    lens = [1, 40, 700, 33, 6000]  # whole units, and one whose positions are dealt out
    k = [rand(torch, n, nkv, hd, dt=dt, seed=i) for i, n in enumerate(lens)]
    v = [rand(torch, n, nkv, hd, dt=dt, seed=20 + i) for i, n in enumerate(lens)]
    v[0] = with_nonfinite(v[0], {(0, 0, 0): inf, (0, nkv - 1, 3): -inf})
    v[1] = with_nonfinite(v[1], {(i, 0, i): inf for i in range(40)})  # a weight each
    v[2] = with_nonfinite(v[2], {(i, nkv - 1, i % 60): -inf for i in range(5, 700, 12)})
    v[3] = with_nonfinite(v[3], {(32, 0, 1): inf, (3, 0, 1): -inf, (9, 0, 2): nan, (9, 0, 8): inf, (31, 0, 2): inf})
    v[4] = with_nonfinite(v[4], {(p, nkv - 1, hd - 1 - i): inf for i, p in enumerate(range(0, 6000, 599))})
    kp, vp, table = make_pages(torch, k, v, page)
    q = rand(torch, len(lens), nh, hd, dt=dt, seed=99, scale=2.0)
    kv = torch.tensor(lens, dtype=torch.int32, device="cuda")
    got = ops.attention_paged(q, kp, vp, table, kv, out_dtype=dt if out == "same" else torch.float32)
    for i, n in enumerate(lens):
        check_nonfinite(torch, got[i:i + 1], q[i:i + 1], k[i], v[i], hd ** -0.5, n - 1, paged_weight(torch, dt, n), dt,
                        f"sequence {i} of {n}")


def test_attention_paged_bad_pages_and_lengths_are_reported(cuda):
    torch = cuda
    k = [rand(torch, 64, 2, 128, dt=torch.float16, seed=i) for i in range(3)]
    kp, vp, table = make_pages(torch, k, k, 16, width_extra=0)
    q = rand(torch, 3, 4, 128, dt=torch.float16, seed=7)
    kv = torch.tensor([64, 64, 64], dtype=torch.int32, device="cuda")
    good = ops.attention_paged(q, kp, vp, table, kv)
    for bad in (-1, kp.shape[0], 2 ** 31 - 1):
        t = table.clone()
        t[1, 2] = bad
        got = ops.attention_paged(q, kp, vp, t, kv)
        assert ops.device_error() == native.DEVERR_DECODE_RANGE
        assert torch.equal(got[0], good[0]) and torch.equal(got[2], good[2]) and torch.isfinite(got[1]).all()
    got = ops.attention_paged(q, kp, vp, table, torch.tensor([64, 65, -3], dtype=torch.int32, device="cuda"))
    assert ops.device_error() == native.DEVERR_DECODE_RANGE
    assert torch.equal(got[:2], good[:2]) and (got[2] == 0).all()


def test_attention_paged_offsets_past_32_bits(cuda):
    # a pool of over 2^32 bytes and over 2^31 elements; only two far pages are filled
    torch = cuda
    pages, page, hd = 2 ** 31 // (16 * 128) + 40, 16, 128
    kp = torch.empty(pages, page, 1, hd, dtype=torch.float16, device="cuda")
    vp = torch.empty_like(kp)
    k, v = (rand(torch, 30, 1, hd, dt=torch.float16, seed=i) for i in (1, 2))
    where = [pages - 1, 5]
    for i, pg in enumerate(where):
        rows = k[16 * i:16 * i + 16]
        kp[pg, :rows.shape[0]] = rows
        vp[pg, :rows.shape[0]] = v[16 * i:16 * i + 16]
    table = torch.tensor([where], dtype=torch.int32, device="cuda")
    kv = torch.tensor([30], dtype=torch.int32, device="cuda")
    q = rand(torch, 1, 1, hd, dt=torch.float16, seed=3)
    got = ops.attention_paged(q, kp, vp, table, kv, out_dtype=torch.float32)
    want, pv, serr = exact_attention(torch, q, k, v, hd ** -0.5, 29)
    close(torch, got, want, pv, serr, 30, paged_weight(torch, torch.float16, 30), torch.float16)
    got = ops.attention_prompt(q, kp, vp, torch.tensor([0, 1], dtype=torch.int32, device="cuda"), kv_len=kv,
                               page_table=table)
    close(torch, got, want, pv, serr, 30, prompt_weight(torch, torch.float16, 30), torch.float16)
    rope = torch.from_numpy(D.rope_table(64, hd, 10000.0)).cuda()
    x = rand(torch, 1, 3 * hd, dt=torch.float32, seed=4)
    kv = torch.tensor([16], dtype=torch.int32, device="cuda")  # offset 15 of the last page
    ops.rope_append(x, rope, kv, table, kp, vp, 1)
    assert torch.equal(vp[pages - 1, 15, 0], x[0, 2 * hd:].half())


# ------------------------------------------------------------------ prompt attention
PROMPT = [
    # nh, nkv, hd, q lengths, extra keys before them (paged only), page (0: packed)
    (4, 4, 128, [1], None, 0),
    (2, 2, 128, [64, 65, 63, 1, 128, 127, 129], None, 0),
    (4, 2, 128, [300, 0, 5, 257, 256, 255], None, 0),
    (6, 2, 64, [33, 513, 1, 100], None, 0),      # three query heads per KV head
    (8, 1, 64, [1025, 7], None, 0),
    (32, 32, 128, [130], None, 0),
    (8, 1, 128, [40, 1, 130, 3], [0, 700, 17, 255], 16),
    (4, 4, 128, [200, 129, 1], [56, 1, 1000], 64),
    (8, 2, 64, [128, 128], [128, 0], 128),
    (5, 1, 128, [260, 9], [300, 4], 256),
    (16, 2, 128, [1, 1, 1, 2], [0, 300, 15, 16], 32),
    # few items over many keys: their key tiles are dealt out in equal shares and joined
    (2, 1, 128, [5, 1, 128], [3000, 1290, 0], 64),
    (1, 1, 64, [300, 1], [2000, 0], 16),
    (3, 1, 128, [1, 257, 0, 2], [5000, 1100, 0, 127], 128),
    (8, 1, 128, [130, 64], [4000, 1], 256),
    (2, 2, 64, [1500], None, 0),
    (4, 2, 128, [1100, 3, 129], None, 0),
]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("nh,nkv,hd,q_len,prefix,page", PROMPT)
@pytest.mark.parametrize("out", ["same", "float32"])
def test_attention_prompt(cuda, dtype, nh, nkv, hd, q_len, prefix, page, out):
    torch = cuda
    dt = getattr(torch, dtype)
    T, tail = sum(q_len), 70
    kv_len = [n + p for n, p in zip(q_len, prefix or [0] * len(q_len))]
    q = rand(torch, T + tail, nh, hd, dt=dt, seed=1, scale=2.0)
    cu_h = np.concatenate([[0], np.cumsum(q_len)])
    cu = torch.tensor(cu_h, dtype=torch.int32, device="cuda")
    odt = dt if out == "same" else torch.float32
    got = torch.full((T + tail, nh, hd), 55.0, dtype=odt, device="cuda")
    if page:
        k = [rand(torch, n, nkv, hd, dt=dt, seed=20 + i) for i, n in enumerate(kv_len)]
        v = [rand(torch, n, nkv, hd, dt=dt, seed=60 + i) for i, n in enumerate(kv_len)]
        kp, vp, table = make_pages(torch, k, v, page, ["token", "head", "padded"][len(q_len) % 3])
        kv = torch.tensor(kv_len, dtype=torch.int32, device="cuda")
        call = lambda: ops.attention_prompt(q, kp, vp, cu, kv_len=kv, page_table=table, out=got)  # noqa: E731
    else:
        K, V = (rand(torch, T + 30, nkv, hd, dt=dt, seed=i) for i in (2, 3))
        K[T:] = float("nan")  # behind the last sequence
        V[T:] = float("nan")
        k, v = ([X[cu_h[i]:cu_h[i + 1]] for i in range(len(q_len))] for X in (K, V))
        call = lambda: ops.attention_prompt(q, K, V, cu, cu_k=cu, out=got)  # noqa: E731
    call()
    first = got.clone()
    call()
    torch.cuda.synchronize()
    assert torch.equal(first, got)
    assert (got[T:] == 55.0).all()
    for i, (n, m) in enumerate(zip(q_len, kv_len)):
        rows = slice(int(cu_h[i]), int(cu_h[i + 1]))
        want, pv, serr = exact_attention(torch, q[rows], k[i], v[i], hd ** -0.5, m - n)
        close(torch, got[rows], want, pv, serr, max(m, 1), prompt_weight(torch, dt, m), dt, f"sequence {i}")


@pytest.mark.parametrize("dtype", DTYPES)
def test_attention_prompt_long(cuda, dtype):
    torch = cuda
    dt = getattr(torch, dtype)
    n, nh, hd = 4100, 2, 128
    q = rand(torch, n, nh, hd, dt=dt, seed=1, scale=2.0)
    k, v = (rand(torch, n, 1, hd, dt=dt, seed=i) for i in (2, 3))
    cu = torch.tensor([0, n], dtype=torch.int32, device="cuda")
    got = ops.attention_prompt(q, k, v, cu)
    want, pv, serr = exact_attention(torch, q, k, v, hd ** -0.5, 0)
    close(torch, got, want, pv, serr, n, prompt_weight(torch, dt, n), dt)


@pytest.mark.parametrize("step", [0.05, 0.5, 5.0])
def test_attention_prompt_rising_scores(cuda, step):
    # every key's score is above all before it: the running maximum rises in every tile
    torch = cuda
    n, hd = 700, 128
    q = torch.zeros(n, 1, hd, dtype=torch.float16, device="cuda")
    q[..., 0] = 1.0
    q[..., 1] = 1.0
    k = torch.zeros_like(q)
    x = torch.arange(n, device="cuda").float() * step
    k[:, 0, 0] = x.half()
    k[:, 0, 1] = (x - k[:, 0, 0].float()).half()
    v = rand(torch, n, 1, hd, dt=torch.float16, seed=3)
    cu = torch.tensor([0, n], dtype=torch.int32, device="cuda")
    for sign in (1.0, -1.0):
        got = ops.attention_prompt(q * sign, k, v, cu, scale=1.0)
        want, pv, serr = exact_attention(torch, q * sign, k, v, 1.0, 0)
        close(torch, got, want, pv, serr, n, prompt_weight(torch, torch.float16, n), torch.float16)


@pytest.mark.parametrize("page,width", [(0, 0), (16, 0), (16, 100)])  # 100 more columns: dealt out in shares
def test_attention_prompt_later_values_do_not_reach_earlier_rows(cuda, page, width):
    torch = cuda
    q_len, nh, nkv, hd = [150, 300], 4, 2, 128
    T = sum(q_len)
    q = rand(torch, T, nh, hd, dt=torch.bfloat16, seed=1)
    k, v = (rand(torch, T, nkv, hd, dt=torch.bfloat16, seed=i) for i in (2, 3))
    cu = torch.tensor([0, 150, 450], dtype=torch.int32, device="cuda")

    def call(k, v):
        if not page:
            return ops.attention_prompt(q, k, v, cu)
        kp, vp, table = make_pages(torch, [k[:150], k[150:]], [v[:150], v[150:]], page, width_extra=width)
        kv = torch.tensor(q_len, dtype=torch.int32, device="cuda")
        return ops.attention_prompt(q, kp, vp, cu, kv_len=kv, page_table=table)

    good = call(k, v)
    k2, v2 = k.clone(), v.clone()
    v2[100, 0, 5] = float("nan")    # position 100 of the first sequence, KV head 0
    v2[150 + 200, 1, 7] = float("inf")  # position 200 of the second, KV head 1
    k2[150 + 250, 0] = float("nan")     # position 250, KV head 0
    got = call(k2, v2)
    assert torch.isfinite(good).all()
    u = half_step(torch, torch.bfloat16)
    # rows before the position: computed another way at most, each way within 2u of the exact value
    same = lambda a, b: ((a.float() - b.float()).abs() <= 4 * u * (1 + b.float().abs())).all()  # noqa: E731
    assert same(got[:100], good[:100]) and torch.equal(got[:150, 2:], good[:150, 2:])
    assert torch.isnan(got[100:150, :2, 5]).all()
    assert same(got[100:150, :2, 6:], good[100:150, :2, 6:])
    assert same(got[150:350], good[150:350])
    assert (~torch.isfinite(got[350:, 2:, 7])).all()
    assert same(got[150:400, :2], good[150:400, :2]) and torch.isnan(got[400:, :2]).all()


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("out", ["same", "float32"])
@pytest.mark.parametrize("nh,nkv,hd,page,width", [(4, 2, 128, 0, 0), (3, 1, 64, 16, 0), (2, 2, 128, 32, 300)])
def test_attention_prompt_infinite_values(cuda, dtype, out, nh, nkv, hd, page, width):
    # an attended infinity shows whatever is left of its weight in 16 bits; one behind the row does not
    torch = cuda
    dt = getattr(torch, dtype)
    inf, nan = math.inf, math.nan
    q_len = [200, 1, 150]
    kv_len = [200, 90, 400] if page else q_len
    k = [rand(torch, n, nkv, hd, dt=dt, seed=i) for i, n in enumerate(kv_len)]
    v = [rand(torch, n, nkv, hd, dt=dt, seed=20 + i) for i, n in enumerate(kv_len)]
    q = [rand(torch, n, nh, hd, dt=dt, seed=40 + i, scale=2.0) for i, n in enumerate(q_len)]
    for x in q:
        x[..., 0] = 4.0
    faint = [10, 0, 77]  # a key some 40 below the others: e^-40 = 2^-58 of their weight
    for x, j in zip(k, faint):
        x[j, :, 0] = -10.0 * hd ** 0.5
    v[0] = with_nonfinite(v[0], {(10, 0, 2): inf, (10, nkv - 1, 5): -inf, (60, 0, 5): inf, (150, 0, 7): nan})
    v[1] = with_nonfinite(v[1], {(0, nkv - 1, 9): inf})
    v[2] = with_nonfinite(v[2], {(77, 0, 11): -inf, (77, nkv - 1, 50): inf, (149, 0, 50): -inf, (3, 0, 12): inf})
    cu_h = np.concatenate([[0], np.cumsum(q_len)])
    cu = torch.tensor(cu_h, dtype=torch.int32, device="cuda")
    odt = dt if out == "same" else torch.float32
    if page:
        kp, vp, table = make_pages(torch, k, v, page, width_extra=width)
        got = ops.attention_prompt(torch.cat(q), kp, vp, cu, page_table=table, out_dtype=odt,
                                   kv_len=torch.tensor(kv_len, dtype=torch.int32, device="cuda"))
    else:
        got = ops.attention_prompt(torch.cat(q), torch.cat(k), torch.cat(v), cu, out_dtype=odt)
    for i, (n, m) in enumerate(zip(q_len, kv_len)):
        check_nonfinite(torch, got[int(cu_h[i]):int(cu_h[i + 1])], q[i], k[i], v[i], hd ** -0.5, m - n,
                        prompt_weight(torch, dt, m), dt, f"sequence {i}")


@pytest.mark.parametrize("split", [False, True])
def test_attention_prompt_later_value_behind_a_long_prefix(cuda, split):
    # the rows computed again have 20000 keys each, while the CTA's other roles wait
    torch = cuda
    nh, hd, page, prefix, n = (1, 128, 64, 20000, 100) if split else (160, 128, 64, 20000, 100)
    k = rand(torch, prefix + n, 1, hd, dt=torch.float16, seed=2)
    v = rand(torch, prefix + n, 1, hd, dt=torch.float16, seed=3)
    v[prefix + 60, 0, 9] = float("nan")
    kp, vp, table = make_pages(torch, [k], [v], page)
    q = rand(torch, n, nh, hd, dt=torch.float16, seed=1)
    cu = torch.tensor([0, n], dtype=torch.int32, device="cuda")
    kv = torch.tensor([prefix + n], dtype=torch.int32, device="cuda")
    got = ops.attention_prompt(q, kp, vp, cu, kv_len=kv, page_table=table)
    v[prefix + 60, 0, 9] = 0.0
    heads = [0, nh - 1] if nh > 1 else [0]
    want, pv, serr = exact_attention(torch, q[:60, heads], k, v, hd ** -0.5, prefix)
    close(torch, got[:60, heads], want, pv, serr, prefix, prompt_weight(torch, torch.float16, prefix), torch.float16)
    assert torch.isnan(got[60:, :, 9]).all() and torch.isfinite(got[:60]).all()


def test_attention_prompt_rows_without_keys_and_strided_inputs(cuda):
    torch = cuda
    nh, nkv, hd = 4, 2, 128
    buf = rand(torch, 90, (nh + 2 * nkv) * hd + 8, dt=torch.float16, seed=1)
    heads = buf[:, :(nh + 2 * nkv) * hd].unflatten(1, (nh + 2 * nkv, hd))
    q, k, v = heads[:, :nh], heads[:, nh:nh + nkv], heads[:, nh + nkv:]
    cu_q = torch.tensor([0, 50, 90], dtype=torch.int32, device="cuda")
    cu_k = torch.tensor([0, 20, 90], dtype=torch.int32, device="cuda")  # 20 keys for 50 rows; 70 for 40
    got = ops.attention_prompt(q, k, v, cu_q, cu_k=cu_k)
    assert (got[:30] == 0).all()
    for a, b, ka, kb in ((30, 50, 0, 20), (50, 90, 20, 90)):
        want, pv, serr = exact_attention(torch, q[a:b], k[ka:kb], v[ka:kb], hd ** -0.5, (kb - ka) - (b - a))
        close(torch, got[a:b], want, pv, serr, kb - ka, prompt_weight(torch, torch.float16, 100), torch.float16)


def test_attention_prompt_packed_without_any_key(cuda):
    torch = cuda
    q = rand(torch, 6, 4, 64, dt=torch.float16, seed=1)
    none = q.new_empty(0, 2, 64)
    cu = torch.tensor([0, 2, 5], dtype=torch.int32, device="cuda")
    for stream in (None, torch.cuda.Stream()):
        torch.cuda.synchronize()
        out = torch.full((6, 4, 64), 7.0, device="cuda")
        torch.cuda.synchronize()
        ops.attention_prompt(q, none, none, cu, cu_k=torch.zeros_like(cu), out=out, stream=stream)
        torch.cuda.synchronize()
        assert (out[:5] == 0).all() and (out[5] == 7.0).all()
    with pytest.raises(ValueError):
        ops.attention_prompt(q, none, q.new_empty(1, 2, 64), cu, cu_k=torch.zeros_like(cu))


@pytest.mark.parametrize("nh,nkv,hd,long,empty", [(64, 8, 64, 3, 0.5), (64, 8, 128, 300, 0.9), (32, 32, 128, 40, 1.0),
                                                  (1, 1, 128, 60000, 0.9), (2, 1, 64, 30000, 0.7)])
def test_attention_prompt_runs_of_sequences_without_keys(cuda, nh, nkv, hd, long, empty):
    # rows of sequences that hold no position yet, several to a CTA behind one that has keys; the last two cases are
    # dealt out by key tiles
    torch = cuda
    rng = np.random.default_rng(5)
    B, page = (100 if nh < 4 else 300), 64
    q_len = rng.integers(1, 4, B)
    kv_len = np.where(rng.random(B) < empty, 0, q_len + rng.integers(0, 4, B))
    kv_len[[0, B // 3]] = q_len[[0, B // 3]] + [long, 1]
    if empty < 1.0:
        q_len[B // 2], kv_len[B // 2] = 700, 150  # whole tiles of rows before the first key
    T = int(q_len.sum())
    k, v = ([rand(torch, int(n), nkv, hd, dt=torch.float16, seed=c + i) for i, n in enumerate(kv_len)] for c in (0, 900))
    kp, vp, table = make_pages(torch, k, v, page)
    q = rand(torch, T, nh, hd, dt=torch.float16, seed=1, scale=2.0)
    cu_h = np.concatenate([[0], np.cumsum(q_len)])
    out = torch.full((T, nh, hd), 99.0, dtype=torch.float16, device="cuda")
    ops.attention_prompt(q, kp, vp, torch.tensor(cu_h, dtype=torch.int32, device="cuda"), page_table=table, out=out,
                         kv_len=torch.tensor(kv_len, dtype=torch.int32, device="cuda"))
    assert ops.device_error() == 0  # a role that waited for what could not come would have given up
    for s in range(B):
        a, b, n = int(cu_h[s]), int(cu_h[s + 1]), int(kv_len[s])
        assert (out[a:max(a, b - n)] == 0).all(), f"sequence {s}"
        if n:
            want, pv, serr = exact_attention(torch, q[a:b], k[s], v[s], hd ** -0.5, n - (b - a))
            close(torch, out[a:b], want, pv, serr, n, prompt_weight(torch, torch.float16, n), torch.float16, f"{s}")


def test_attention_prompt_bits_do_not_depend_on_what_shared_memory_held(cuda):
    # sequences of 3 rows and 200 keys, in tiles of 128 of each: the rest of a tile must not change a bit
    torch = cuda
    B, n, nh, hd, page = 200, 200, 2, 128, 16
    k = [rand(torch, n, 1, hd, dt=torch.bfloat16, seed=i) for i in range(B)]
    kp, vp, table = make_pages(torch, k, k, page)
    q = rand(torch, 3 * B, nh, hd, dt=torch.bfloat16, seed=1, scale=2.0)
    cu = torch.arange(B + 1, dtype=torch.int32, device="cuda") * 3
    kv = torch.full((B,), n, dtype=torch.int32, device="cuda")
    other = torch.arange(65, dtype=torch.int32, device="cuda") * 512
    got = []
    for size in (0.0, 300.0, 0.01):  # keys that a call before this one leaves behind
        x = rand(torch, 64 * 512, 4, hd, dt=torch.bfloat16, seed=5) * size
        ops.attention_prompt(x, x, x, other)
        got.append(ops.attention_prompt(q, kp, vp, cu, kv_len=kv, page_table=table, out_dtype=torch.float32))
    for size in (0.0, 300.0, float("nan")):  # rows behind the last sequence
        padded = torch.cat([q, torch.full_like(q[:100], 1.0) * size])
        got.append(ops.attention_prompt(padded, kp, vp, cu, kv_len=kv, page_table=table, out_dtype=torch.float32)[:3 * B])
    torch.cuda.synchronize()
    assert all(torch.equal(got[0], g) for g in got[1:])


def test_attention_prompt_many_sequences(cuda):
    torch = cuda
    nh, nkv, hd = 2, 1, 128
    rng = np.random.default_rng(0)
    q_len = rng.integers(0, 9, 1000)
    q_len[500] = 400
    T = int(q_len.sum())
    q = rand(torch, T, nh, hd, dt=torch.bfloat16, seed=1)
    k, v = (rand(torch, T, nkv, hd, dt=torch.bfloat16, seed=i) for i in (2, 3))
    cu_h = np.concatenate([[0], np.cumsum(q_len)])
    got = ops.attention_prompt(q, k, v, torch.tensor(cu_h, dtype=torch.int32, device="cuda"))
    for s in list(range(0, 1000, 37)) + [500, 999]:
        a, b = int(cu_h[s]), int(cu_h[s + 1])
        want, pv, serr = exact_attention(torch, q[a:b], k[a:b], v[a:b], hd ** -0.5, 0)
        close(torch, got[a:b], want, pv, serr, max(1, b - a), prompt_weight(torch, torch.bfloat16, b - a),
              torch.bfloat16, f"sequence {s}")


def test_attention_prompt_many_sequences_of_many_lengths(cuda):
    # more sequences than the scheduler holds, many items a CTA: rows and keys of every count of key tiles, some none
    torch = cuda
    rng = np.random.default_rng(7)
    B, nh, nkv, hd, page = 350, 4, 2, 64, 32
    q_len = np.where(rng.random(B) < 0.1, 0, np.exp(rng.uniform(0, math.log(300), B)).astype(int))
    kv_len = np.where(rng.random(B) < 0.1, q_len // 2, q_len + rng.integers(0, 900, B) * (rng.random(B) < 0.5))
    T = int(q_len.sum())
    k, v = ([rand(torch, int(n), nkv, hd, dt=torch.bfloat16, seed=c + i) for i, n in enumerate(kv_len)] for c in (0, 900))
    kp, vp, table = make_pages(torch, k, v, page)
    q = rand(torch, T, nh, hd, dt=torch.bfloat16, seed=1, scale=2.0)
    cu_h = np.concatenate([[0], np.cumsum(q_len)])
    got = ops.attention_prompt(q, kp, vp, torch.tensor(cu_h, dtype=torch.int32, device="cuda"), page_table=table,
                               kv_len=torch.tensor(kv_len, dtype=torch.int32, device="cuda"))
    for s in range(B):
        a, b, n = int(cu_h[s]), int(cu_h[s + 1]), int(kv_len[s])
        if b > a:
            want, pv, serr = exact_attention(torch, q[a:b], k[s], v[s], hd ** -0.5, n - (b - a))
            close(torch, got[a:b], want, pv, serr, max(1, n), prompt_weight(torch, torch.bfloat16, n), torch.bfloat16,
                  f"sequence {s}")


def test_attention_prompt_time_grows_with_the_sequences_not_their_square(cuda):
    # four times the sequences are four times the work; where every item was looked for from the start it took 18
    # times as long
    torch = cuda
    best = {}
    for B in (256, 1024):
        lens = torch.randint(1, 101, (B,), generator=torch.Generator().manual_seed(B))
        cu = torch.cat([torch.zeros(1, dtype=torch.long), lens.cumsum(0)]).int().cuda()
        q, k, v = (torch.randn(int(lens.sum()), n, 128, device="cuda").half() for n in (32, 8, 8))
        times = []
        for _ in range(6):
            a, b = (torch.cuda.Event(enable_timing=True) for _ in range(2))
            a.record()
            ops.attention_prompt(q, k, v, cu)
            b.record()
            torch.cuda.synchronize()
            times.append(a.elapsed_time(b))
        best[B] = min(times)
    assert best[1024] < 8 * best[256], best


def test_attention_prompt_bad_offsets_and_pages_are_reported(cuda):
    torch = cuda
    q = rand(torch, 60, 2, 128, dt=torch.float16, seed=1)
    k = rand(torch, 60, 1, 128, dt=torch.float16, seed=2)
    cu = torch.tensor([0, 30, 60], dtype=torch.int32, device="cuda")
    good = ops.attention_prompt(q, k, k, cu)
    for bad in ([0, 30, 61], [-1, 30, 60], [0, 61, 60]):
        got = ops.attention_prompt(q, k, k, cu, cu_k=torch.tensor(bad, dtype=torch.int32, device="cuda"))
        assert ops.device_error() == native.DEVERR_DECODE_RANGE
        if bad[1] == 30:
            ok = slice(0, 30) if bad[0] == 0 else slice(30, 60)
            assert torch.equal(got[ok], good[ok])
    kp, vp, table = make_pages(torch, [k[:30], k[30:]], [k[:30], k[30:]], 16, width_extra=0)
    kv = torch.tensor([30, 30], dtype=torch.int32, device="cuda")
    table[0, 1] = 99
    got = ops.attention_prompt(q, kp, vp, cu, kv_len=kv, page_table=table)
    assert ops.device_error() == native.DEVERR_DECODE_RANGE
    assert torch.equal(got[30:], good[30:]) and torch.isfinite(got).all()


def test_attention_prompt_many_sequences_few_items(cuda):
    # 100 sequences on one head, most without new rows: dealt out by key tiles over more than one warp of sequences
    torch = cuda
    rng = np.random.default_rng(3)
    B, hd, page = 100, 128, 64
    q_len = np.where(rng.random(B) < 0.2, rng.integers(1, 6, B), 0)
    q_len[70] = 200
    kv_len = np.maximum(q_len, rng.integers(0, 2500, B))
    T = int(q_len.sum())
    k = [rand(torch, int(n), 1, hd, dt=torch.float16, seed=100 + i) for i, n in enumerate(kv_len)]
    v = [rand(torch, int(n), 1, hd, dt=torch.float16, seed=300 + i) for i, n in enumerate(kv_len)]
    kp, vp, table = make_pages(torch, k, v, page)
    q = rand(torch, T, 1, hd, dt=torch.float16, seed=1, scale=2.0)
    cu_h = np.concatenate([[0], np.cumsum(q_len)])
    got = ops.attention_prompt(q, kp, vp, torch.tensor(cu_h, dtype=torch.int32, device="cuda"), page_table=table,
                               kv_len=torch.tensor(kv_len, dtype=torch.int32, device="cuda"))
    for s in range(B):
        a, b, n = int(cu_h[s]), int(cu_h[s + 1]), int(kv_len[s])
        if b > a:
            want, pv, serr = exact_attention(torch, q[a:b], k[s], v[s], hd ** -0.5, n - (b - a))
            close(torch, got[a:b], want, pv, serr, n, prompt_weight(torch, torch.float16, n), torch.float16, f"{s}")


def test_attention_paged_many_sequences(cuda):
    # more sequences than a CTA has threads, many of them without positions
    torch = cuda
    rng = np.random.default_rng(4)
    B, nh, nkv, hd, page = 700, 2, 1, 64, 16
    lens = np.where(rng.random(B) < 0.3, 0, rng.integers(1, 90, B))
    lens[650] = 3000
    k = [rand(torch, int(n), nkv, hd, dt=torch.bfloat16, seed=i) for i, n in enumerate(lens)]
    kp, vp, table = make_pages(torch, k, k, page)
    q = rand(torch, B, nh, hd, dt=torch.bfloat16, seed=9)
    got = ops.attention_paged(q, kp, vp, table, torch.tensor(lens, dtype=torch.int32, device="cuda"))
    for s in list(range(0, B, 13)) + [650]:
        n = int(lens[s])
        want, pv, serr = exact_attention(torch, q[s:s + 1], k[s], k[s], hd ** -0.5, n - 1)
        close(torch, got[s:s + 1], want, pv, serr, max(1, n), paged_weight(torch, torch.bfloat16, n), torch.bfloat16,
              f"{s}")


def test_calls_without_rows(cuda):
    torch = cuda
    kp = torch.zeros(2, 16, 1, 128, dtype=torch.float16, device="cuda")
    none = torch.zeros(0, dtype=torch.int32, device="cuda")
    table = torch.zeros(0, 3, dtype=torch.int32, device="cuda")
    q = torch.zeros(0, 4, 128, dtype=torch.float16, device="cuda")
    assert ops.attention_paged(q, kp, kp, table, none).shape == (0, 4, 128)
    cu = torch.zeros(1, dtype=torch.int32, device="cuda")
    assert ops.attention_prompt(q, kp, kp, cu, kv_len=none, page_table=table).shape == (0, 4, 128)
    rope = torch.from_numpy(D.rope_table(8, 128, 10000.0)).cuda()
    x = torch.zeros(0, 6 * 128, device="cuda")
    assert ops.rope_append(x, rope, none, table, kp, kp, 4).shape == (0, 4, 128)
    logits = torch.zeros(0, 50, device="cuda")
    assert ops.rows_sample(logits, torch.zeros(0, device="cuda")).shape == (0,)
    two = torch.zeros(3, dtype=torch.int32, device="cuda")  # two sequences, none with a row
    out = torch.full((5, 4, 128), 3.0, dtype=torch.float16, device="cuda")
    rows = torch.zeros(5, 4, 128, dtype=torch.float16, device="cuda")
    ops.attention_prompt(rows, kp[0], kp[0], two, out=out)
    assert (out == 3.0).all()


def test_refusals_of_the_python_layer(cuda):
    torch = cuda
    h = lambda *s, dt=torch.float16: torch.zeros(*s, dtype=dt, device="cuda")  # noqa: E731
    i32 = lambda *s: torch.zeros(*s, dtype=torch.int32, device="cuda")  # noqa: E731
    kp, vp, table, n = h(4, 16, 2, 128), h(4, 16, 2, 128), i32(3, 2), i32(3)
    q, cu = h(3, 4, 128), i32(4)
    rope = torch.from_numpy(D.rope_table(8, 128, 10000.0)).cuda()
    x = torch.zeros(3, 8 * 128, device="cuda")
    sample = lambda **kw: ops.rows_sample(torch.zeros(3, 50, device="cuda"), torch.zeros(3, device="cuda"), **kw)  # noqa: E731
    for error, call in [
        (TypeError, lambda: ops.attention_paged(q.float(), kp, vp, table, n)),
        (ValueError, lambda: ops.attention_paged(q.bfloat16(), kp, vp, table, n)),
        (ValueError, lambda: ops.attention_paged(h(3, 5, 128), kp, vp, table, n)),          # 5 heads on 2
        (ValueError, lambda: ops.attention_paged(h(2, 4, 128), kp, vp, table, n)),          # 2 rows, 3 sequences
        (ValueError, lambda: ops.attention_paged(h(3, 4, 64), kp, vp, table, n)),
        (ValueError, lambda: ops.attention_paged(q, kp, vp[:, :, :1], table, n)),
        (ValueError, lambda: ops.attention_paged(q, kp, vp.transpose(1, 2).contiguous().transpose(1, 2), table, n)),
        (TypeError, lambda: ops.attention_paged(q, kp, vp, table.long(), n)),
        (TypeError, lambda: ops.attention_paged(q, kp, vp, table, n.long())),
        (ValueError, lambda: ops.attention_paged(q, kp, vp, table, i32(2))),
        (ValueError, lambda: ops.attention_paged(q, kp, vp, None, n)),
        (ValueError, lambda: ops.attention_paged(q, kp, vp, i32(2, 3).T, n)),
        (TypeError, lambda: ops.attention_paged(q, kp, vp, table, n, out_dtype=torch.bfloat16)),
        (ValueError, lambda: ops.attention_paged(q, kp, vp, table, n, out=h(3, 4, 64))),
        (ValueError, lambda: ops.attention_paged(q, kp, vp, table, n, out=q)),
        (ValueError, lambda: ops.attention_prompt(q, kp, vp, cu, kv_len=n, page_table=table, out=q)),
        (ops.AsmError, lambda: ops.attention_paged(q, kp, vp, table, n, scale=0.0)),
        (ops.AsmError, lambda: ops.attention_paged(q, kp, vp, table, n, scale=float("nan"))),
        (ops.AsmError, lambda: ops.attention_paged(q, kp, vp, table, n, workspace=h(16, dt=torch.uint8))),
        (ops.AsmError, lambda: ops.attention_paged(q, h(4, 24, 2, 128), h(4, 24, 2, 128), table, n)),
        (ops.AsmError, lambda: ops.attention_paged(h(3, 4, 96), h(4, 16, 2, 96), h(4, 16, 2, 96), table, n)),
        (ops.AsmError, lambda: ops.attention_paged(q[:, :1].expand(3, 4, 128), kp, vp, table, n)),
        (ops.AsmError, lambda: ops.attention_paged(h(3, 4, 132)[..., 4:], kp, vp, table, n)),  # rows of 264 bytes
        (ValueError, lambda: ops.attention_prompt(q, kp, vp, cu, kv_len=n)),
        (ValueError, lambda: ops.attention_prompt(q, kp, vp, cu, page_table=table)),
        (ValueError, lambda: ops.attention_prompt(q, kp, vp, cu, kv_len=n, page_table=table, cu_k=cu)),
        (ValueError, lambda: ops.attention_prompt(q, kp, vp, i32(3), kv_len=n, page_table=table)),
        (ValueError, lambda: ops.attention_prompt(q, kp, vp, cu)),                           # four axes, packed
        (ops.AsmError, lambda: ops.attention_prompt(q, h(5, 2, 128), h(5, 2, 128), cu, scale=-1.0)),
        (ValueError, lambda: ops.rope_append(x[:, :-128], rope, n, table, kp, vp, 4)),
        (ValueError, lambda: ops.rope_append(x, rope[:, :32], n, table, kp, vp, 4)),
        (ValueError, lambda: ops.rope_append(x[:2], rope, n, table, kp, vp, 4)),
        (TypeError, lambda: ops.rope_append(x.bfloat16(), rope, n, table, kp, vp, 4)),
        (ValueError, lambda: ops.rope_append(x, rope, n, table, kp, vp, 4, cu_q=i32(3))),
        (ValueError, lambda: ops.rope_append(x, rope, n, table, kp, vp, 4, q_out=h(3, 5, 128))),
        (TypeError, lambda: sample(temperature=torch.ones(3))),
        (ValueError, lambda: sample(top_p=torch.ones(2, device="cuda"))),
        (TypeError, lambda: sample(top_k=torch.ones(3, device="cuda"))),
        (TypeError, lambda: ops.rows_sample(torch.zeros(3, 50, device="cuda").double(), torch.zeros(3, device="cuda"))),
        (ops.AsmError, lambda: ops.rows_sample(h(1, 262145), torch.zeros(1, device="cuda"))),
    ]:
        with pytest.raises(error):
            call()


def test_outputs_over_inputs_are_refused(cuda):
    torch = cuda
    B, nh, nkv, hd, page = 3, 4, 2, 128, 16
    row = nh * hd
    arena = torch.zeros(1 << 16, dtype=torch.float16, device="cuda")
    part = lambda at, *s: arena[at:at + math.prod(s)].view(s)  # noqa: E731
    zeros = lambda *s, dt=torch.float16: torch.zeros(*s, dtype=dt, device="cuda")  # noqa: E731
    kp, vp = zeros(4, page, nkv, hd), zeros(4, page, nkv, hd)
    table, n, cu = (zeros(*s, dt=torch.int32) for s in ((B, 2), (B,), (B + 1,)))
    rope = torch.from_numpy(D.rope_table(8, hd, 10000.0)).cuda()
    x = zeros(B, (nh + 2 * nkv) * hd)
    q = part(0, B, nh, hd)
    paged = lambda q=q, k=kp, v=vp, **kw: ops.attention_paged(q, k, v, table, n, **kw)  # noqa: E731
    prompt = lambda q=q, k=kp, v=vp, **kw: ops.attention_prompt(q, k, v, cu, kv_len=n, page_table=table, **kw)  # noqa: E731
    append = lambda x=x, k=kp, v=vp, **kw: ops.rope_append(x, rope, n, table, k, v, nh, **kw)  # noqa: E731
    pool = part(1 << 14, 4, page, nkv, hd)
    behind = part((1 << 14) + 4 * page * nkv * hd, B, nh, hd)
    inside = part((1 << 14) + 4 * page * nkv * hd - 8, B, nh, hd)  # begins in the pool's last key
    before = part((1 << 14) - B * row + 8, B, nh, hd)              # ends in its first
    wide = arena.view(4, -1)[:B, :row].view(B, nh, hd)             # rows with room between them
    between = arena.view(4, -1)[0, row:2 * row].view(1, nh, hd)
    packed = arena[:6 * nkv * hd].view(6, nkv, hd)
    logits = torch.zeros(B, 64, device="cuda")
    need = ops.attention_paged_workspace(B, nh, nkv, hd)
    room = zeros(need + 4096, dt=torch.uint8)
    refused = [
        lambda: paged(out=part(8, B, nh, hd)), lambda: paged(out=part(B * row - 8, B, nh, hd)),
        lambda: prompt(out=part(8, B, nh, hd)), lambda: prompt(out=part(B * row - 8, B, nh, hd)),
        lambda: paged(k=pool, out=inside), lambda: paged(v=pool, out=inside), lambda: paged(k=pool, out=before),
        lambda: prompt(k=pool, out=before), lambda: prompt(v=pool, out=inside),
        lambda: ops.attention_prompt(zeros(3, nh, hd), packed, zeros(6, nkv, hd), cu, out=part(5 * nkv * hd, 3, nh, hd)),
        lambda: paged(q=wide, out=part(1 << 14, B, nh, hd)),  # the second row of q
        lambda: paged(out=room[-3 * row * 4:].view(torch.float32).view(B, nh, hd), workspace=room),
        lambda: paged(q=room[:B * row * 2].view(torch.float16).view(B, nh, hd), workspace=room),
        lambda: append(x=part(0, B, (nh + 2 * nkv) * hd), q_out=part(16, B, nh, hd)),
        lambda: append(k=pool, q_out=inside), lambda: append(v=pool, q_out=before),
        lambda: append(x=arena[1 << 14:][:B * 8 * hd].view(B, 8 * hd), v=pool),
        lambda: append(v=kp),
        lambda: ops.rows_sample(logits, logits[0, :B].clone(), tokens=logits.view(torch.int32)[1, 61:64]),
        lambda: ops.rows_sample(logits, u := torch.zeros(B, device="cuda"), tokens=u.view(torch.int32)),
    ]
    for call in refused:
        with pytest.raises(ops.AsmError, match="overlaps an input|same pages"):
            call()
    # beside an input, or between its rows, is not over it
    paged(q=wide[:, :], out=part(row, B, nh, hd)[:0].new_zeros(B, nh, hd))
    assert paged(k=pool, out=behind) is behind and prompt(v=pool, out=behind) is behind
    one = wide[1:2]
    ops.attention_paged(one, kp, vp, table[:1], n[:1], out=between)
    ops.attention_prompt(wide, kp, vp, cu, kv_len=n, page_table=table, out=part((1 << 14) + row, B, nh, hd))
    sliced = zeros(4, 3, page, nkv, hd)  # one layer's pages of a pool of three
    assert paged(k=sliced[:, 0], v=sliced[:, 2], out=sliced[1, 1].view(-1)[:B * row].view(B, nh, hd)) is not None
    append(k=sliced[:, 0], v=sliced[:, 1])
    both = zeros(4, page, 2 * nkv, hd)  # keys and values side by side
    append(k=both[:, :, :nkv], v=both[:, :, nkv:])
    torch.cuda.synchronize()


def test_two_streams_at_once(cuda):
    torch = cuda
    nh, nkv, hd, lens = 16, 2, 128, [2900, 17, 900]
    k = [rand(torch, n, nkv, hd, dt=torch.bfloat16, seed=i) for i, n in enumerate(lens)]
    kp, vp, table = make_pages(torch, k, k, 32)
    kv = torch.tensor(lens, dtype=torch.int32, device="cuda")
    q = rand(torch, 3, nh, hd, dt=torch.bfloat16, seed=7)
    cu = torch.arange(4, dtype=torch.int32, device="cuda")
    logits, u = rand(torch, 3, 32000, dt=torch.float32, seed=8), torch.rand(3, device="cuda")
    call = lambda st=None: (ops.attention_paged(q, kp, vp, table, kv, stream=st),  # noqa: E731
                            ops.attention_prompt(q, kp, vp, cu, kv_len=kv, page_table=table, stream=st),
                            ops.rows_sample(logits, u, stream=st))
    want = call()
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    got = [call(streams[i % 2]) for i in range(20)]
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for g in got for a, b in zip(g, want))
    graphs = []  # the prompt's keys are dealt out here: its scratch belongs to each graph
    for _ in range(2):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            out = call()
        graphs.append((g, out))
    for _ in range(3):
        for (g, out), st in zip(graphs, streams):
            with torch.cuda.stream(st):
                g.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for _, out in graphs for a, b in zip(out, want))


# ------------------------------------------------------------------ sampling
def sample_ref(x, u, T, k, p, mp):
    """One row in 64 bits: numpy, the definition word by word."""
    x = x.astype(np.float64)
    x[np.isnan(x)] = -np.inf
    m = x.max()
    if m == -np.inf:
        return -1
    order = np.argsort(-x, kind="stable")
    if not T > 0:
        return int(order[0])
    with np.errstate(invalid="ignore"):
        w = np.where(x == m, 1.0, np.exp((x - m) / T))
    keep = order[:k] if k > 0 else order
    c = np.cumsum(w[keep])
    n = int(np.sum(c - w[keep] < float(p) * c[-1])) if p < 1 else len(keep)
    keep = keep[:max(1, n)]
    keep = np.concatenate([keep[:1], keep[1:][w[keep[1:]] >= mp]])
    keep.sort()
    c = np.cumsum(w[keep])
    return int(keep[np.searchsorted(c, float(u) * c[-1], side="right")]) if float(u) * c[-1] < c[-1] else int(
        keep[np.nonzero(w[keep])[0][-1]])


def f32(v):
    return float(np.float32(v))


@pytest.mark.parametrize("dtype", ["float32", "float16", "bfloat16"])
@pytest.mark.parametrize("V", [1, 2, 31, 1000, 32000, 50257, 128256])
def test_rows_sample(cuda, dtype, V):
    torch = cuda
    rng = np.random.default_rng(V)
    B = 40
    x = torch.from_numpy((rng.standard_normal((B, V)) * rng.uniform(0.2, 6, (B, 1))).astype(np.float32)).cuda().to(
        getattr(torch, dtype))
    par = dict(temperature=rng.choice([0.0, 0.3, 0.8, 1.0, 2.5], B), top_k=rng.choice([0, 1, 2, 40, V, V + 9, -3], B),
               top_p=rng.choice([1.0, 0.95, 0.5, 0.01, 0.0, 2.0], B), min_p=rng.choice([0.0, 0.0, 0.05, 0.9, 1.0], B))
    u = rng.random(B).astype(np.float32)
    u[:3] = [0.0, np.nextafter(np.float32(1), np.float32(0)), 0.5]
    dev = {n: torch.tensor(a, dtype=torch.int32 if n == "top_k" else torch.float32, device="cuda")
           for n, a in par.items()}
    got = ops.rows_sample(x, torch.from_numpy(u).cuda(), **dev).cpu().numpy()
    xs = x.float().cpu().numpy()
    want = [sample_ref(xs[r].copy(), u[r], f32(par["temperature"][r]), int(par["top_k"][r]), f32(par["top_p"][r]),
                       f32(par["min_p"][r])) for r in range(B)]
    np.testing.assert_array_equal(got, want)


def test_rows_sample_ties_masks_and_infinities(cuda):
    torch = cuda
    inf, nan = float("inf"), float("nan")
    V = 300
    rows, want = [], []

    def add(x, token, u=0.0, T=1.0, k=0, p=1.0, mp=0.0):
        rows.append((x, u, T, k, p, mp))
        want.append(token)

    flat = np.zeros(V, np.float32)
    add(flat, 0, u=0.0)
    add(flat, 150, u=0.5)                     # cumulative mass 151/300 is the first above 1/2
    add(flat, 9, u=0.999, k=10)               # ties: the lowest indices are the first ten
    add(flat, 37, u=0.999, p=0.125)           # 38 of 300 words reach an eighth of the mass
    add(flat, 4, u=0.9, k=10, p=0.5)          # five of the ten
    mask = np.full(V, -inf, np.float32)
    add(mask, -1)
    add(np.full(V, nan, np.float32), -1, T=0.0)
    one = mask.copy()
    one[77] = -1e30
    add(one, 77, u=0.7)
    add(one, 77, T=0.0)
    lowest = np.full(V, np.finfo(np.float32).min, np.float32)
    lowest[5] = 0.0
    add(lowest, 5, u=0.9999)
    add(np.full(V, np.finfo(np.float32).min, np.float32), 150, u=0.5)  # all at the type's lowest value
    holes = flat.copy()
    holes[::2] = nan
    add(holes, 1, u=0.0)
    add(holes, 151, u=0.5)                    # the 76th of 150 words
    big = flat.copy()
    big[[10, 20]] = inf
    add(big, 10, u=0.3)
    add(big, 20, u=0.6)
    add(big, 10, T=0.0)
    signed = flat.copy()
    signed[::3] = -0.0                        # the two zeros are one value
    add(signed, 4, u=0.9, k=5)
    add(flat, 0, u=0.9, p=0.0)
    add(flat, 0, u=-1.0)
    add(flat, 299, u=2.0)                     # a number outside [0, 1): the nearest word
    add(flat, 299, u=0.999, T=inf)
    add(flat, 0, u=0.9, T=-1.0)
    B = len(rows)
    x = torch.from_numpy(np.stack([r[0] for r in rows])).cuda()
    col = lambda i, dt: torch.tensor([r[i] for r in rows], dtype=dt, device="cuda")  # noqa: E731
    args = dict(temperature=col(2, torch.float32), top_k=col(3, torch.int32), top_p=col(4, torch.float32),
                min_p=col(5, torch.float32))
    got = ops.rows_sample(x, col(1, torch.float32), **args)
    assert got.tolist() == want
    wide = torch.full((B, V + 13), inf, device="cuda")  # a strided view: what is beside it is not read
    wide[:, 5:5 + V] = x
    got = ops.rows_sample(wide[:, 5:5 + V], col(1, torch.float32), **args)
    assert got.tolist() == want


@pytest.mark.parametrize("V", [300, 5000, 40000])  # one CTA a row, two, eight
def test_rows_sample_min_p_above_one_keeps_the_first_word_alone(cuda, V):
    # equal maxima: no weight reaches min_p, the first word stays, with and without top_k and top_p
    torch = cuda
    x = np.full(V, -2.0, np.float32)
    ties = [V // 5, V // 3, V - 1]
    x[ties] = 1.5
    settings = [(k, p, mp) for k in (0, 2, 40, V - 1) for p in (1.0, 0.9, 0.0) for mp in (1.0, 1.5, math.inf)]
    B = len(settings)
    u = np.full(B, 0.999, np.float32)
    got = ops.rows_sample(torch.from_numpy(np.tile(x, (B, 1))).cuda(), torch.from_numpy(u).cuda(),
                          top_k=torch.tensor([s[0] for s in settings], dtype=torch.int32, device="cuda"),
                          top_p=torch.tensor([s[1] for s in settings], device="cuda"),
                          min_p=torch.tensor([s[2] for s in settings], device="cuda"))
    want = [sample_ref(x.copy(), u[r], 1.0, k, f32(p), f32(mp)) for r, (k, p, mp) in enumerate(settings)]
    assert got.tolist() == want
    assert all(t == ties[0] for t, (_, _, mp) in zip(want, settings) if mp > 1.0)


def test_rows_sample_greedy_is_rows_argmax_and_defaults(cuda):
    torch = cuda
    x = rand(torch, 9, 32000, dt=torch.float32, seed=4).mul_(4).round_()  # many equal maxima
    u = torch.rand(9, device="cuda")
    keys = torch.zeros(9, dtype=torch.int64, device="cuda")
    ops.rows_argmax(x, keys)
    got = ops.rows_sample(x, u, temperature=torch.zeros(9, device="cuda"))
    assert torch.equal(got.long(), ops.key_index(keys))
    got = ops.rows_sample(x, u)
    xs = x.cpu().numpy()
    assert got.tolist() == [sample_ref(xs[r].copy(), u[r].item(), 1.0, 0, 1.0, 0.0) for r in range(9)]


def test_rows_sample_borders_at_the_edge_of_a_part(cuda):
    # The bin that holds a border is divided in 512 parts.  Words whose part is another one when (m - x) 32 / T - bin
    # is rounded once, not twice: with each the last that top_p keeps, it has to be found all the same.
    torch = cuda
    rng = np.random.default_rng(11)
    T = np.float32(1.1)
    scale = np.float32(np.float32(32.0) / T)
    v = -rng.uniform(0.05, 15.0, 200000).astype(np.float32)
    twice = (-v) * scale
    b = twice.astype(np.int64)
    once = (-v.astype(np.float64) * np.float64(scale) - b).astype(np.float32)
    part = lambda t: np.clip((t * np.float32(512)).astype(np.int64), 0, 511)  # noqa: E731
    v = v[part(twice - b.astype(np.float32)) != part(once)][:600]
    assert len(v) == 600
    x = np.stack([np.zeros_like(v), v, v - 5, v - 6], 1)
    w = np.exp(x.astype(np.float64) / np.float64(T))
    p = ((1 + w[:, 1] / 2) / w.sum(1)).astype(np.float32)  # half way through the second word
    for u, token in ((0.99999994, 1), (0.0, 0)):
        for _ in range(3):
            tokens = torch.full((600,), -77, dtype=torch.int32, device="cuda")
            ops.rows_sample(torch.from_numpy(x).cuda(), torch.full((600,), u, device="cuda"),
                            temperature=torch.full((600,), float(T), device="cuda"), top_p=torch.from_numpy(p).cuda(),
                            tokens=tokens)
            assert (tokens == token).all(), f"{int((tokens != token).sum())} of 600"


def test_rows_sample_full_batches_give_the_definitions_tokens(cuda):
    # large rows with settings of their own, beside each other: the borders lie anywhere
    torch = cuda
    B, V = 128, 128256
    r = torch.arange(B, device="cuda")
    for seed in range(12):
        g = torch.Generator(device="cuda").manual_seed(1000 + seed)
        x = torch.randn(B, V, generator=g, device="cuda") * 2.0
        x += 6.0 * (torch.rand(B, V, generator=g, device="cuda") < 40.0 / V) * torch.randn(
            B, V, generator=g, device="cuda").abs()
        u = torch.rand(B, generator=g, device="cuda")
        T = torch.where(r % 5 == 0, 0.0, 0.7 + 0.1 * (r % 7))
        k = torch.where(r % 3 == 1, 50 + 40 * r, 0).int()
        p = torch.where(r % 4 == 3, 1.0, 0.5 + 0.004 * (r % 120))
        mp = torch.where(r % 6 == 1, 0.001, 0.0)
        # the definition in 64 bits
        v, order = torch.sort(x.double(), dim=-1, descending=True, stable=True)
        w = torch.exp((v - v[:, :1]) / T.double().masked_fill(T == 0, 1.0)[:, None])
        w = w * (torch.arange(V, device="cuda") < torch.where(k > 0, k, V)[:, None])
        keep = (w.cumsum(-1) - w < p.double()[:, None] * w.sum(-1, keepdim=True)) | (p >= 1)[:, None]
        keep &= w >= mp.double()[:, None]
        keep[:, 0] = True
        w = torch.zeros_like(w).scatter_(1, order, w * keep)
        cum = w.cumsum(-1)
        want = (cum > u.double()[:, None] * cum[:, -1:]).int().argmax(-1)
        want = torch.where(T == 0, order[:, 0], want).int()
        for _ in range(4):
            tokens = torch.full((B,), -77, dtype=torch.int32, device="cuda")
            ops.rows_sample(x, u, temperature=T, top_k=k, top_p=p, min_p=mp, tokens=tokens)
            assert torch.equal(tokens, want), (seed, (tokens != want).nonzero().flatten().tolist())


def test_rows_sample_frequencies(cuda):
    # 20000 evenly spaced numbers over one row: every word comes up as often as its probability says, to one
    torch = cuda
    V, N = 50, 20000
    x = rand(torch, 1, V, dt=torch.float32, seed=8).expand(N, V).contiguous()
    u = ((torch.arange(N, device="cuda").double() + 0.5) / N).float()
    got = torch.bincount(ops.rows_sample(x, u).long(), minlength=V).double()
    want = torch.softmax(x[0].double(), 0) * N
    assert (got - want).abs().max() <= 2.0


# ------------------------------------------------------------------ streams, graphs, the operators together
def test_side_stream_and_graph_replay(cuda):
    torch = cuda
    nh, nkv, hd, B, page = 8, 2, 128, 3, 16
    lens = [40, 17, 90]
    k = [rand(torch, n, nkv, hd, dt=torch.float16, seed=i) for i, n in enumerate(lens)]
    kp, vp, table = make_pages(torch, k, k, page)
    rope = torch.from_numpy(D.rope_table(256, hd, 10000.0)).cuda()
    x = rand(torch, B, (nh + 2 * nkv) * hd, dt=torch.float32, seed=5)
    kv = torch.tensor(lens, dtype=torch.int32, device="cuda")
    logits = rand(torch, B, 1000, dt=torch.float32, seed=6)
    u = torch.rand(B, device="cuda")
    cu = torch.tensor([0, 1, 2, 3], dtype=torch.int32, device="cuda")

    def step(stream=None):
        q = ops.rope_append(x, rope, kv, table, kp, vp, nh, stream=stream)
        a = ops.attention_paged(q, kp, vp, table, kv, stream=stream)
        b = ops.attention_prompt(q, kp, vp, cu, kv_len=kv, page_table=table, stream=stream)
        return q, a, b, ops.rows_sample(logits, u, top_k=cu[1:], stream=stream)

    want = [t.clone() for t in step()]
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    got = step(side)
    side.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    graphs = []
    for _ in range(2):  # two graphs at once, replayed in turn and on two streams
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            res = step()
        graphs.append((g, res))
    for _ in range(2):
        for g, _ in graphs:
            g.replay()
    torch.cuda.synchronize()
    for _, res in graphs:
        assert all(torch.equal(a, b) for a, b in zip(res, want))
    # other contents in the same buffers: nothing was kept from the capture
    x.mul_(-0.5)
    kv.copy_(torch.tensor([39, 3, 88], dtype=torch.int32))
    logits.neg_()
    want = [t.clone() for t in step()]
    for (g, _), s in zip(graphs, (torch.cuda.Stream(), torch.cuda.Stream())):
        s.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(s):
            g.replay()
    torch.cuda.synchronize()
    for _, res in graphs:
        assert all(torch.equal(a, b) for a, b in zip(res, want))


def test_prompts_of_different_lengths_then_sampled_decode(cuda):
    """A two-layer model served as a user would: ragged prompts in one pass into a paged cache, then sampled
    tokens step by step.  Every attention is held to the 64-bit one over a dense record of the rotated keys
    and values, every token to the sampling's definition, and the logits to the lockstep decoder's."""
    torch = cuda
    from asmllm_b200 import batch_decode as BD

    shape = D.LlamaShape(n_layers=2, dim=512, n_heads=4, n_kv_heads=2, head_dim=128, ffn=1536, vocab=1000)
    ctx, page, n_new = 64, 16, 5
    sh = D.shard_plan(shape, 1, 0)
    W = D.make_weights(shape, sh, 3, native.FMT_Q4_0, torch.device("cuda"))
    rng = np.random.default_rng(1)
    prompts = [rng.integers(0, shape.vocab, n) for n in (7, 1, 19)]
    B = len(prompts)
    nh, nkv, hd = shape.n_heads, shape.n_kv_heads, shape.head_dim
    rope = torch.from_numpy(D.rope_table(ctx, hd, shape.theta)).cuda()
    pools = [[torch.full((B * 4, page, nkv, hd), float("nan"), dtype=torch.float16, device="cuda") for _ in "kv"]
             for _ in range(shape.n_layers)]
    table = torch.randperm(B * 4, generator=torch.Generator().manual_seed(0)).view(B, 4).int().cuda()

    record = [[[] for _ in range(B)] for _ in range(shape.n_layers)]  # per layer and sequence: (keys, values) so far

    def check_attention(li, qkv, q, got, starts, first):
        """The attention of one layer against 64 bits; starts: row offsets, first: the first position of each."""
        x = qkv.view(-1, nh + 2 * nkv, hd)
        for s in range(B):
            a, b = starts[s], starts[s + 1]
            p = torch.arange(first[s], first[s] + b - a, device="cuda")
            c, d = rope[p, None, :, 0], rope[p, None, :, 1]
            z = x[a:b, :nh + nkv].unflatten(-1, (hd // 2, 2))
            z = torch.stack([z[..., 0] * c - z[..., 1] * d, z[..., 0] * d + z[..., 1] * c], -1).flatten(-2).half()
            assert torch.equal(q[a:b], z[:, :nh])
            record[li][s].append((z[:, nh:], x[a:b, nh + nkv:].half()))
            k, v = (torch.cat([r[i] for r in record[li][s]]) for i in (0, 1))
            want, pv, serr = exact_attention(torch, q[a:b], k, v, hd ** -0.5, first[s])
            n = k.shape[0]
            close(torch, got[a:b], want, pv, serr, n, prompt_weight(torch, torch.float16, n), torch.float16)

    def forward(ids, cu, kv_len, last):
        """Logits of rows `last` of the packed token ids."""
        starts = cu.tolist() if cu is not None else list(range(B + 1))
        first = [int(kv_len[s]) - (starts[s + 1] - starts[s]) for s in range(B)]
        x = W["embed"][ids].contiguous()
        T = x.shape[0]
        delta = None
        for li, L in enumerate(W["layers"]):
            t = torch.empty(ops.act_tiles_bytes(T, shape.dim), dtype=torch.uint8, device="cuda")
            ops.rows_norm_tiles(x, t, L["attn_norm"], shape.eps, delta=delta)
            qkv = ops.gemm_tiles(native.FMT_Q4_0, *L["wqkv"], t, T)
            k, v = pools[li]
            q = ops.rope_append(qkv, rope, kv_len, table, k, v, nh, cu_q=cu)
            if cu is None:
                a = ops.attention_paged(q, k, v, table, kv_len, out_dtype=torch.float32)
            else:
                a = ops.attention_prompt(q, k, v, cu, kv_len=kv_len, page_table=table, out_dtype=torch.float32)
            check_attention(li, qkv, q, a, starts, first)
            o = ops.gemm(native.FMT_Q4_0, *L["wo"], a.view(T, nh * hd))
            ops.rows_norm_tiles(x, t, L["ffn_norm"], shape.eps, delta=o)
            gu = ops.gemm_tiles(native.FMT_Q4_0, *L["wgu"], t, T)
            th = torch.empty(ops.act_tiles_bytes(T, shape.ffn), dtype=torch.uint8, device="cuda")
            ops.rows_swiglu_tiles(gu, th)
            delta = ops.gemm_tiles(native.FMT_Q4_0, *L["wdown"], th, T)
        t = torch.empty(ops.act_tiles_bytes(T, shape.dim), dtype=torch.uint8, device="cuda")
        ops.rows_norm_tiles(x, t, W["final_norm"], shape.eps, delta=delta)
        return ops.gemm_tiles(native.FMT_Q4_0, *W["lm_head"], t, T)[last]

    lens = [len(p) for p in prompts]
    cu = torch.tensor(np.concatenate([[0], np.cumsum(lens)]), dtype=torch.int32, device="cuda")
    kv = torch.tensor(lens, dtype=torch.int32, device="cuda")
    ids = torch.from_numpy(np.concatenate(prompts)).cuda()
    temperature = torch.tensor([0.0, 0.8, 1.0], device="cuda")
    top_k = torch.tensor([0, 20, 0], dtype=torch.int32, device="cuda")
    top_p = torch.tensor([1.0, 1.0, 0.9], device="cuda")
    numbers = torch.rand(n_new, B, generator=torch.Generator().manual_seed(2)).cuda()
    steps, tokens = [], []
    logits = forward(ids, cu, kv, cu[1:].long() - 1)
    for i in range(n_new):
        steps.append(logits.clone())
        tok = ops.rows_sample(logits, numbers[i], temperature=temperature, top_k=top_k, top_p=top_p)
        tokens.append(tok)
        kv += 1
        logits = forward(tok.long(), None, kv, slice(None))
    tokens = torch.stack(tokens, 1).cpu().numpy()
    for i in range(n_new):
        for s in range(B):
            assert tokens[s, i] == sample_ref(steps[i][s].cpu().numpy(), numbers[i, s].item(), temperature[s].item(),
                                              int(top_k[s]), top_p[s].item(), 0.0)
    for s in range(B):  # the lockstep decoder, teacher-forced with the same tokens
        forced = np.concatenate([prompts[s], tokens[s]])
        dec = BD.BatchDecoder(shape, 1, ctx=ctx, weights=W)
        dec.reset(forced[None])
        for i in range(len(forced) - 1):
            dec.step()
            j = i - (len(prompts[s]) - 1)
            if j >= 0:
                a, b = steps[j][s].cpu().numpy(), dec.logits[0].cpu().numpy()
                # The lockstep decoder keeps q in fp32; the rounding to fp16 here tips Q8_0 quants by one
                # step, at most 1/127 of the block's largest value for each of its 32: sqrt(32)/127 of the
                # vector's norm, at each of the nine quantised vectors (four a layer and the lm_head's).
                # A wrong position, page or mask gives about 1.
                assert np.linalg.norm(a - b) <= 9 * math.sqrt(32) / 127 * np.linalg.norm(b)
        dec.close()
