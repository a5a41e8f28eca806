"""The Q8_0 decode attention where scales of a block lie far apart or are not finite: a large scale at a position without
weight must not cost the others their bits."""
from __future__ import annotations

import math

import pytest

from asmllm_b200 import ops
from test_serving_gpu import rand
from test_serving_q8_gpu import clean_error_word, ints, make_pages8, random8, values  # noqa: F401

pytestmark = pytest.mark.gpu


def check_flat(torch, got, vals, weights, top):
    """got [heads, hd] of one sequence against the sum of weights [n] times vals [n, nkv, hd], whose scales are at most top.

    Scores of 0 have no error and all the same 2^x, so what is left, for each position: two 16-bit parts of a weight and
    of its product with a scale (2 * 2^-22), the sums of n of them (n 2^-23, truncated or rounded, with each rescaling
    exact), the sum of the weights and the division (n 2^-24 and 2^-23); a product's parts end at 2^-34 of the largest
    weight times the largest scale, times a code of up to 128."""
    n, nkv, hd = vals.shape
    rep = got.shape[0] // nkv
    want = torch.einsum("n,nhd->hd", weights, vals).repeat_interleave(rep, 0)
    size = torch.einsum("n,nhd->hd", weights, vals.abs()).repeat_interleave(rep, 0)
    tol = (2 * 2.0 ** -22 + 2 * n * 2.0 ** -23 + 2.0 ** -22) * size + n * 2.0 ** -34 * float(weights.max()) * 128 * top
    err = (got.double() - want).abs()
    assert bool((err <= tol).all()), f"worst {float((err / tol).max()):.3g} of the tolerance"


@pytest.mark.parametrize("dtype", ["float16", "bfloat16"])
@pytest.mark.parametrize("nh,nkv,hd", [(8, 1, 128), (4, 2, 64), (16, 1, 128), (20, 1, 64)])
@pytest.mark.parametrize("big", [64.0, 32768.0])
def test_large_scale_without_weight(cuda, dtype, nh, nkv, hd, big):
    """One position, first, inside or last, has a score 60 below the others' (a weight of 1e-26) and a scale of `big` in
    its second block; the others' scales there are 2^-14 to 2^-38 of it."""
    torch = cuda
    n, page = 50, 16
    g = torch.Generator(device="cuda").manual_seed(1)
    for at in (0, 17, n - 1):
        for ratio in (-14, -15, -20, -23, -27, -31, -38):
            d = torch.tensor(1.37 * big * 2.0 ** ratio, dtype=torch.float16).item()
            if d == 0.0:
                continue
            kc, kd = torch.zeros(n, nkv, hd, dtype=torch.int8, device="cuda"), torch.ones(n, nkv, hd // 32, device="cuda").half()
            kc[at] = -1
            vc = torch.randint(60, 128, (n, nkv, hd), generator=g, device="cuda").to(torch.int8)
            vd = torch.full((n, nkv, hd // 32), d, dtype=torch.float16, device="cuda")
            vd[at, :, 1] = big
            k, v, ks, vs, table = make_pages8(torch, [(kc, kd, vc, vd)], page)
            q = torch.ones(1, nh, hd, dtype=getattr(torch, dtype), device="cuda")
            got = ops.attention_paged_q8(q, k, v, ks, vs, table, ints(torch, n), scale=60.0 / hd, out_dtype=torch.float32)
            w = torch.ones(n, dtype=torch.float64, device="cuda")
            w[at] = math.exp(-60.0)
            check_flat(torch, got[0], values(vc, vd), w / w.sum(), big)


@pytest.mark.parametrize("nh,nkv,hd", [(8, 1, 128), (16, 1, 64)])
def test_scales_over_the_whole_range_beside_a_large_one(cuda, nh, nkv, hd):
    """Scales from 2^-24 to 2^-10 at positions of equal weight and 2^15 at ten without: zeros, signs and all blocks."""
    torch = cuda
    n, page = 1000, 32
    g = torch.Generator(device="cuda").manual_seed(2)
    kc, kd = torch.zeros(n, nkv, hd, dtype=torch.int8, device="cuda"), torch.ones(n, nkv, hd // 32, device="cuda").half()
    vc = torch.randint(60, 128, (n, nkv, hd), generator=g, device="cuda").to(torch.int8)
    vd = torch.exp2(-24 + 14 * torch.rand(n, nkv, hd // 32, generator=g, device="cuda")).half()
    vd[::7], vd[1::7] = 0.0, -vd[1::7]
    at = torch.randperm(n, generator=torch.Generator().manual_seed(3))[:10].cuda()
    kc[at] = -1
    vd[at] = 2.0 ** 15
    vd[at[:5], :, 0] = 2.0 ** -12  # the first block has fewer
    k, v, ks, vs, table = make_pages8(torch, [(kc, kd, vc, vd)], page)
    q = torch.ones(1, nh, hd, dtype=torch.float16, device="cuda")
    got = ops.attention_paged_q8(q, k, v, ks, vs, table, ints(torch, n), scale=60.0 / hd, out_dtype=torch.float32)
    w = torch.ones(n, dtype=torch.float64, device="cuda")
    w[at] = math.exp(-60.0)
    check_flat(torch, got[0], values(vc, vd), w / w.sum(), 2.0 ** 15)


@pytest.mark.parametrize("nh,nkv,hd,dtype", [(8, 2, 128, "float16"), (40, 2, 64, "bfloat16")])
@pytest.mark.parametrize("code", [-1, 0, 1])
def test_key_scale_that_is_not_finite_shows_in_its_rows_alone(cuda, nh, nkv, hd, dtype, code):
    """A key block with an infinite scale holds infinities of its codes' signs and NaN: no score, whatever their sum's sign."""
    torch = cuda
    n = 40
    for bad in (float("inf"), float("nan")):
        for at, block in ((0, 0), (20, 1), (n - 1, hd // 32 - 1)):
            dense = [list(random8(torch, n, nkv, hd, s)) for s in range(3)]
            q = rand(torch, 3, nh, hd, dt=getattr(torch, dtype), seed=5).abs()
            lens = ints(torch, n, n, n)
            args = make_pages8(torch, dense, 16)
            want = ops.attention_paged_q8(q, *args, lens, out_dtype=torch.float32)
            dense[1][0][at, 1, 32 * block:32 * block + 32] = code
            dense[1][1][at, 1, block] = bad
            got = ops.attention_paged_q8(q, *make_pages8(torch, dense, 16), lens, out_dtype=torch.float32)
            hit = torch.zeros_like(got, dtype=torch.bool)
            hit[1, nh // 2:] = True
            assert torch.isnan(got[hit]).all()
            assert torch.equal(got[~hit], want[~hit])


def test_key_beyond_a_scale_of_16_bits_is_nan(cuda):
    """Finite keys past what an fp16 scale holds (about 8.3e6): their row has no answer, instead of one without them."""
    torch = cuda
    x = rand(torch, 1, 3 * 64, dt=torch.float32, seed=3).abs()
    x[0, 64:96] = -1e7
    rope = torch.zeros(32, 32, 2, device="cuda")
    rope[..., 0] = 1.0
    k, v, ks, vs, table = make_pages8(torch, [random8(torch, 20, 1, 64, 0)], 16)
    q = ops.rope_append_q8(x, rope, ints(torch, 20), table, k, v, ks, vs, 1)
    assert torch.isnan(ops.attention_paged_q8(q, k, v, ks, vs, table, ints(torch, 20))).all()


def test_a_short_neighbour_does_not_slow_a_long_sequence(cuda):
    """Parts of one unit are joined one after the other: their number does not grow with the rest of the batch (1.4 times
    the time where it did)."""
    torch = cuda
    n, nh, nkv, hd, page = 131071, 8, 1, 128, 64
    pages = -(-n // page) + 1
    k, v = (torch.randint(-127, 128, (pages, page, nkv, hd), device="cuda").to(torch.int8) for _ in "kv")
    ks, vs = (torch.full((pages, nkv, page, hd // 32), 0.01, dtype=torch.float16, device="cuda") for _ in "kv")
    table = torch.stack([torch.arange(pages), torch.arange(pages).flip(0)]).int().cuda()
    q = rand(torch, 2, nh, hd, dt=torch.float16, seed=1)

    def least(batch, lens):
        call = lambda: ops.attention_paged_q8(q[:batch], k, v, ks, vs, table[:batch], lens)  # noqa: E731
        call()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            for _ in range(10):
                call()
        times = []
        for _ in range(20):
            begin, end = (torch.cuda.Event(enable_timing=True) for _ in "be")
            begin.record()
            graph.replay()
            end.record()
            end.synchronize()
            times.append(begin.elapsed_time(end))
        return min(times)

    assert least(2, ints(torch, n, 1)) < 1.2 * least(1, ints(torch, n))
