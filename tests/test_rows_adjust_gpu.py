"""ops.rows_adjust where a batch's arrays have no entries, and with padded rows."""
from __future__ import annotations

import time

import pytest

from asmllm_b200 import ops
from test_serving_gpu import rand
from test_serving_q8_gpu import check_adjust, clean_error_word, exact_adjust, ints  # noqa: F401

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("B", [1, 3])
@pytest.mark.parametrize("V", [33, 40960])
def test_a_step_where_no_row_has_a_bias_or_a_token(cuda, B, V):
    torch = cuda
    x = rand(torch, B, V, dt=torch.float32, seed=1)
    words, bias = torch.empty(B, 0, dtype=torch.int32, device="cuda"), torch.empty(B, 0, device="cuda")
    assert torch.equal(ops.rows_adjust(x, bias_tokens=words, bias=bias), x)
    assert torch.equal(ops.rows_adjust(x, tokens=words, n_tokens=ints(torch, *[0] * B), bias_tokens=words, bias=bias), x)
    wide = torch.zeros(B, 5, device="cuda")[:, :0]  # strides of another array
    tokens = (torch.rand(B, 50, generator=torch.Generator().manual_seed(6)) * V).int().cuda()
    rep = torch.full((B,), 1.5, device="cuda")
    got = ops.rows_adjust(x, tokens=tokens, repetition=rep, bias_tokens=wide.int(), bias=wide)
    want, size = exact_adjust(torch, x, tokens, [50] * B, [0] * B, rep, 0 * rep, 0 * rep, None, None, None)
    check_adjust(torch, got, want, size)
    with pytest.raises(ValueError, match="equal, dense"):
        ops.rows_adjust(x, bias_tokens=words, bias=torch.zeros(B, 1, device="cuda"))


def test_rows_with_padding_are_looked_at_together(cuda):
    """What lies between the rows of out may hold an input; and a call's time does not grow with the rows there."""
    torch = cuda
    B, V = 300, 1000
    wide = torch.zeros(B, V + 32, device="cuda")
    x = wide[:, :V]
    x.copy_(rand(torch, B, V, dt=torch.float32, seed=1))
    allowed = wide.view(torch.int32)[:, V:V + 32]  # in the padding of the rows it masks
    allowed.copy_(torch.randint(-2 ** 31, 2 ** 31, (B, 32), generator=torch.Generator().manual_seed(2)).int())
    bits = (allowed[:, :, None] >> torch.arange(32, device="cuda") & 1).flatten(1)[:, :V]
    want = torch.where(bits == 1, x, float("-inf"))
    assert torch.equal(ops.rows_adjust(x, allowed=allowed), want)
    keep = allowed.clone()
    ops.rows_adjust(x, allowed=allowed, out=x)
    assert torch.equal(x, want) and torch.equal(allowed, keep)
    for first in (V - 1, 1):  # one word of a row is a word of the mask
        with pytest.raises(ops.AsmError, match="overlaps"):
            ops.rows_adjust(x, allowed=wide.view(torch.int32)[:, first:first + 32], out=x)
    with pytest.raises(ops.AsmError, match="overlaps"):
        ops.rows_adjust(torch.zeros(1, V, device="cuda"), out=x[:1], tokens=wide.view(torch.int32)[:1, :4])

    def host(rows, padding):
        y = torch.zeros(rows, 64 + padding, device="cuda")[:, :64]
        best = 1.0
        for _ in range(20):
            torch.cuda.synchronize()
            begin = time.perf_counter()
            ops.rows_adjust(y, out=y)
            best = min(best, time.perf_counter() - begin)
        return best

    assert host(60000, 8) < 5 * host(60000, 0) + 50e-6


def test_calls_without_torchs_quick_allocation(cuda, monkeypatch):
    torch = cuda
    x = rand(torch, 2, 100, dt=torch.float32, seed=1)
    monkeypatch.setattr(ops, "_ready", False)
    monkeypatch.setattr(ops, "_cuda_empty", None)
    monkeypatch.setattr(torch._C._dynamo.guards, "_empty_strided_cuda", None)
    got = ops.rows_adjust(x)
    assert ops._ready and ops._cuda_empty is None
    assert torch.equal(got, x) and got.data_ptr() != x.data_ptr()
