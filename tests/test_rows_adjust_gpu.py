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
