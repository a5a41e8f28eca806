"""The serving operators' allocation: torch's quick but private way is used only where it does what is expected of it."""
from __future__ import annotations

import pytest

from asmllm_b200 import ops

torch = pytest.importorskip("torch")


def raising(error):
    def f(*args):
        raise error
    return f


@pytest.mark.parametrize("other", [None, raising(TypeError("takes 4 arguments")), raising(RuntimeError("no device")),
                                   lambda *a: torch.empty(2, 3, dtype=torch.int8), lambda *a: None, "gone"])
def test_another_release_of_torch_falls_back(monkeypatch, other):
    guards = pytest.importorskip("torch._C._dynamo.guards")
    monkeypatch.setattr(ops, "_ready", False)
    monkeypatch.setattr(ops, "_cuda_empty", None)
    if other == "gone":
        monkeypatch.delattr(guards, "_empty_strided_cuda", raising=False)
    else:
        monkeypatch.setattr(guards, "_empty_strided_cuda", other, raising=False)
    ops._setup()
    assert ops._ready and ops._cuda_empty is None


def test_host_tensors_are_refused_before_anything_is_allocated(monkeypatch):
    monkeypatch.setattr(ops, "_ready", False)
    with pytest.raises(TypeError, match="CUDA tensor"):
        ops.rows_adjust(torch.zeros(2, 3))
    assert not ops._ready
