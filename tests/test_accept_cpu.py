"""tree_accept's refusals that need no GPU (nothing is launched)."""
import pytest
import torch

from long_vita_amd import _lib, ops

B, ROWS, N, HKV, D = 2, 20, 5, 3, 64


@pytest.fixture
def launches(monkeypatch):
    real, calls = _lib.lib(), []

    class Lib:
        def __getattr__(self, name):
            if name.startswith("lv_tree_accept"):
                return lambda *args: calls.append(args) or 0
            return getattr(real, name)
    lib = Lib()
    monkeypatch.setattr(ops._lib, "lib", lambda: lib)
    monkeypatch.setattr(ops, "_stream", lambda: 0)
    monkeypatch.setattr(ops, "_require_gpu", lambda *tensors: None)
    return calls


def call(weight):
    k, v = (torch.zeros(B, ROWS, HKV, D, dtype=torch.bfloat16) for _ in range(2))
    return ops.tree_accept(k, v, torch.tensor([3, 4], dtype=torch.int32), torch.zeros(B, N, dtype=torch.int32), torch.tensor([1, 2], dtype=torch.int32), weight)


@pytest.mark.parametrize("weight", [torch.zeros(1, HKV, ROWS).expand(B, HKV, ROWS), torch.zeros(B, 1, ROWS).expand(B, HKV, ROWS)], ids=["batch", "heads"])
def test_expanded_weight(launches, weight):
    with pytest.raises(_lib.LvAttnError, match="expanded"):
        call(weight)
    assert not launches


def test_weight_with_strides_of_its_own(launches):
    call(torch.zeros(B, HKV + 2, ROWS + 7)[:, 1:HKV + 1, 3:ROWS + 3])
    call(None)
    assert len(launches) == 2
