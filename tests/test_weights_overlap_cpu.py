"""key_weights' refusal of an out that reaches into what the kernel still reads (no GPU: nothing is launched)."""
import pytest
import torch

from long_vita_amd import _lib, ops

B, N, ROWS, HQ, HKV, D = 2, 3, 20, 4, 2, 64


@pytest.fixture
def launches(monkeypatch):
    real, calls = _lib.lib(), []

    class Lib:
        def __getattr__(self, name):
            return getattr(real, name)

        def lv_key_weights(self, *args):
            calls.append(args)
            return 0
    lib = Lib()
    monkeypatch.setattr(ops._lib, "lib", lambda: lib)
    monkeypatch.setattr(ops, "_stream", lambda: 0)
    monkeypatch.setattr(ops, "_require_gpu", lambda *tensors: None)
    return calls


def inputs():
    return dict(q=torch.zeros(B, N, HQ, D, dtype=torch.bfloat16), k=torch.zeros(B, ROWS, HKV, D, dtype=torch.bfloat16), lse=torch.zeros(B, N, HQ),
                weight=torch.zeros(B, HKV, ROWS), cache_lens=torch.tensor([5, 9], dtype=torch.int32), parents=torch.tensor([-1, 0, 1], dtype=torch.int32),
                row_weight=torch.ones(B, N), alibi_slopes=torch.zeros(HQ))


def test_allowed(launches):
    a = inputs()
    assert ops.key_weights(**a, out=a["weight"]) is a["weight"]
    both = torch.zeros(B, 2, HKV, ROWS)                       # interleaved with the old weights
    a["weight"] = both[:, 0]
    ops.key_weights(**a, out=both[:, 1])
    ops.key_weights(**a)
    assert len(launches) == 3


@pytest.mark.parametrize("name", ["q", "k", "lse", "cache_lens", "parents", "row_weight", "alibi_slopes"])
@pytest.mark.parametrize("in_place", [False, True])
def test_out_holds_an_input(launches, name, in_place):
    a = inputs()
    buf = torch.zeros(1 << 14)
    t = a[name]
    a[name] = buf.view(t.dtype)[8:8 + t.numel()].view(t.shape)
    out = buf[:B * HKV * ROWS].view(B, HKV, ROWS)
    if in_place:
        a["weight"] = out
    with pytest.raises(_lib.LvAttnError, match="overlap"):
        ops.key_weights(**a, out=out)
    assert not launches


@pytest.mark.parametrize("name,bad", [("parents", [-1, 0, 1]), ("alibi_slopes", [0.0] * HQ)])
def test_types_are_looked_at_first(launches, name, bad):
    a = inputs()
    a[name] = bad
    with pytest.raises(_lib.LvAttnError, match=name):
        ops.key_weights(**a, out=torch.zeros(B, HKV, ROWS))
