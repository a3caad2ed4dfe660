"""evict_cache's refusal of output buffers that meet each other or the caches (no GPU: nothing is launched)."""
import pytest
import torch

from long_vita_amd import _lib, ops

B, ROWS, KEEP, HKV, D = 2, 20, 8, 2, 64


@pytest.fixture
def launches(monkeypatch):
    real, calls = _lib.lib(), []

    class Lib:
        def __getattr__(self, name):
            return getattr(real, name)

        def lv_evict_index(self, *args):
            calls.append("index")
            return 0

        def lv_evict_take(self, *args):
            calls.append("take")
            return 0
    lib = Lib()
    monkeypatch.setattr(ops._lib, "lib", lambda: lib)
    monkeypatch.setattr(ops, "_stream", lambda: 0)
    monkeypatch.setattr(ops, "_require_gpu", lambda *tensors: None)
    return calls


def call(out, kv=None):
    kv = torch.zeros(B, ROWS, 2, HKV, D, dtype=torch.bfloat16) if kv is None else kv
    return ops.evict_cache(kv[:, :, 0], kv[:, :, 1], torch.zeros(B, HKV, ROWS), torch.tensor([20, 9], dtype=torch.int32), KEEP, out=out)


def test_interleaved_outputs_are_taken(launches):
    new = torch.zeros(B, KEEP, 2, HKV, D, dtype=torch.bfloat16)
    call((new[:, :, 0], new[:, :, 1], torch.zeros(B, HKV, KEEP)))
    assert launches == ["index", "take"]


def test_outputs_interleaved_with_the_caches_are_taken(launches):
    buf = torch.zeros(B, ROWS, 4, HKV, D, dtype=torch.bfloat16)
    call((buf[:, :, 2], buf[:, :, 3], torch.zeros(B, HKV, KEEP)), buf)
    assert launches == ["index", "take"]


size = B * KEEP * HKV * D


@pytest.mark.parametrize("name,make", [
    ("same_start", lambda buf: (buf[:size].view(B, KEEP, HKV, D), buf[:size].view(B, KEEP, HKV, D), torch.zeros(B, HKV, KEEP))),
    ("one_row_on", lambda buf: (buf[:size].view(B, KEEP, HKV, D), buf[HKV * D:HKV * D + size].view(B, KEEP, HKV, D), torch.zeros(B, HKV, KEEP))),
    ("weights_in_k", lambda buf: (buf[:size].view(B, KEEP, HKV, D), buf[size:2 * size].view(B, KEEP, HKV, D), buf[64:64 + 2 * B * HKV * KEEP].view(torch.float32).view(B, HKV, KEEP))),
    ("weights_in_v", lambda buf: (buf[:size].view(B, KEEP, HKV, D), buf[size:2 * size].view(B, KEEP, HKV, D),
                                  buf[2 * size - 4:2 * size - 4 + 2 * B * HKV * KEEP].view(torch.float32).view(B, HKV, KEEP)))])
def test_outputs_that_meet(launches, name, make):
    with pytest.raises(_lib.LvAttnError, match="overlap"):
        call(make(torch.zeros(4 * size, dtype=torch.bfloat16)))
    assert not launches
