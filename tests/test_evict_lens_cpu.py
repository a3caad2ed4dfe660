"""The copy that evict_cache makes of strided lengths lives until the launch (no GPU: the library call is played)."""
import ctypes

import torch

from long_vita_amd import _lib, ops


def test_copy_of_strided_lengths_lives(monkeypatch):
    real, seen = _lib.lib(), []

    class Lib:
        def __getattr__(self, name):
            return getattr(real, name)

        def lv_evict_index(self, weight, lens, *args):
            new = [torch.full((300,), -7, dtype=torch.int32) for _ in range(8)]      # what another thread may be given by now
            seen.append((list((ctypes.c_int32 * 300).from_address(lens)), new))
            return 0

        def lv_evict_take(self, *args):
            return 0
    lib = Lib()
    monkeypatch.setattr(ops._lib, "lib", lambda: lib)
    monkeypatch.setattr(ops, "_stream", lambda: 0)
    monkeypatch.setattr(ops, "_require_gpu", lambda *tensors: None)
    b = 300
    lens = torch.arange(2 * b, dtype=torch.int32)[::2]
    k = torch.zeros(b, 4, 1, 64, dtype=torch.bfloat16)
    ops.evict_cache(k, torch.zeros_like(k), torch.zeros(b, 1, 4), lens, 2)
    assert seen[0][0] == lens.tolist()
