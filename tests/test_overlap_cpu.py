"""Whether two strided views share memory, against the bytes themselves."""
import random

import pytest
import torch

from long_vita_amd.ops import _overlap


def touched(t, base):
    """Every byte of t, counted from `base`."""
    at = torch.tensor([t.data_ptr() - base])
    for n, s in zip(t.shape, t.stride()):
        at = (at[:, None] + torch.arange(n)[None] * s * t.element_size()).reshape(-1)
    return set((at[:, None] + torch.arange(t.element_size())[None]).reshape(-1).tolist())


def view(rng, store):
    size = {torch.uint8: 1, torch.bfloat16: 2, torch.float32: 4}
    dtype = rng.choice(list(size))
    flat = store.view(dtype)
    while True:
        shape = [rng.choice([1, 1, 2, 3, 5]) for _ in range(rng.randint(1, 4))]
        stride = [rng.choice([0, 1, 2, 3, 8, 20, 64, 160]) for _ in shape]
        need = 1 + sum((n - 1) * s for n, s in zip(shape, stride))
        if need <= flat.numel():
            return torch.as_strided(flat, shape, stride, rng.randint(0, flat.numel() - need))


@pytest.mark.parametrize("seed", range(6))
def test_random_views(seed):
    rng = random.Random(seed)
    store = torch.zeros(1024, dtype=torch.uint8)
    seen = [0, 0]
    for _ in range(500):
        a, b = view(rng, store), view(rng, store)
        want = bool(touched(a, store.data_ptr()) & touched(b, store.data_ptr()))
        assert _overlap(a, b) == want == _overlap(b, a)
        seen[want] += 1
    assert min(seen) > 10                  # both answers occur


def test_interleaved_layouts():
    kv = torch.zeros(3, 50, 2, 4, 64, dtype=torch.bfloat16)
    k, v = kv[:, :, 0], kv[:, :, 1]
    assert not _overlap(k, v) and _overlap(k, kv) and _overlap(k, k[1:, 7:]) and not _overlap(k[:, :, :2], k[:, :, 2:])
    assert not _overlap(k[:, :20], k[:, 20:]) and _overlap(k[:, :21], k[:, 20:])
    heads = torch.zeros(2, 5, 14, 64, dtype=torch.bfloat16)
    assert not _overlap(heads[:, :, :4], heads[:, :, 4:]) and _overlap(heads[:, :, :5], heads[:, :, 4:])
    w = torch.zeros(1 << 20)
    assert not _overlap(w[::2], w[1::2]) and _overlap(w[::2], w[4::6])
    assert not _overlap(w[:0], w) and not _overlap(torch.zeros(8), torch.zeros(8))
