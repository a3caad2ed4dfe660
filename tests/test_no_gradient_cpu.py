"""Derivatives that an operator does not have are refused, not dropped: tensors that require a gradient, tangents of forward mode (no GPU:
the refusal comes before the tensors' device matters)."""
import pytest
import torch
from torch.autograd import forward_ad

from long_vita_amd import _lib, ops


def calls():
    bf = dict(dtype=torch.bfloat16)
    q, k, v = torch.zeros(2, 3, 4, 64, **bf), torch.zeros(2, 20, 2, 64, **bf), torch.zeros(2, 20, 2, 64, **bf)
    lens, w, lse = torch.tensor([5, 9], dtype=torch.int32), torch.zeros(2, 2, 20), torch.zeros(2, 3, 4)
    path, cnt = torch.zeros(2, 3, dtype=torch.int32), torch.zeros(2, dtype=torch.int32)
    packed = dict(q=torch.zeros(8, 4, 64, **bf), k=torch.zeros(8, 2, 64, **bf), v=torch.zeros(8, 2, 64, **bf), cu_seqlens=[0, 8])
    return {
        "score": (ops.score_attention, packed, "qkv", False),
        "tree": (ops.tree_attention, dict(q=q, k=k, v=v, cache_lens=lens), "qkv", True),
        "accept": (ops.tree_accept, dict(k=k, v=v, cache_lens=lens, path=path, n_accept=cnt, weight=w), ["k", "v", "weight"], True),
        "weights": (ops.key_weights, dict(q=q, k=k, lse=lse, weight=w, cache_lens=lens, row_weight=torch.ones(2, 3)), ["q", "k", "lse", "weight", "row_weight"], True),
        "evict": (ops.evict_cache, dict(k=k, v=v, weight=w, cache_lens=lens, keep=4), ["k", "v", "weight"], True),
    }


CASES = [(name, arg) for name, (_, _, args, _) in calls().items() for arg in args]


@pytest.mark.parametrize("name,arg", CASES)
def test_tangents(name, arg):
    fn, args, _, _ = calls()[name]
    with forward_ad.dual_level():
        args[arg] = forward_ad.make_dual(args[arg], torch.ones_like(args[arg]))
        for grad in (True, False):
            with torch.set_grad_enabled(grad), pytest.raises(_lib.LvAttnError, match="forward-mode"):
                fn(**args)


@pytest.mark.parametrize("name,arg", [c for c in CASES if calls()[c[0]][3]])
def test_requires_grad(name, arg):
    fn, args, _, _ = calls()[name]
    args[arg].requires_grad_(True)
    with pytest.raises(_lib.LvAttnError, match="no gradient"):
        fn(**args)
    with torch.no_grad(), pytest.raises(_lib.LvAttnError, match="GPU"):       # allowed, as far as the device
        fn(**args)


def test_slopes_with_tangents(monkeypatch):
    monkeypatch.setattr(ops, "_require_gpu", lambda *tensors: None)
    for name in ("score", "tree", "weights"):
        fn, args, _, _ = calls()[name]
        with forward_ad.dual_level():
            with pytest.raises(_lib.LvAttnError, match="forward-mode"):
                fn(**args, alibi_slopes=forward_ad.make_dual(torch.zeros(4), torch.ones(4)))


def test_a_level_without_tangents_is_fine():
    for name, (fn, args, _, _) in calls().items():
        with forward_ad.dual_level(), pytest.raises(_lib.LvAttnError, match="GPU"):
            fn(**args)
