"""Caps far above the scores, around them and far below, in every operator that takes one, against float64 on the CPU.

Tolerances.  A capped score is off by less than 4e-7 of its own magnitude (caps above 64) or 1.4e-7 of the cap (up to 64, below
1e-5), on top of the product's own fp32 sum, whose terms add up to a few times the largest score: 2e-5 + 1e-6 max |t| on a log-sum-exp
and relative on a weight.  Outputs and gradients round to bf16 as without a cap (2^-7 and 2^-6 of the largest value); a relative error
of 1e-6 max |t| on every P, with |t| up to 400, is 4e-4 beside that."""
import math

import pytest
import torch

from tests import test_gpu_evict as evict_tests
from tests import test_gpu_score as score_tests
from tests import test_gpu_tree as tree_tests

pytestmark = pytest.mark.gpu


def t_max(q, k, scale, cap):
    """Bound of |t| from the largest rows."""
    x = float(q.double().norm(dim=-1).max() * k.double().norm(dim=-1).max()) * scale
    return min(x, cap)


# cap, std of q (scores have the same): caps beside which the scores vanish, caps that the scores cross, the border between the forms
CAPS = [(64.0, 2.0), (64.5, 2.0), (64.5, 40.0), (200.0, 120.0), (1e3, 2.0), (1e4, 4.0), (1e5, 2.0), (1e7, 2.0), (1e9, 2.0), (9e29, 2.0)]


@pytest.mark.parametrize("split", [(0, 0), (128, 64)], ids=["whole", "cut"])
@pytest.mark.parametrize("hq,hkv,d,alibi,causal", [(5, 1, 128, False, True), (4, 2, 64, True, True), (4, 2, 128, True, False), (70, 1, 64, False, True)])
@pytest.mark.parametrize("cap,std", CAPS)
def test_score_attention(cap, std, hq, hkv, d, alibi, causal, split):
    from long_vita_amd import ops
    cu, scale = [0, 70, 293], d ** -0.5
    q, k, v, do = score_tests.make(cu[-1], hq, hkv, d, 17, std)
    slopes = score_tests.slopes_of(hq) if alibi else None
    want = score_tests.ref(q, k, v, cu, scale, causal, cap, slopes, do=do)
    ops.set_split_override(*split)
    try:
        leaves = [t.cuda().requires_grad_(True) for t in (q, k, v)]
        out, lse = ops.score_attention(*leaves, cu, None, causal, softcap=cap, alibi_slopes=None if slopes is None else slopes.cuda())
        grads = torch.autograd.grad(out, leaves, do.cuda())
    finally:
        ops.set_split_override(None, None)
    assert score_tests.rel(out, want[0]) <= score_tests.REL_TOL
    assert float((lse.double().cpu() - want[1]).abs().max()) <= 2e-5 + 1e-6 * t_max(q, k, scale, cap)
    for g, w in zip(grads, want[2:]):
        assert score_tests.rel(g, w) <= score_tests.GRAD_TOL


@pytest.mark.parametrize("cap", [1e5, 1e9, 9e29])
def test_far_cap_is_no_cap(cap):
    """Beside these caps the scores are what they are: out, lse and the gradients of the operator without one."""
    from long_vita_amd import ops
    q, k, v, do = (t.cuda() for t in score_tests.make(600, 5, 1, 128, 3))
    res = []
    for c in (cap, None):
        leaves = [t.clone().requires_grad_(True) for t in (q, k, v)]
        out, lse = ops.score_attention(*leaves, [0, 600], softcap=c)
        res.append([out.detach(), lse, *torch.autograd.grad(out, leaves, do)])
    # cap tanh(x / cap) = x - x^3 / (3 cap^2): with |x| < 30 less than 1e-6 away
    assert float((res[0][1] - res[1][1]).abs().max()) <= 4e-5
    for a, b in zip(res[0], res[1]):
        assert score_tests.rel(a, b.double().cpu()) <= 2.0 ** -7


@pytest.mark.parametrize("n,hq,hkv,d", [(1, 5, 1, 128), (9, 4, 1, 64), (12, 5, 1, 128), (25, 5, 1, 128), (70, 4, 1, 64), (260, 1, 1, 128)])
@pytest.mark.parametrize("alibi", [False, True], ids=["plain", "alibi"])
@pytest.mark.parametrize("cap,std", [CAPS[i] for i in (0, 2, 4, 6, 9)])
def test_tree_attention_and_key_weights(cap, std, alibi, n, hq, hkv, d):
    from long_vita_amd import ops
    lens, scale = [200, 31], d ** -0.5
    rows = max(lens) + n + 10
    q, k, v = tree_tests.make(2, n, rows, hq, hkv, d, 5, lens)
    q = (q.float() * (std / 2)).to(torch.bfloat16)
    par = tree_tests.random_parents(2, n, 5) if 1 < n <= 256 else None
    slopes = score_tests.slopes_of(hq) if alibi else None
    lists = None if par is None else par.tolist()
    kw = dict(parents=None if par is None else par.cuda(), softcap=cap, alibi_slopes=None if slopes is None else slopes.cuda())
    L = torch.tensor(lens, dtype=torch.int32, device="cuda")
    want, want_lse = tree_tests.ref(q, k, v, lens, scale, lists, cap, slopes)
    tol = 2e-5 + 1e-6 * t_max(q, k.nan_to_num(), scale, cap)
    if n <= 256:
        out, lse = ops.tree_attention(q.cuda(), k.cuda(), v.cuda(), L, return_lse=True, **kw)
        assert score_tests.rel(out, want) <= 2.0 ** -7
        assert float((lse.double().cpu() - want_lse).abs().max()) <= tol
    lse = want_lse.float()
    w = torch.rand(2, hkv, rows, generator=torch.Generator().manual_seed(2))
    for rho in (None, torch.rand(2, n, generator=torch.Generator().manual_seed(3))):
        got = ops.key_weights(q.cuda(), k.cuda(), lse.cuda(), w.cuda(), L, row_weight=None if rho is None else rho.cuda(), **kw)
        ref = evict_tests.ref_weights(q, k, lens, scale, lse, w, lists, cap, slopes, rho)
        # (t and lse, rounded to fp32, each enter the exponent: 2^-24 max |t| more for lse)
        assert float((got.double().cpu() - ref).abs().max()) <= 2 * tol * float(ref.max())
