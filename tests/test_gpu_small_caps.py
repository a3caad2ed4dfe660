"""Caps far below the scores, down to what fp32 cannot hold: every score is (all but) 0, the softmax is uniform and the scores pass on
no gradient, also in rows whose products are exactly 0.  Tolerances: test_gpu_caps."""
import math

import pytest
import torch

from tests import test_gpu_evict as evict_tests
from tests import test_gpu_score as score_tests
from tests import test_gpu_tree as tree_tests

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("scale", [None, 1e6])
@pytest.mark.parametrize("cap", [1e-3, 1e-30, 2.0 ** -126, 1e-40, 1e-60])
def test_small_caps(cap, scale):
    from long_vita_amd import ops
    T, hq, hkv, d = 200, 4, 2, 64
    q, k, v, do = score_tests.make(T, hq, hkv, d, 5)
    q[::3] = 0                                        # products of exactly 0
    leaves = [t.cuda().requires_grad_(True) for t in (q, k, v)]
    out, lse = ops.score_attention(*leaves, [0, T], scale, softcap=cap)
    dq, dk, dv = torch.autograd.grad(out, leaves, do.cuda())
    want = score_tests.ref(q, k, v, [0, T], d ** -0.5 if scale is None else scale, True, cap, do=do)
    assert score_tests.rel(out, want[0]) <= score_tests.REL_TOL
    assert float((lse.double().cpu() - want[1]).abs().max()) <= score_tests.LSE_TOL
    assert score_tests.rel(dv, want[4]) <= score_tests.GRAD_TOL and bool(torch.isfinite(dq).all()) and bool(torch.isfinite(dk).all())
    # a row of zeros stands where the tanh is steepest: dq = scale sum P (dP - delta) K as without a cap
    assert score_tests.rel(dq[::3], want[2][::3]) <= score_tests.GRAD_TOL
    L = torch.tensor([150], dtype=torch.int32, device="cuda")
    qt, kt, vt = q[None, :7], k[None], v[None]
    o, ls = ops.tree_attention(qt.cuda(), kt.cuda(), vt.cuda(), L, scale, softcap=cap, return_lse=True)
    wo, wl = tree_tests.ref(qt, kt, vt, [150], d ** -0.5 if scale is None else scale, None, cap)
    assert score_tests.rel(o, wo) <= 2.0 ** -7 and float((ls.double().cpu() - wl).abs().max()) <= score_tests.LSE_TOL
    w = ops.key_weights(qt.cuda(), kt.cuda(), ls, torch.zeros(1, hkv, T, device="cuda"), L, scale, softcap=cap)
    ww = evict_tests.ref_weights(qt, kt, [150], d ** -0.5 if scale is None else scale, ls.cpu(), torch.zeros(1, hkv, T), None, cap)
    assert float((w.double().cpu() - ww).abs().max()) <= evict_tests.W_TOL * float(ww.max())


def test_refused():
    from long_vita_amd import _lib, ops
    q, k, v, _ = (t.cuda() for t in score_tests.make(8, 2, 1, 64, 1))
    for cap in (0.0, -1e-60, 1e30, math.inf, math.nan):
        with pytest.raises(_lib.LvAttnError, match="softcap"):
            ops.score_attention(q, k, v, [0, 8], softcap=cap)
