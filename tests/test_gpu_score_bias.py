"""The roundings on the way to score_attention's gradients cancel on average: no gradient comes out systematically short or long.

Tolerance.  c = <g, g64> / <g64, g64> - 1.  What rounds to bf16 and is shared by many elements is P (for dV) and dS (for dQ and dK) of a
(row, key) pair: an error of e_ij moves c by e_ij w_ij, where w_ij is the pair's own share of <g64, g64> / <g64, g64> = 1 (computed
below in 64 bits).  The e_ij are independent roundings to nearest, zero on average, at most 2^-8 and so 2^-8 / sqrt(3) or less in the
mean square: c has a standard deviation of sigma = 2^-8 / sqrt(3) sqrt(sum w^2), here 5.7e-5 to 7.6e-5, and stays within 4 sigma.  (The
results' own roundings, one per element, add 2^-8 / sqrt(3 * 38400) / 4 to that in the squares: nothing.)  A bound from the number of
elements alone, 8e-5, forgets that the d elements of a row share the roundings.  P rounded towards zero to 11 bits shifts c of
dK by 2^-11 / (2 ln 2) = 3.5e-4, beyond 4 sigma."""
import math

import pytest
import torch

from tests import test_gpu_score as score_tests

pytestmark = pytest.mark.gpu


def sigmas(q, k, v, do, scale, cap, slopes, lse, grads):
    q, k, v, do = (t.double() for t in (q, k, v, do))
    dq, dk, dv = grads
    n, hq = q.shape[:2]
    gap = torch.arange(n)[:, None] - torch.arange(n)[None]
    squares = [0.0, 0.0, 0.0]
    for h in range(hq):                                     # one KV head
        x = scale * q[:, h] @ k[:, 0].T
        th = torch.tanh(x / cap) if cap else None
        t = cap * th if cap else x
        if slopes is not None:
            t = t - float(slopes[h]) * gap.abs()
        P = torch.exp(t.masked_fill(gap < 0, -math.inf) - lse[h][:, None])
        dt = P * (do[:, h] @ v[:, 0].T - (do[:, h] * (P @ v[:, 0])).sum(1, keepdim=True))
        ds = scale * (dt * (1 - th * th) if cap else dt)
        for i, w in enumerate((ds * (dq[:, h] @ k[:, 0].T), ds * (q[:, h] @ dk[:, 0].T), P * (do[:, h] @ dv[:, 0].T))):
            squares[i] += float((w * w).sum())
    return [2.0 ** -8 / math.sqrt(3) * math.sqrt(s) / float((g * g).sum()) for s, g in zip(squares, grads)]


@pytest.mark.parametrize("cap,alibi,d,split", [(None, False, 128, 0), (30.0, False, 128, 0), (30.0, True, 64, 0), (None, True, 128, 128), (1e4, False, 64, 0)])
def test_mean_error(cap, alibi, d, split):
    from long_vita_amd import ops
    T, hq, hkv = 600, 4, 1
    q, k, v, do = score_tests.make(T, hq, hkv, d, 11)
    slopes = score_tests.slopes_of(hq) if alibi else None
    want = score_tests.ref(q, k, v, [0, T], d ** -0.5, True, cap, slopes, do=do)
    ops.set_split_override(split, split)
    try:
        leaves = [t.cuda().requires_grad_(True) for t in (q, k, v)]
        out, _ = ops.score_attention(*leaves, [0, T], softcap=cap, alibi_slopes=None if slopes is None else slopes.cuda())
        grads = torch.autograd.grad(out, leaves, do.cuda())
    finally:
        ops.set_split_override(None, None)
    bounds = sigmas(q, k, v, do, d ** -0.5, cap, slopes, want[1], want[2:])
    for name, g, w, s in zip(("dq", "dk", "dv"), grads, want[2:], bounds):
        c = float((g.double().cpu() * w).sum() / (w * w).sum()) - 1
        print(name, c, s)
        assert abs(c) <= 4 * s, name
