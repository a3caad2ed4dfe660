"""Distance bias over a cache of more than 2^24 keys, where fp32 no longer tells neighbouring positions apart: the distances are small,
and so exact.  Tolerance: test_gpu_evict's."""
import math

import pytest
import torch

from tests.test_gpu_evict import W_TOL

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("n,tree", [(1, False), (40, True), (260, False)])
def test_positions_past_fp32(n, tree):
    from long_vita_amd import ops
    length, hq, d, last = (1 << 24) + 1001, 1, 64, 90
    rows = length + n
    g = torch.Generator(device="cuda").manual_seed(n)
    k = torch.randn(1, rows, 1, d, generator=g, device="cuda", dtype=torch.bfloat16)
    q = torch.randn(1, n, hq, d, generator=g, device="cuda", dtype=torch.bfloat16)
    slopes = torch.tensor([0.5], device="cuda")
    depth = torch.arange(n) // 2 if tree else torch.arange(n)       # pairs of siblings, the next pair under the first of them
    par = torch.tensor([-1, -1] + [2 * (i // 2) - 2 for i in range(2, n)], dtype=torch.int32) if tree else None
    see = torch.zeros(n, n, dtype=torch.bool)
    for i in range(n):
        at = i
        while at >= 0:
            see[i, at] = True
            at = (int(par[at]) if tree else at - 1)
    L = torch.tensor([length], dtype=torch.int32, device="cuda")
    kw = dict(parents=None if par is None else par.cuda(), alibi_slopes=slopes)
    pos = torch.cat([torch.arange(length - last, length), length + depth])
    x = (q[0, :, 0].double().cpu() @ k[0, length - last:, 0].double().cpu().T) * d ** -0.5
    t = (x - 0.5 * (length + depth[:, None] - pos[None]).abs()).masked_fill(~torch.cat([torch.ones(n, last, dtype=torch.bool), see], 1), -math.inf)
    lse = torch.logsumexp(t, 1)                                     # (what lies farther back weighs less than e^-45)
    if n <= 256:
        _, got_lse = ops.tree_attention(q, k, k, L, return_lse=True, **kw)
        assert float((got_lse[0, :, 0].double().cpu() - lse).abs().max()) <= W_TOL
    w = ops.key_weights(q, k, lse.float().cuda()[None, :, None], torch.zeros(1, 1, rows, device="cuda"), L, **kw)
    want = torch.exp(t - lse.float().double()[:, None]).sum(0)
    assert float((w[0, 0, length - last:].double().cpu() - want).abs().max()) <= W_TOL * float(want.max())
    assert float(w[0, 0, :length - last].double().sum()) <= 1e-15 * n
