"""Rows of ``key_weights`` whose lse is -inf (or NaN) count for nothing, whatever their row of q holds: without parents and row
weights too, in every kernel.  Tolerance: test_gpu_evict's."""
import math

import pytest
import torch

from tests import test_gpu_evict as evict_tests
from tests import test_gpu_tree as tree_tests

pytestmark = pytest.mark.gpu

# query rows per KV head: n * hq / hkv = 5, 32, 60, 125 (streamed, one to four row tiles), 140 and 255 (two passes), 257, 700 and 1,800
# (streaming the rows; in pieces)
SIZES = [([300, 40], 1, 10, 2, 128), ([300, 40], 8, 4, 1, 64), ([300, 40], 12, 5, 1, 128), ([90, 257], 25, 5, 1, 128), ([200], 35, 4, 1, 64),
         ([200, 17], 51, 5, 1, 128), ([130], 257, 1, 1, 128), ([0, 60], 140, 5, 1, 64), ([0], 360, 5, 1, 128)]


@pytest.mark.parametrize("cap,alibi", [(None, False), (30.0, True), (1e4, False)], ids=["plain", "rule", "wide"])
@pytest.mark.parametrize("lens,n,hq,hkv,d", SIZES, ids=[f"rows{s[1] * s[2] // s[3]}" for s in SIZES])
def test_lse_without_a_sum(lens, n, hq, hkv, d, cap, alibi):
    from long_vita_amd import ops
    b, rows = len(lens), max(lens) + n + 20
    q, k, v = tree_tests.make(b, n, rows, hq, hkv, d, n, lens)
    slopes = tree_tests.slopes_of(hq) if alibi else None
    _, lse = tree_tests.ref(q, k, v, lens, d ** -0.5, None, cap, slopes)
    lse = lse.float()
    g = torch.Generator().manual_seed(n)
    dead = torch.rand(b, n, hq, generator=g) < 0.1            # per token and head
    dead[:, -1], dead[0, 0] = True, True                      # the last token (its row is the one that padding repeats) and the first
    w = torch.rand(b, hkv, rows, generator=g)
    want = evict_tests.ref_weights(q, k, lens, d ** -0.5, lse.masked_fill(dead, math.inf), w, None, cap, slopes)
    junk = torch.tensor([math.nan, math.inf, -math.inf, 3e38])[torch.randint(0, 4, q.shape, generator=g)]
    q = torch.where(dead[..., None], junk, q.float()).to(torch.bfloat16)
    lse = torch.where(dead, torch.where(torch.rand(lse.shape, generator=g) < 0.3, math.nan, -math.inf), lse)
    L = torch.tensor(lens, dtype=torch.int32, device="cuda")
    kw = dict(softcap=cap, alibi_slopes=None if slopes is None else slopes.cuda())
    wg = w.cuda()
    got = ops.key_weights(q.cuda(), k.cuda(), lse.cuda(), wg, L, **kw)
    assert float((got.double().cpu() - want).abs().max()) <= evict_tests.W_TOL * float(want.max())
    assert torch.equal(ops.key_weights(q.cuda(), k.cuda(), lse.cuda(), wg, L, out=wg, **kw), got)


def test_padded_prompt():
    """A prompt behind which the buffers hold NaN: score_attention's lse there is -inf, and the weights are the prompt's own."""
    from long_vita_amd import ops
    n, T, hq, hkv, d = 200, 320, 5, 1, 128
    q, k, v = tree_tests.make(1, T, T, hq, hkv, d, 7, [0])
    q[:, n:] = math.nan
    _, lse = ops.score_attention(q[0].cuda(), k[0].cuda(), v[0].cuda(), [0, n], softcap=30.0)
    assert bool((lse[:, n:] == -math.inf).all())
    zero, w = torch.zeros(1, dtype=torch.int32, device="cuda"), torch.zeros(1, hkv, T, device="cuda")
    got = ops.key_weights(q.cuda(), k.cuda(), lse.t().contiguous()[None], w, zero, softcap=30.0)
    want = ops.key_weights(q[:, :n].cuda(), k[:, :n].cuda(), lse[:, :n].t().contiguous()[None], w[..., :n], zero, softcap=30.0)
    # the terms are the same numbers, in a different order of compensated sums: 2^-23 of a sum of at most n hq
    assert float((got[..., :n] - want).abs().max()) <= 2.0 ** -22 * float(want.max()) and not bool(got[..., n:].any())
    assert abs(float(want.double().sum()) - n * hq) <= 1e-5 * n * hq
