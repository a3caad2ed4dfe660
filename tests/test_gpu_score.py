"""Attention with a rule on its scores (tanh cap, distance bias, prefix, band) against a float64 computation on the CPU:
outputs, log-sum-exps, gradients, run-to-run equality, whole and cut sweeps, graph replay.

Tolerances.  The kernels round P (and dS) to bf16 once before the second product and the result once more: two half steps of
2^-8 relative to the largest magnitude of the row / tensor, plus the fp32 sums; 2^-7 on max-norm relative error covers both with
no room for a wrong key (one key in a thousand with equal weight would show as 1e-3 of the value, a missing row entirely)."""
import math

import numpy as np
import pytest
import torch

from long_vita_amd import _lib

pytestmark = pytest.mark.gpu

REL_TOL = 2.0 ** -7        # out: two half steps of bf16
GRAD_TOL = 2.0 ** -6       # gradients: P' / dS and delta (from the rounded out) add two more half steps
LSE_TOL = 2e-5             # fp32 sums of fp32 exponentials, |lse| up to ~60


def ref(q, k, v, cu, scale, causal=True, cap=None, slopes=None, prefix=None, band=None, do=None):
    """float64, one segment and head at a time, from the definition."""
    q, k, v = (t.double() for t in (q, k, v))
    T, hq, d = q.shape
    g = hq // k.shape[1]
    out, lse = torch.zeros_like(q), torch.full((hq, T), -math.inf, dtype=torch.float64)
    dq, dk, dv = torch.zeros_like(q), torch.zeros_like(k), torch.zeros_like(v)
    for s, (a, z) in enumerate(zip(cu[:-1], cu[1:])):
        n = z - a
        if n == 0:
            continue
        i, j = torch.arange(n)[:, None], torch.arange(n)[None, :]
        see = torch.ones(n, n, dtype=torch.bool)
        if causal:
            see = (j <= i) | (j < (prefix[s] if prefix is not None else 0))
        if band is not None:
            see &= j >= i - band
        for h in range(hq):
            K, V, Q = k[a:z, h // g], v[a:z, h // g], q[a:z, h]
            x = scale * Q @ K.T
            th = torch.tanh(x / cap) if cap else None
            t = cap * th if cap else x
            if slopes is not None:
                t = t - float(slopes[h]) * (i - j).abs()
            t = t.masked_fill(~see, -math.inf)
            L = torch.logsumexp(t, 1)
            P = torch.exp(t - L[:, None])
            O = P @ V
            out[a:z, h], lse[h, a:z] = O, L
            if do is not None:
                G = do[a:z, h].double()
                dt = P * (G @ V.T - (G * O).sum(1, keepdim=True))
                dx = scale * (dt * (1 - th * th) if cap else dt)
                dq[a:z, h] = dx @ K
                dk[a:z, h // g] += dx.T @ Q
                dv[a:z, h // g] += P.T @ G
    return (out, lse) if do is None else (out, lse, dq, dk, dv)


def rel(got, want):
    return float((got.detach().double().cpu() - want).abs().max() / want.abs().max().clamp_min(1e-30))


def make(T, hq, hkv, d, seed, q_std=2.0):
    g = torch.Generator().manual_seed(seed)
    q = (torch.randn(T, hq, d, generator=g) * q_std).to(torch.bfloat16)
    k, v = (torch.randn(T, hkv, d, generator=g).to(torch.bfloat16) for _ in range(2))
    do = torch.randn(T, hq, d, generator=g).to(torch.bfloat16)
    return q, k, v, do


def slopes_of(hq):
    return torch.tensor([2.0 ** (-8.0 * (h + 1) / hq) for h in range(hq)], dtype=torch.float32)


CASES = [
    # name, cu, hq, hkv, d, causal, cap, alibi, prefix, band
    ("one_token", [0, 1], 5, 1, 128, True, 30.0, True, None, None),
    ("tiny_segments", [0, 1, 3, 3, 36, 65], 4, 2, 64, True, 20.0, False, None, None),
    ("cap_odd", [0, 257, 700], 5, 1, 128, True, 50.0, False, None, None),
    ("cap_dense_d64", [0, 321], 4, 4, 64, False, 30.0, False, None, None),
    ("cap_dense_d128", [0, 130, 400], 6, 2, 128, False, 30.0, False, None, None),
    ("alibi_long", [0, 1111], 8, 2, 128, True, None, True, None, None),
    ("alibi_dense", [0, 300], 4, 1, 128, False, None, True, None, None),
    ("alibi_d64", [0, 90, 640], 12, 2, 64, True, None, True, None, None),
    ("both", [0, 513, 600], 10, 2, 128, True, 25.0, True, None, None),
    ("both_dense_d64", [0, 513], 4, 2, 64, False, 25.0, True, None, None),
    ("prefix", [0, 500, 900, 1000], 5, 1, 128, True, None, False, [256, 0, 100], None),
    ("prefix_edges", [0, 256, 512, 800], 4, 2, 64, True, None, False, [1, 255, 129], None),
    ("prefix_long", [0, 1300], 5, 1, 128, True, 40.0, True, [700], None),
    ("band_cap", [0, 700, 1000], 4, 2, 128, True, 30.0, False, None, 100),
    ("band_zero", [0, 300], 4, 2, 64, True, 30.0, False, None, 0),
    ("band_alibi", [0, 900], 5, 1, 64, True, None, True, None, 257),
    ("gap_before_and_behind", [7, 300, 333], 5, 1, 128, True, 30.0, True, None, None),
    ("group_64", [0, 200], 64, 1, 64, True, None, True, None, None),
]


@pytest.mark.parametrize("split", [(0, 0), (256, 96), (None, None)], ids=["whole", "cut", "planned"])
@pytest.mark.parametrize("name,cu,hq,hkv,d,causal,cap,alibi,prefix,band", CASES, ids=[c[0] for c in CASES])
def test_forward_backward(name, cu, hq, hkv, d, causal, cap, alibi, prefix, band, split):
    from long_vita_amd import ops
    T = cu[-1] + (9 if name.startswith("gap") else 0)
    q, k, v, do = make(T, hq, hkv, d, len(name) + T)
    slopes = slopes_of(hq) if alibi else None
    scale = 1.0 / math.sqrt(d)
    want = ref(q, k, v, cu, scale, causal, cap, slopes, prefix, band, do)
    ops.set_split_override(*split)
    ops._poison_workspaces = True
    try:
        runs = []
        for _ in range(2):
            qc, kc, vc = (t.cuda().requires_grad_(True) for t in (q, k, v))
            out, lse = ops.score_attention(qc, kc, vc, cu, None, causal, softcap=cap, alibi_slopes=None if slopes is None else slopes.cuda(),
                                           prefix_lens=prefix, band=band)
            out.backward(do.cuda())
            torch.cuda.synchronize()
            runs.append((out, lse, qc.grad, kc.grad, vc.grad))
    finally:
        ops.set_split_override(None, None)
        ops._poison_workspaces = False
    for a, b in zip(*runs):
        assert torch.equal(a, b)                     # bitwise reproducible
    out, lse, dq, dk, dv = runs[0]
    assert rel(out, want[0]) <= REL_TOL
    finite = torch.isfinite(want[1])
    assert torch.equal(torch.isfinite(lse.cpu()), finite)
    assert float((lse.double().cpu() - want[1])[finite].abs().max()) <= LSE_TOL
    if not finite.all():
        outside = torch.ones(T, dtype=torch.bool)
        outside[cu[0]:cu[-1]] = False
        for t in (out, dq, dk, dv):
            assert not t.detach().cpu()[outside].any()
    for got, w in zip((dq, dk, dv), want[2:]):
        if float(w.abs().max()) < 1e-12:             # one visible key: P = 1 and dP = delta, the scores have no gradient
            assert float(got.abs().max()) <= 2.0 ** -6
        else:
            assert rel(got, w) <= GRAD_TOL


def test_plain_rule_matches_plain_attention():
    """No cap, no bias, no prefix: the results of varlen_attention on the same kernels, within the rounding of one product."""
    from long_vita_amd import ops
    q, k, v, do = (t.cuda() for t in make(900, 5, 1, 128, 3))
    cu = [0, 400, 900]
    a, la = ops.score_attention(q, k, v, cu)
    b, lb = ops.varlen_attention(q, k, v, cu)
    assert float((a.float() - b.float()).abs().max()) <= 2.0 ** -7 * float(b.abs().max())
    assert float((la - lb).abs().max()) <= LSE_TOL


def test_gradient_against_differences():
    """d/dx of sum(out * w) by central differences of the float64 definition, along random directions."""
    from long_vita_amd import ops
    cu, cap = [0, 33, 97], 5.0
    q, k, v, do = make(97, 4, 2, 64, 11)
    slopes = slopes_of(4)
    leaves = [t.cuda().requires_grad_(True) for t in (q, k, v)]
    out, _ = ops.score_attention(*leaves, cu, softcap=cap, alibi_slopes=slopes.cuda())
    grads = torch.autograd.grad(out, leaves, do.cuda())
    g = torch.Generator().manual_seed(5)
    for n in range(3):
        base = [q.double(), k.double(), v.double()]
        direction = torch.randn(base[n].shape, generator=g, dtype=torch.float64)
        eps = 1e-5
        val = []
        for sgn in (1, -1):
            x = list(base)
            x[n] = x[n] + sgn * eps * direction
            val.append((ref(*x, cu, 0.125, True, cap, slopes)[0] * do.double()).sum())
        want = float((val[0] - val[1]) / (2 * eps))
        got = float((grads[n].double().cpu() * direction).sum())
        # each gradient element is off by at most GRAD_TOL of the largest; random signs: a few standard deviations of the sum
        bound = 4 * GRAD_TOL * float(grads[n].abs().max()) * math.sqrt(direction.numel()) / 4
        assert abs(got - want) <= bound


def test_strided_views_and_offsets():
    from long_vita_amd import ops
    T, hq, hkv, d = 300, 4, 2, 128
    q, k, v, do = make(T, hq, hkv, d, 21)
    fused = torch.zeros(T, hq + 2 * hkv, d + 8, dtype=torch.bfloat16)
    fused[:, :hq, :d], fused[:, hq:hq + hkv, :d], fused[:, hq + hkv:, :d] = q, k, v
    f = fused.cuda()
    views = [f[:, :hq, :d], f[:, hq:hq + hkv, :d], f[:, hq + hkv:, :d]]
    a, la = ops.score_attention(*views, [0, T], softcap=20.0)
    b, lb = ops.score_attention(q.cuda(), k.cuda(), v.cuda(), [0, T], softcap=20.0)
    assert torch.equal(a, b) and torch.equal(la, lb)
    odd = torch.zeros(T * hq * d + 1, dtype=torch.bfloat16, device="cuda")[1:].view(T, hq, d)   # 2-byte alignment: copied
    odd.copy_(q)
    qt = q.transpose(0, 1).contiguous().cuda().transpose(0, 1)                                     # head-major
    for alt in (odd, qt):
        c, _ = ops.score_attention(alt, k.cuda(), v.cuda(), [0, T], softcap=20.0)
        assert torch.equal(c, b)
    # gradients through the views, dout expanded (stride 0)
    leaf = f.detach().requires_grad_(True)
    out, _ = ops.score_attention(leaf[:, :hq, :d], leaf[:, hq:hq + hkv, :d], leaf[:, hq + hkv:, :d], [0, T], softcap=20.0)
    out.sum().backward()
    want = ref(q, k, v, [0, T], 1 / math.sqrt(d), True, 20.0, do=torch.ones(T, hq, d))
    assert rel(leaf.grad[:, :hq, :d], want[2]) <= GRAD_TOL
    assert rel(leaf.grad[:, hq + hkv:, :d], want[4]) <= GRAD_TOL


def test_saturated_cap_and_large_bias():
    """Scores far beyond the cap (tanh = +-1 to the last bit) and slopes that hide all but the nearest keys."""
    from long_vita_amd import ops
    q, k, v, do = make(260, 4, 2, 128, 31, q_std=200.0)
    cu = [0, 260]
    sl = torch.tensor([0.0, 1.0, 50.0, 1000.0])
    want = ref(q, k, v, cu, 1.0, True, 10.0, sl)
    out, lse = ops.score_attention(q.cuda(), k.cuda(), v.cuda(), cu, 1.0, softcap=10.0, alibi_slopes=sl.cuda())
    assert rel(out, want[0]) <= REL_TOL
    # a product q.k is a sum of 128 terms of size ~200 whose partial sums reach 8192 (3.5 standard deviations of 200 sqrt(128));
    # it is formed in at least 8 fp32 additions (16 terms per matrix instruction), each off by up to half a step there, 2^-12:
    # 8 * 2^-12 on a score that the tanh does not flatten, and lse moves by no more than the scores do
    assert float((lse.double().cpu() - want[1]).abs().max()) <= 8 * 2.0 ** -12


@pytest.mark.parametrize("scale", [0.0, -0.11, 1e-25, 1e-6])
@pytest.mark.parametrize("cap,alibi", [(None, True), (20.0, False), (20.0, True)])
def test_scales(scale, cap, alibi):
    """A scale of 0, below 0 or next to nothing is a scale like any other."""
    from long_vita_amd import ops
    q, k, v, do = make(330, 4, 2, 64, 51)
    cu, slopes = [0, 70, 330], slopes_of(4) if alibi else None
    want = ref(q, k, v, cu, scale, True, cap, slopes, do=do)
    leaves = [t.cuda().requires_grad_(True) for t in (q, k, v)]
    out, lse = ops.score_attention(*leaves, cu, scale, softcap=cap, alibi_slopes=None if slopes is None else slopes.cuda())
    out.backward(do.cuda())
    assert rel(out, want[0]) <= REL_TOL and float((lse.double().cpu() - want[1]).abs().max()) <= LSE_TOL
    for t, w in zip(leaves, want[2:]):
        # (a scale of 1e-25 leaves gradients of 1e-25: still a part of the largest one)
        assert rel(t.grad, w) <= GRAD_TOL if float(w.abs().max()) > 0 else not t.grad.any()


def test_broadcast_inputs():
    """Heads and rows that are one tensor seen several times: their gradients add up."""
    from long_vita_amd import ops
    T, hq, hkv, d = 140, 4, 2, 64
    q, k, v, do = make(T, hq, hkv, d, 61)
    q[:], k[:, 1] = q[:1], k[:, 0]
    want = ref(q, k, v, [0, T], 0.2, True, 15.0, do=do)
    q1, k1, v1 = (t.cuda().requires_grad_(True) for t in (q[:1], k[:, :1], v))
    out, _ = ops.score_attention(q1.expand(T, hq, d), k1.expand(T, hkv, d), v1, [0, T], 0.2, softcap=15.0)
    out.backward(do.cuda())
    assert rel(out, want[0]) <= REL_TOL and rel(v1.grad, want[4]) <= GRAD_TOL
    # a sum over rows (heads) of gradients that were each rounded: random signs, a few standard deviations against the largest
    assert float((q1.grad.double().cpu() - want[2].sum(0, keepdim=True)).abs().max()) <= GRAD_TOL * float(want[2].abs().max()) * math.sqrt(T)
    assert float((k1.grad.double().cpu() - want[3].sum(1, keepdim=True)).abs().max()) <= GRAD_TOL * float(want[3].abs().max()) * math.sqrt(hkv)


@pytest.mark.parametrize("piece", [0, 256])
def test_cut_off_bytes(piece):
    """Out and its cut-off byte are the result to 16 bits of mantissa.  With equal scores P is 1, exact in bf16, so the result
    is a mean of v in fp32 (row lengths up to 600: 600 * 2^-24 of |v| <= 5)."""
    from long_vita_amd import ops
    T, hq, hkv, d = 600, 2, 1, 128
    _q, k, v, do = (t.cuda() for t in make(T, hq, hkv, d, 71))
    rule = ops._ScoreRule((0, T), True, None, None, 0.0)
    ops.set_split_override(piece, piece)
    try:
        out, lse, lo, pieces, covered = ops._score_forward(torch.zeros(T, hq, d, dtype=torch.bfloat16, device="cuda"), k, v, None, rule, 0.1, True)
    finally:
        ops.set_split_override(None, None)
    assert covered and pieces[0] == piece
    want = (v.double().cumsum(0) / torch.arange(1, T + 1, device="cuda", dtype=torch.float64)[:, None, None]).expand(T, hq, d)
    b = lo.to(torch.int32)
    bits = ((out.contiguous().view(torch.int16).to(torch.int32) & 0xffff) - (b >> 7)) * 65536 + b * 256 + 128
    full = bits.view(torch.float32).double()
    assert float((full - want).abs().max()) <= 2.0 ** -16 * float(want.abs().max()) + 600 * 2.0 ** -24 * 5
    assert float((full - out.double()).abs().max()) <= 2.0 ** -8 * float(want.abs().max())


@pytest.mark.parametrize("piece", [0, 128])
def test_rows_past_32_bit_offsets(piece):
    """A segment whose rows lie behind 2^31 elements (and 2^32 bytes) gives what it gives at the front, bit for bit."""
    from long_vita_amd import ops
    n, T, hq, hkv, d = 300, 430000, 40, 8, 128
    q, k, v, do = (t.cuda() for t in make(n, hq, hkv, d, 81))
    big = [torch.zeros(T, t.shape[1], d, dtype=torch.bfloat16, device="cuda") for t in (q, k, v, do)]
    for b, t in zip(big, (q, k, v, do)):
        b[-n:] = t
    assert big[0].numel() > 2 ** 31
    ops.set_split_override(piece, piece)
    try:
        res = []
        for (x, y, z, w), cu in (((q, k, v, do), [0, n]), (big, [T - n, T])):
            leaves = [t.requires_grad_(True) for t in (x, y, z)]
            out, lse = ops.score_attention(*leaves, cu, softcap=30.0)
            res.append((out, lse, torch.autograd.grad(out, leaves, w)))
    finally:
        ops.set_split_override(None, None)
    (o1, l1, g1), (o2, l2, g2) = res
    assert torch.equal(o2[-n:], o1) and torch.equal(l2[:, -n:], l1)
    for a, b in zip(g1, g2):
        assert torch.equal(b[-n:], a) and not b[:1000].any()


def test_other_stream_and_graph():
    from long_vita_amd import ops
    q, k, v, do = (t.cuda() for t in make(700, 5, 1, 128, 41))
    sl = slopes_of(5).cuda()
    leaves = [t.clone().requires_grad_(True) for t in (q, k, v)]

    def step():
        out, lse = ops.score_attention(*leaves, [0, 300, 700], softcap=30.0, alibi_slopes=sl)
        return (out, lse, *torch.autograd.grad(out, leaves, do))
    eager = [t.detach().clone() for t in step()]     # (no graph of the leaves lives on into the capture)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for _ in range(2):
            other = step()
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(eager, other))
    del other
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        captured = step()
    for it in range(3):
        for t in captured:
            t.detach().zero_()
        with torch.no_grad():
            leaves[0].copy_(q * (1 + it))
        graph.replay()
        torch.cuda.synchronize()
        want = step()
        assert all(torch.equal(a, b) for a, b in zip(captured, want))


def test_graph_outlives_the_table_cache():
    """A captured call keeps its work-item tables when other packings have pushed them out of the cache."""
    from long_vita_amd import ops
    q, k, v, do = (t.cuda() for t in make(500, 4, 2, 64, 43))
    leaves = [t.clone().requires_grad_(True) for t in (q, k, v)]

    def step():
        out, lse = ops.score_attention(*leaves, [0, 123, 500], softcap=30.0, prefix_lens=[50, 60])
        return (out, lse, *torch.autograd.grad(out, leaves, do))
    want = [t.detach().clone() for t in step()]
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        step()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        captured = step()
    store = dict(ops._blocks.store)
    mine = [key for key in store if key[0] == "score" and key[1][0] == (0, 123, 500)]
    assert mine and all(any(store[key] is t for t in ops._captured_tables.values()) for key in mine)
    for n in range(ops._blocks.capacity + 1):
        ops._blocks.get(("other", n), lambda: None)
    del store
    junk = [torch.full((64,), -1, dtype=torch.int32, device="cuda") for _ in range(2000)]
    for _ in range(3):
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(captured, want))
    del junk
    fresh = torch.cuda.CUDAGraph()
    with torch.cuda.graph(fresh):
        with pytest.raises(_lib.LvAttnError, match="before the capture"):
            ops.score_attention(q, k, v, [0, 77, 500])
        after = q + 1
    fresh.replay()
    torch.cuda.synchronize()
    assert torch.equal(after, q + 1)


REFUSED = [
    ("rank", lambda q, k, v: ((q[0], k, v, [0, 8]), {})),
    ("dtype", lambda q, k, v: ((q.float(), k, v, [0, 8]), {})),
    ("rows", lambda q, k, v: ((q[:7], k, v, [0, 7]), {})),
    ("past_end", lambda q, k, v: ((q, k, v, [0, 9]), {})),
    ("decreasing", lambda q, k, v: ((q, k, v, [0, 5, 4, 8]), {})),
    ("empty_cu", lambda q, k, v: ((q, k, v, []), {})),
    ("cap_zero", lambda q, k, v: ((q, k, v, [0, 8]), dict(softcap=0.0))),
    ("cap_nan", lambda q, k, v: ((q, k, v, [0, 8]), dict(softcap=float("nan")))),
    ("scale_inf", lambda q, k, v: ((q, k, v, [0, 8], float("inf")), {})),
    ("slopes_shape", lambda q, k, v: ((q, k, v, [0, 8]), dict(alibi_slopes=torch.ones(3, device=q.device)))),
    ("slopes_type", lambda q, k, v: ((q, k, v, [0, 8]), dict(alibi_slopes=torch.ones(4, device=q.device, dtype=torch.bfloat16)))),
    ("slopes_grad", lambda q, k, v: ((q, k, v, [0, 8]), dict(alibi_slopes=torch.ones(4, device=q.device, requires_grad=True)))),
    ("prefix_count", lambda q, k, v: ((q, k, v, [0, 8]), dict(prefix_lens=[1, 2]))),
    ("prefix_negative", lambda q, k, v: ((q, k, v, [0, 8]), dict(prefix_lens=[-1]))),
    ("prefix_not_causal", lambda q, k, v: ((q, k, v, [0, 8], None, False), dict(prefix_lens=[1]))),
    ("band_prefix", lambda q, k, v: ((q, k, v, [0, 8]), dict(prefix_lens=[1], band=2))),
    ("band_negative", lambda q, k, v: ((q, k, v, [0, 8]), dict(band=-1))),
    ("band_not_causal", lambda q, k, v: ((q, k, v, [0, 8], None, False), dict(band=2))),
    ("head_dim", lambda q, k, v: ((q[..., :32], k[..., :32], v[..., :32], [0, 8]), {})),
    ("heads", lambda q, k, v: ((q[:, :3], k, v, [0, 8]), {})),
    ("cpu", lambda q, k, v: ((q.cpu(), k, v, [0, 8]), {})),
    ("slopes_cpu", lambda q, k, v: ((q, k, v, [0, 8]), dict(alibi_slopes=torch.ones(4)))),
]


@pytest.mark.parametrize("name,call", REFUSED, ids=[r[0] for r in REFUSED])
def test_refusals(name, call):
    from long_vita_amd import ops
    q, k, v, _ = (t.cuda() for t in make(8, 4, 2, 64, 1))
    args, kw = call(q, k, v)
    with pytest.raises(_lib.LvAttnError):
        ops.score_attention(*args, **kw)


@pytest.mark.parametrize("layout", ["TND", "SBH", "BSH", "BNSD"])
@pytest.mark.parametrize("prefix", [[70, 3], [33, 33]])
def test_fused_op_with_a_prefix(layout, prefix):
    """The fused op's prefix mode in its layouts is score_attention on the packed rows, forward and backward, bit for bit."""
    from long_vita_amd import ops
    from long_vita_amd.fusion_attention import npu_fusion_attention
    b, s, hq, hkv, d = 2, 150, 4, 2, 64
    q, k, v, _do = (t.cuda() for t in make(b * s, hq, hkv, d, 3))
    do = torch.randn(b * s, hq, d, generator=torch.Generator().manual_seed(4)).to(torch.bfloat16).cuda()
    leaves = [t.clone().requires_grad_(True) for t in (q, k, v)]
    want, want_lse = ops.score_attention(*leaves, [0, s, 2 * s], scale=0.1, prefix_lens=prefix)
    want.backward(do)
    mine = [t.clone().requires_grad_(True) for t in (q, k, v)]
    put = {"TND": lambda x: x, "SBH": lambda x: x.reshape(b, s, -1).transpose(0, 1), "BSH": lambda x: x.reshape(b, s, -1),
           "BNSD": lambda x: x.reshape(b, s, -1, d).permute(0, 2, 1, 3)}[layout]
    back = {"TND": lambda x: x, "SBH": lambda x: x.transpose(0, 1).reshape(b * s, hq, d), "BSH": lambda x: x.reshape(b * s, hq, d),
            "BNSD": lambda x: x.permute(0, 2, 1, 3).reshape(b * s, hq, d)}[layout]
    kw = dict(actual_seq_qlen=[s, 2 * s], actual_seq_kvlen=[s, 2 * s]) if layout == "TND" else {}
    out, lse, _one = npu_fusion_attention(*(put(x) for x in mine), hq, layout, atten_mask=True, scale=0.1, sparse_mode=6, prefix=prefix, **kw)
    assert torch.equal(back(out), want)
    back(out).backward(do)
    for x, y in zip(mine, leaves):
        assert torch.equal(x.grad, y.grad)
    if layout == "SBH":
        assert torch.equal(lse.reshape(b, hq, s).transpose(0, 1).reshape(hq, b * s), want_lse)
    for bad in (dict(sparse_mode=6), dict(sparse_mode=2, prefix=prefix), dict(sparse_mode=6, prefix=[1, 2, 3])):
        with pytest.raises((NotImplementedError, ValueError)):
            npu_fusion_attention(*(put(x) for x in mine), hq, layout, atten_mask=True, scale=0.1, **bad, **kw)


def test_empty_batches():
    from long_vita_amd import ops
    q, k, v, _ = (t.cuda() for t in make(8, 4, 2, 64, 1))
    for cu in ([0], [0, 0], [5, 5, 5]):
        a, b = ops.score_attention(q, k, v, cu, softcap=5.0)
        assert not a.any() and torch.isinf(b).all()
    e = [t[:0].requires_grad_(True) for t in (q, k, v)]
    out, lse = ops.score_attention(*e, [0, 0], softcap=5.0)
    assert out.shape == (0, 4, 64) and lse.shape == (4, 0)
    out.sum().backward()
