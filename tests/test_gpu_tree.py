"""Drafted tokens over a KV cache against a float64 computation on the CPU: trees, chains, single tokens, ragged and empty
caches, strides, refusals, garbage behind the keys, graph replay; the accepted path's move.

Tolerances: P is rounded to bf16 before the product with V and the result once more, two half steps of 2^-8 relative to the
largest magnitude: 2^-7.  The log-sum-exp is fp32 throughout: 2e-5 covers the sums at |lse| up to ~60."""
import math

import pytest
import torch

from long_vita_amd import _lib

pytestmark = pytest.mark.gpu
REL_TOL, LSE_TOL = 2.0 ** -7, 2e-5


def slopes_of(hq):
    return torch.tensor([2.0 ** (-8.0 * (h + 1) / hq) for h in range(hq)], dtype=torch.float32)


def ref(q, k, v, lens, scale, parents=None, cap=None, slopes=None):
    """float64; parents [b][n] lists or None (chain)."""
    q, k, v = (t.double() for t in (q, k, v))
    b, n, hq, d = q.shape
    g = hq // k.shape[2]
    out, lse = torch.zeros_like(q), torch.full((b, n, hq), -math.inf, dtype=torch.float64)
    for s in range(b):
        L = int(lens[s])
        see, depth, used = torch.zeros(n, n, dtype=torch.bool), [0] * n, [True] * n
        for i in range(n):
            par = [j - 1 for j in range(n)] if parents is None else parents[s]
            if par[i] == -2:
                used[i] = False
                continue
            at = i
            while at >= 0:
                see[i, at] = True
                depth[i] += 1
                at = par[at] if par[at] < at else -1
            depth[i] -= 1
        dep = torch.tensor(depth)
        pos = torch.cat([torch.arange(L), L + dep])
        for h in range(hq):
            K, V = k[s, :L + n, h // g].clone(), v[s, :L + n, h // g].clone()
            for i in range(n):
                if not used[i]:
                    K[L + i], V[L + i] = 0, 0
            x = scale * q[s, :, h] @ K.T
            t = cap * torch.tanh(x / cap) if cap else x
            if slopes is not None:
                t = t - float(slopes[h]) * (L + dep[:, None] - pos[None, :]).abs()
            t[:, L:] = t[:, L:].masked_fill(~see, -math.inf)
            for i in range(n):
                if used[i]:
                    lse[s, i, h] = torch.logsumexp(t[i], 0)
                    out[s, i, h] = torch.exp(t[i] - lse[s, i, h]) @ V
    return out, lse


def rel(got, want):
    return float((got.detach().double().cpu() - want).abs().max() / want.abs().max().clamp_min(1e-30))


def random_parents(b, n, seed, unused=0):
    g = torch.Generator().manual_seed(seed)
    out = torch.full((b, n), -1, dtype=torch.int32)
    for s in range(b):
        for i in range(1, n):
            out[s, i] = int(torch.randint(max(-1, i - 6), i, (1,), generator=g))
        if unused:
            out[s, n - 1 - s % unused:] = -2
            for i in range(n):                      # no token hangs on an unused slot
                if out[s, i] >= 0 and out[s, out[s, i]] == -2:
                    out[s, i] = -1
    return out


def make(b, n, rows, hq, hkv, d, seed, lens, q_std=2.0):
    g = torch.Generator().manual_seed(seed)
    q = (torch.randn(b, n, hq, d, generator=g) * q_std).to(torch.bfloat16)
    k, v = (torch.randn(b, rows, hkv, d, generator=g).to(torch.bfloat16) for _ in range(2))
    for s, L in enumerate(lens):                    # what lies behind a sequence's keys must not matter
        k[s, L + n:], v[s, L + n:] = float("nan"), float("nan")
    return q, k, v


CASES = [
    # name, lens, n, hq, hkv, d, tree, unused, cap, alibi
    ("decode_one", [0], 1, 5, 1, 128, False, 0, None, False),
    ("decode_ragged", [0, 1, 127, 128, 129, 700], 1, 40, 8, 128, False, 0, None, False),
    ("decode_rule", [511, 64, 1203], 1, 10, 2, 128, False, 0, 30.0, True),
    ("decode_mqa_d64", [300, 5], 1, 16, 16, 64, False, 0, 20.0, False),
    ("decode_group_40", [200], 1, 40, 1, 128, False, 0, None, True),
    ("chain", [100, 0, 255], 7, 5, 1, 128, False, 0, None, False),
    ("chain_long", [130], 200, 2, 1, 64, False, 0, 25.0, True),
    ("tree_small", [0, 33, 640], 6, 5, 1, 128, True, 0, None, False),
    ("tree_64_rows", [513, 127], 12, 10, 2, 128, True, 0, 30.0, False),
    ("tree_128_rows", [1000], 25, 5, 1, 128, True, 0, None, True),
    ("tree_many_rows", [700, 12], 64, 10, 2, 128, True, 0, None, False),
    ("tree_256", [90], 256, 4, 2, 64, True, 0, 40.0, True),
    ("tree_unused", [129, 60, 1], 33, 4, 2, 64, True, 5, None, True),
    ("tree_unused_d128", [500, 127], 20, 5, 1, 128, True, 7, 20.0, True),
    ("tree_edge", [127, 128, 96, 97], 32, 8, 8, 64, True, 0, None, False),
    ("batch_70", [(37 * i) % 300 for i in range(70)], 3, 4, 2, 64, True, 0, None, False),
    ("batch_50_wide", [(53 * i) % 290 for i in range(50)], 14, 20, 4, 128, True, 2, None, True),
    ("batch_40_rows_100", [(97 * i) % 400 for i in range(40)], 20, 20, 4, 128, True, 2, 30.0, False),
    ("batch_one_long", [3, 5000, 0, 40, 7, 2500, 11], 9, 16, 8, 128, True, 0, None, False),
]


@pytest.mark.parametrize("name,lens,n,hq,hkv,d,tree,unused,cap,alibi", CASES, ids=[c[0] for c in CASES])
def test_matches_definition(name, lens, n, hq, hkv, d, tree, unused, cap, alibi):
    from long_vita_amd import ops
    b, rows = len(lens), max(lens) + n + 5
    q, k, v = make(b, n, rows, hq, hkv, d, len(name), lens)
    par = random_parents(b, n, 3, unused) if tree else None
    if unused:
        for s in range(b):
            for i in range(n):
                if par[s, i] == -2:
                    k[s, lens[s] + i], v[s, lens[s] + i], q[s, i] = float("nan"), float("inf"), float("nan")
    slopes = slopes_of(hq) if alibi else None
    want, want_lse = ref(q, k, v, lens, d ** -0.5, None if par is None else par.tolist(), cap, slopes)
    args = (q.cuda(), k.cuda(), v.cuda(), torch.tensor(lens, dtype=torch.int32, device="cuda"))
    kw = dict(parents=None if par is None else par.cuda(), softcap=cap, alibi_slopes=None if slopes is None else slopes.cuda(), return_lse=True)
    out, lse = ops.tree_attention(*args, **kw)
    again, lse2 = ops.tree_attention(*args, **kw)
    assert torch.equal(out, again) and torch.equal(lse, lse2)
    assert torch.isfinite(out).all()
    fin = torch.isfinite(want_lse)
    assert torch.equal(torch.isfinite(lse.cpu()), fin)
    assert float((lse.double().cpu() - want_lse)[fin].abs().max()) <= LSE_TOL
    assert rel(out, want) <= REL_TOL
    assert not out.cpu()[~fin].any()


def test_one_tree_for_all_and_chain_as_tree():
    from long_vita_amd import ops
    lens = [50, 200]
    q, k, v = (t.cuda() for t in make(2, 9, 220, 4, 2, 128, 5, lens))
    L = torch.tensor(lens, dtype=torch.int32, device="cuda")
    par = random_parents(1, 9, 7)[0].cuda()
    a = ops.tree_attention(q, k, v, L, parents=par)
    b = ops.tree_attention(q, k, v, L, parents=par.expand(2, 9).contiguous())
    c = ops.tree_attention(q, k, v, L, parents=par.expand(2, 9))             # batch stride 0
    assert torch.equal(a, b) and torch.equal(a, c)
    chain = torch.arange(-1, 8, dtype=torch.int32, device="cuda")
    sl = slopes_of(4).cuda()
    assert torch.equal(ops.tree_attention(q, k, v, L, alibi_slopes=sl), ops.tree_attention(q, k, v, L, parents=chain, alibi_slopes=sl))
    # an entry that does not point backwards counts as a root
    bad = torch.tensor([0, 5, -1, 2, 3, 8, 100, -1, 4], dtype=torch.int32, device="cuda")
    good = torch.tensor([-1, -1, -1, 2, 3, -1, -1, -1, 4], dtype=torch.int32, device="cuda")
    assert torch.equal(ops.tree_attention(q, k, v, L, parents=bad), ops.tree_attention(q, k, v, L, parents=good))


def test_parents_that_are_none():
    """A parent behind its child, the token itself, a number past the tree or an unused slot: the token continues the cache."""
    from long_vita_amd import ops
    q, k, v = (t.cuda() for t in make(1, 8, 60, 4, 2, 64, 9, [50]))
    L = _lens("cuda", 50)
    t = lambda *x: torch.tensor(x, dtype=torch.int32, device="cuda")
    sl = slopes_of(4).cuda()
    want = ops.tree_attention(q, k, v, L, parents=t(-1, -2, -1, 2, -1, -1, -1, 6), alibi_slopes=sl, return_lse=True)
    got = ops.tree_attention(q, k, v, L, parents=t(-9 + 8, -2, 1, 2, 4, 7, 2 ** 31 - 1, 6), alibi_slopes=sl, return_lse=True)
    assert all(torch.equal(a, b) for a, b in zip(got, want))


def test_matches_decode_attention():
    from long_vita_amd import ops
    q, k, v = (t.cuda() for t in make(2, 1, 1000, 40, 8, 128, 9, [999, 999]))
    L = torch.full((2,), 999, dtype=torch.int32, device="cuda")
    a, la = ops.tree_attention(q, k, v, L, return_lse=True)
    b, lb = ops.decode_attention(q[:, 0], k, v, 128 ** -0.5, return_lse=True)
    assert float((a[:, 0].float() - b.float()).abs().max()) <= 2.0 ** -7 * float(b.abs().max())
    assert float((la[:, 0] - lb).abs().max()) <= LSE_TOL


def test_lengths_out_of_range_stay_inside():
    from long_vita_amd import ops
    q, k, v = (t.cuda() for t in make(2, 4, 64, 4, 2, 64, 13, [60, 60]))
    bad = torch.tensor([-5, 1000], dtype=torch.int32, device="cuda")
    good = torch.tensor([0, 60], dtype=torch.int32, device="cuda")
    assert torch.equal(ops.tree_attention(q, k, v, bad), ops.tree_attention(q, k, v, good))


def test_strides_out_workspace_and_views():
    from long_vita_amd import ops
    lens = [70, 129]
    b, n, rows, hq, hkv, d = 2, 5, 140, 4, 2, 128
    q, k, v = make(b, n, rows, hq, hkv, d, 17, lens)
    L = torch.tensor(lens, dtype=torch.int32, device="cuda")
    want = ops.tree_attention(q.cuda(), k.cuda(), v.cuda(), L)
    kv = torch.empty(rows, b, 2 * hkv, d + 8, dtype=torch.bfloat16, device="cuda")     # [s, b, h, d] cache, K and V side by side
    kv[:, :, :hkv, :d], kv[:, :, hkv:, :d] = k.cuda().transpose(0, 1), v.cuda().transpose(0, 1)
    kc, vc = kv[:, :, :hkv, :d].transpose(0, 1), kv[:, :, hkv:, :d].transpose(0, 1)
    qs = torch.empty(n, b, hq, d + 16, dtype=torch.bfloat16, device="cuda")
    qs[..., :d] = q.cuda().transpose(0, 1)
    big = torch.full((b, n, hq, d + 4), 7.0, dtype=torch.bfloat16, device="cuda")
    ws = torch.empty(ops.tree_workspace_bytes(b, n, rows, hq, hkv, d), dtype=torch.uint8, device="cuda").fill_(255)
    got = ops.tree_attention(qs[..., :d].transpose(0, 1), kc, vc, L, out=big[..., :d], workspace=ws)
    assert torch.equal(got, want) and (big[..., d:] == 7).all()
    odd = torch.empty(q.numel() + 1, dtype=torch.bfloat16, device="cuda")[1:].view(q.shape)
    odd.copy_(q)
    assert torch.equal(ops.tree_attention(odd, k.cuda(), v.cuda(), L), want)


@pytest.mark.parametrize("n,hq,hkv", [(1, 8, 4), (9, 16, 4), (20, 16, 4)])
def test_many_sequences_one_by_one(n, hq, hkv):
    """A sequence's result does not depend on the batch around it beyond the order in which its keys are joined, nor on where
    it is stored: buffers whose rows start at odd elements get the same numbers."""
    from long_vita_amd import ops
    lens = [(61 * i) % 500 for i in range(64)]
    rows, d = max(lens) + n + 3, 128
    q, k, v = (t.cuda() for t in make(64, n, rows, hq, hkv, d, 5, lens))
    L = torch.tensor(lens, dtype=torch.int32, device="cuda")
    out, lse = ops.tree_attention(q, k, v, L, return_lse=True)
    buf = torch.full((64, n, hq + 1, d + 3), -7.0, dtype=torch.bfloat16, device="cuda")
    odd = buf[:, :, 1:, 1:d + 1]
    assert ops.tree_attention(q, k, v, L, out=odd) is odd
    # rounded once from fp32 in either case; the joins' order of adding moves a sum by a few 2^-24
    assert torch.allclose(odd.float(), out.float(), rtol=2 ** -7, atol=2 ** -16)
    buf[:, :, 1:, 1:d + 1] = -7.0
    assert bool((buf == -7.0).all())
    for s in range(0, 64, 7):
        one, one_lse = ops.tree_attention(q[s:s + 1], k[s:s + 1], v[s:s + 1], L[s:s + 1], return_lse=True)
        # P is rounded to bf16 against running maxima that may differ by the split: 2^-9 of every term, |v| up to ~4
        assert float((one.float() - out[s:s + 1].float()).abs().max()) <= 2 ** -5
        assert torch.allclose(one_lse, lse[s:s + 1], rtol=0, atol=1e-5)


def test_cache_past_32_bit_offsets():
    """Row offsets of the second sequence's keys pass 2^31 elements and 2^32 bytes."""
    from long_vita_amd import ops
    rows, hkv, d = 1100000, 8, 128                 # 1.13e9 elements per sequence
    k = torch.empty(2, rows, hkv, d, dtype=torch.bfloat16, device="cuda").fill_(float("nan"))
    v = torch.empty_like(k).fill_(float("nan"))
    g = torch.Generator(device="cuda").manual_seed(1)
    tail = 300
    q = torch.randn(2, 2, 16, d, generator=g, device="cuda").to(torch.bfloat16)
    small_k, small_v = (torch.randn(2, tail + 2, hkv, d, generator=g, device="cuda").to(torch.bfloat16) for _ in range(2))
    k[:, :tail + 2], v[:, :tail + 2] = small_k, small_v
    L = torch.full((2,), tail, dtype=torch.int32, device="cuda")
    a = ops.tree_attention(q, k, v, L)
    b = ops.tree_attention(q, small_k, small_v, L)
    # (the two calls deal the tiles to different numbers of workgroups: equal up to the partial results' fp32 joins)
    assert float((a.float() - b.float()).abs().max()) <= 2.0 ** -7 * float(b.abs().max())
    k.zero_(), v.zero_()
    k[1, -tail:], v[1, -tail:] = 1.0, 3.0          # far rows are read: everything else scores 0 against them
    full = torch.full((2,), rows - 2, dtype=torch.int32, device="cuda")
    out = ops.tree_attention(torch.ones_like(q), k, v, full)
    e = math.exp(128 ** 0.5)
    seen = (tail - 1) * e                           # token 0 sees all but the last row
    assert abs(float(out[1, 0].float().mean()) - 3 * seen / (seen + rows - 1 - (tail - 1))) < 0.02
    assert not out[0].any()


def test_graph_replay_with_new_lengths_and_streams():
    from long_vita_amd import ops
    lens = [100, 37]
    q, k, v = (t.cuda() for t in make(2, 6, 300, 10, 2, 128, 23, [294, 294]))
    L = torch.tensor(lens, dtype=torch.int32, device="cuda")
    par = random_parents(2, 6, 3).cuda()
    ws = [torch.empty(ops.tree_workspace_bytes(2, 6, 300, 10, 2, 128), dtype=torch.uint8, device="cuda") for _ in range(2)]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        ops.tree_attention(q, k, v, L, parents=par, workspace=ws[0])
    torch.cuda.synchronize()
    graphs = []
    for w in ws:
        gr = torch.cuda.CUDAGraph()
        with torch.cuda.graph(gr):
            o = ops.tree_attention(q, k, v, L, parents=par, workspace=w)
        graphs.append((gr, o))
    for it in range(3):
        L.copy_(torch.tensor([100 + 60 * it, 37 * it], dtype=torch.int32))
        par.copy_(random_parents(2, 6, 40 + it))
        want = ops.tree_attention(q, k, v, L, parents=par)
        for gr, o in graphs:
            o.zero_()
            gr.replay()
            torch.cuda.synchronize()
            assert torch.equal(o, want)


@pytest.mark.parametrize("hkv,d,strided", [(2, 128, False), (3, 64, True)])
def test_accept_moves_the_path(hkv, d, strided):
    from long_vita_amd import ops
    lens, n, rows = [10, 0, 77, 3], 70, 160
    b = len(lens)
    g = torch.Generator().manual_seed(3)
    k, v = (torch.randn(b, rows, hkv, d, generator=g).to(torch.bfloat16) for _ in range(2))
    w = torch.rand(b, hkv, rows, generator=g)
    paths, counts = torch.full((b, n), 12345, dtype=torch.int32), [5, 0, 70, 40]
    for s, c in enumerate(counts):
        paths[s, :c] = torch.sort(torch.randperm(n, generator=g)[:c]).values.int()
    if strided:
        kc = k.cuda().transpose(0, 1).contiguous().transpose(0, 1)
        vc = torch.zeros(b, rows, hkv + 1, d + 8, dtype=torch.bfloat16, device="cuda")[:, :, :hkv, :d]
        vc.copy_(v)
        wc = torch.zeros(b, hkv, rows + 3, device="cuda")[..., :rows]
        wc.copy_(w)
    else:
        kc, vc, wc = k.cuda(), v.cuda(), w.cuda()
    new = ops.tree_accept(kc, vc, torch.tensor(lens, dtype=torch.int32, device="cuda"), paths.cuda(),
                          torch.tensor(counts, dtype=torch.int32, device="cuda"), wc)
    assert new.tolist() == [a + c for a, c in zip(lens, counts)] and new.dtype == torch.int32
    for s, (L, c) in enumerate(zip(lens, counts)):
        src = torch.arange(rows)
        src[L:L + c] = L + paths[s, :c].long()
        for got, was in ((kc[s].cpu(), k[s][src]), (vc[s].cpu(), v[s][src]), (wc[s].cpu(), w[s][:, src])):
            assert torch.equal(got, was)


def _lens(dev, *x):
    return torch.tensor(x, dtype=torch.int32, device=dev)


REFUSED = [
    ("rank", lambda q, k, v, L: ((q[0], k, v, L), {})),
    ("dtype", lambda q, k, v, L: ((q.float(), k, v, L), {})),
    ("batch", lambda q, k, v, L: ((q[:1], k, v, L[:1]), {})),
    ("kv_shapes", lambda q, k, v, L: ((q, k, v[:, :-1], L), {})),
    ("rows", lambda q, k, v, L: ((q, k[:, :2], v[:, :2], L), {})),
    ("lens_type", lambda q, k, v, L: ((q, k, v, L.long()), {})),
    ("lens_shape", lambda q, k, v, L: ((q, k, v, L[:1]), {})),
    ("parents_type", lambda q, k, v, L: ((q, k, v, L), dict(parents=torch.zeros(3, dtype=torch.int64, device=q.device)))),
    ("parents_shape", lambda q, k, v, L: ((q, k, v, L), dict(parents=torch.zeros(4, dtype=torch.int32, device=q.device)))),
    ("parents_cpu", lambda q, k, v, L: ((q, k, v, L), dict(parents=torch.zeros(3, dtype=torch.int32)))),
    ("cap", lambda q, k, v, L: ((q, k, v, L), dict(softcap=-1.0))),
    ("slopes", lambda q, k, v, L: ((q, k, v, L), dict(alibi_slopes=torch.zeros(2, device=q.device)))),
    ("scale", lambda q, k, v, L: ((q, k, v, L, float("nan")), {})),
    ("scale_zero", lambda q, k, v, L: ((q, k, v, L, 0.0), {})),
    ("grad", lambda q, k, v, L: ((q.clone().requires_grad_(True), k, v, L), {})),
    ("out", lambda q, k, v, L: ((q, k, v, L), dict(out=torch.empty(1, device=q.device)))),
    ("out_is_q", lambda q, k, v, L: ((q, k, v, L), dict(out=q))),
    ("out_in_cache", lambda q, k, v, L: ((q, (kk := torch.zeros(2, 20, 4, 64, dtype=torch.bfloat16, device=q.device))[:, :, :2], v, L), dict(out=kk[:, :3]))),
    ("out_expanded", lambda q, k, v, L: ((q, k, v, L), dict(out=torch.empty_like(q[:1]).expand(2, -1, -1, -1)))),
    ("lse", lambda q, k, v, L: ((q, k, v, L), dict(lse=torch.empty(1, device=q.device)))),
    ("workspace", lambda q, k, v, L: ((q, k, v, L), dict(workspace=torch.empty(8, dtype=torch.uint8, device=q.device)))),
    ("cache_strides", lambda q, k, v, L: ((q, k.transpose(2, 3).contiguous().transpose(2, 3), v, L), {})),
    ("cpu", lambda q, k, v, L: ((q.cpu(), k, v, L), {})),
    ("too_many_tokens", lambda q, k, v, L: ((q[:, :1].expand(2, 257, 4, 64), k[:, :1].expand(2, 300, 2, 64), v[:, :1].expand(2, 300, 2, 64), L), {})),
    ("no_tokens", lambda q, k, v, L: ((q[:, :0], k, v, L), {})),
]


@pytest.mark.parametrize("name,call", REFUSED, ids=[r[0] for r in REFUSED])
def test_refusals(name, call):
    from long_vita_amd import ops
    q, k, v = (t.cuda() for t in make(2, 3, 20, 4, 2, 64, 1, [5, 9]))
    args, kw = call(q, k, v, _lens("cuda", 5, 9))
    with pytest.raises(_lib.LvAttnError):
        ops.tree_attention(*args, **kw)


def test_accept_refusals():
    from long_vita_amd import ops
    k, v = (torch.zeros(2, 20, 2, 64, dtype=torch.bfloat16, device="cuda") for _ in range(2))
    L, path, cnt = _lens("cuda", 3, 4), torch.zeros(2, 5, dtype=torch.int32, device="cuda"), _lens("cuda", 1, 2)
    for bad in ((k.float(), v, L, path, cnt), (k, v[:1], L, path, cnt), (k, v, L.long(), path, cnt), (k, v, L, path[0], cnt), (k, v, L, path.long(), cnt),
                (k, v, L, path, cnt[:1]), (k[:1].expand(2, 20, 2, 64), v, L, path, cnt), (k, v, L, path, cnt, torch.zeros(2, 2, 19, device="cuda"))):
        with pytest.raises(_lib.LvAttnError):
            ops.tree_accept(*bad)
