"""Accumulated attention weights and cache eviction against float64 / exact computations on the CPU, and a run of the cache
operators together.

Tolerances of the weights: every term is an fp32 exponential of an fp32 score: at |t| up to 30 in log2 units the argument is
off by a few 2^-24 * 32, i.e. a few 2e-6 relative, and the sums are compensated: 2e-5 relative to the largest weight, plus the
rounding of the result.  What eviction keeps, and in which order, is exact."""
import math

import pytest
import torch

from long_vita_amd import _lib
from tests.test_gpu_tree import make, random_parents, ref, slopes_of

pytestmark = pytest.mark.gpu
W_TOL = 2e-5


def ref_weights(q, k, lens, scale, lse, w, parents=None, cap=None, slopes=None, rho=None):
    """float64: the terms of each row, from its own scores."""
    b, n, hq, d = q.shape
    g = hq // k.shape[2]
    w = w.double().clone()
    for s in range(b):
        L = int(lens[s])
        par = [j - 1 for j in range(n)] if parents is None else parents[s]
        see, depth = torch.zeros(n, n, dtype=torch.bool), [0] * n
        for i in range(n):
            at = i if par[i] != -2 else -1
            while at >= 0:
                see[i, at] = True
                depth[i] += 1
                at = par[at]
            depth[i] = max(depth[i] - 1, 0)
        dep = torch.tensor(depth)
        pos = torch.cat([torch.arange(L), L + dep])
        for i in range(n):
            if par[i] == -2 or (rho is not None and not float(rho[s, i]) > 0):
                continue
            vis = torch.cat([torch.ones(L, dtype=torch.bool), see[i]])
            cols = torch.nonzero(vis)[:, 0]
            for h in range(hq):
                x = scale * (k[s, cols, h // g].double() @ q[s, i, h].double())
                t = cap * torch.tanh(x / cap) if cap else x
                if slopes is not None:
                    t = t - float(slopes[h]) * (L + dep[i] - pos[cols]).abs()
                w[s, h // g, cols] += (1.0 if rho is None else float(rho[s, i])) * torch.exp(t - lse[s, i, h].double())
    return w


W_CASES = [
    # name, lens, n, hq, hkv, d, tree, unused, cap, alibi, rho
    ("decode", [0, 1, 63, 64, 500], 1, 40, 8, 128, False, 0, None, False, False),
    ("decode_rule", [300, 17], 1, 10, 2, 64, False, 0, 30.0, True, False),
    ("tree", [200, 31], 12, 5, 1, 128, True, 0, None, False, True),
    ("tree_rule", [129, 64], 40, 4, 2, 64, True, 0, 20.0, True, True),
    ("tree_unused", [255, 0, 90], 33, 4, 2, 128, True, 6, None, True, False),
    ("prompt", [0], 333, 5, 1, 128, False, 0, None, False, False),
    ("prompt_cap", [0], 260, 4, 4, 64, False, 0, 25.0, False, False),
    ("prompt_tail", [700, 100], 64, 5, 1, 128, False, 0, None, True, True),
    ("group_40", [150], 3, 40, 1, 64, False, 0, None, False, False),
    ("rows_128", [600, 33, 256], 32, 4, 1, 128, True, 3, None, False, True),
    ("rows_128_rule", [300, 70], 25, 5, 1, 128, True, 0, 25.0, True, False),
    ("rows_129", [255, 128], 43, 3, 1, 128, True, 2, None, False, True),
    ("tree_long_rows", [400, 90], 100, 5, 1, 64, True, 9, 30.0, True, True),
    ("batch_60", [(41 * i) % 310 for i in range(60)], 5, 8, 2, 64, True, 0, None, False, False),
]


@pytest.mark.parametrize("name,lens,n,hq,hkv,d,tree,unused,cap,alibi,with_rho", W_CASES, ids=[c[0] for c in W_CASES])
def test_key_weights(name, lens, n, hq, hkv, d, tree, unused, cap, alibi, with_rho):
    from long_vita_amd import ops
    b, rows = len(lens), max(lens) + n + 70
    q, k, v = make(b, n, rows, hq, hkv, d, len(name) + 1, lens)
    par = random_parents(b, n, 5, unused) if tree else None
    g = torch.Generator().manual_seed(2)
    rho = torch.rand(b, n, generator=g) * (torch.rand(b, n, generator=g) < 0.6) if with_rho else None
    slopes = slopes_of(hq) if alibi else None
    lists = None if par is None else par.tolist()
    _, lse = ref(q, k, v, lens, d ** -0.5, lists, cap, slopes)
    lse = lse.float()
    w = torch.rand(b, hkv, rows, generator=g)
    want = ref_weights(q, k, lens, d ** -0.5, lse, w, lists, cap, slopes, rho)
    for s in range(b):
        for i in range(n):
            if unused and par[s, i] == -2:
                k[s, lens[s] + i], q[s, i], lse[s, i] = float("nan"), float("nan"), float("nan")
            if rho is not None and not rho[s, i] > 0:      # a token that counts for nothing may hold anything
                q[s, i], lse[s, i] = float("inf"), float("nan")
    gpu = [t.cuda() for t in (q, k, lse, w)]
    L = torch.tensor(lens, dtype=torch.int32, device="cuda")
    kw = dict(parents=None if par is None else par.cuda(), softcap=cap, alibi_slopes=None if slopes is None else slopes.cuda(),
              row_weight=None if rho is None else rho.cuda())
    got = ops.key_weights(*gpu, L, **kw)
    assert torch.equal(gpu[3].cpu(), w)                                       # a new tensor
    err = (got.double().cpu() - want).abs()
    assert float(err.max()) <= W_TOL * float(want.max())
    for s, x in enumerate(lens):
        assert torch.equal(got[s, :, x + n:].cpu(), w[s, :, x + n:])          # rows that hold no key
    assert torch.equal(ops.key_weights(*gpu, L, **kw), got)
    inplace = ops.key_weights(*gpu, L, out=gpu[3], **kw)
    assert inplace is gpu[3] and torch.equal(inplace, got)


def test_weights_sum_to_rows():
    """Every row's terms sum to 1: the totals are the number of rows per KV head (a long prompt, cut into row pieces)."""
    from long_vita_amd import ops
    n, hq, hkv = 3500, 5, 1
    g = torch.Generator(device="cuda").manual_seed(1)
    q, k, v = (torch.randn(1, n, h, 128, generator=g, device="cuda").to(torch.bfloat16) for h in (hq, hkv, hkv))
    out, lse = ops.varlen_attention(q[0], k[0], v[0], [0, n])
    w = ops.key_weights(q, k, lse.t().contiguous()[None], torch.zeros(1, hkv, n, device="cuda"), torch.zeros(1, dtype=torch.int32, device="cuda"))
    # the log-sum-exps are fp32 at ~8 (2^-22): relative 5e-7 on every term; 1e-5 of the total
    assert abs(float(w.double().sum()) - n * hq) <= 1e-5 * n * hq
    late = torch.randperm(n, generator=torch.Generator().manual_seed(2))[:5]
    for j in late.tolist():
        x = (q[0, j:].double() @ k[0, j, 0].double()) * 128 ** -0.5
        want = torch.exp(x - lse[:, j:].t().double()).sum()
        assert abs(float(w[0, 0, j]) - float(want)) <= W_TOL * max(1.0, float(want))


def kept_ref(w, length, keep, sink, recent):
    if length <= keep:
        return list(range(length))
    mid = list(range(sink, length - recent))
    nan = [math.isnan(float(w[j])) for j in range(len(w))]
    mid.sort(key=lambda j: (0 if nan[j] else 1, 0.0 if nan[j] else -float(w[j]), j))
    return list(range(sink)) + sorted(mid[:keep - sink - recent]) + list(range(length - recent, length))


E_CASES = [
    # name, rows, lens, hkv, d, keep, sink, recent
    ("one_row", 1, [1, 0], 1, 64, 1, 0, 0),
    ("tiny", 9, [9, 3, 5, 0], 2, 128, 4, 1, 1),
    ("all_fixed", 300, [300, 10], 2, 64, 40, 20, 20),
    ("middle_only", 777, [777, 776, 100], 3, 64, 100, 0, 0),
    ("budget", 4096, [4096, 1500, 900, 1024, 0], 8, 128, 1024, 4, 128),
    ("largest_small", 16384, [16384, 16383, 9000], 2, 64, 5000, 4, 1000),
    ("smallest_long", 16385, [16385, 8192, 8193, 100], 2, 64, 5000, 4, 1000),
    ("long", 70001, [70001, 65536, 300, 0], 2, 128, 8191, 8, 4097),
    ("long_keep_most", 40000, [40000, 39999], 1, 64, 39998, 0, 39000),
    ("keep_all", 500, [500, 400], 2, 64, 500, 4, 4),
]


@pytest.mark.parametrize("values", ["spread", "ties", "odd"])
@pytest.mark.parametrize("name,rows,lens,hkv,d,keep,sink,recent", E_CASES, ids=[c[0] for c in E_CASES])
def test_evict(name, rows, lens, hkv, d, keep, sink, recent, values):
    from long_vita_amd import ops
    b = len(lens)
    g = torch.Generator().manual_seed(rows + len(values))
    k, v = (torch.randn(b, rows, hkv, d, generator=g).to(torch.bfloat16) for _ in range(2))
    w = torch.randn(b, hkv, rows, generator=g).mul(3).exp()
    if values == "ties":
        w = torch.randint(0, 3, w.shape, generator=g).float()
    if values == "odd":          # signs, both zeros, infinities, NaN of both signs, denormals
        pool = torch.tensor([0.0, -0.0, 1.0, -1.0, math.inf, -math.inf, math.nan, -math.nan, 1e-42, -1e-42, 3e38])
        w = pool[torch.randint(0, len(pool), w.shape, generator=g)]
    L = torch.tensor(lens, dtype=torch.int32, device="cuda")
    k2, v2, w2, l2, idx = ops.evict_cache(k.cuda(), v.cuda(), w.cuda(), L, keep, sink, recent)
    assert l2.tolist() == [min(x, keep) for x in lens] and l2.dtype == torch.int32
    for s, x in enumerate(lens):
        for h in range(hkv):
            want = kept_ref(w[s, h], x, keep, sink, recent)
            m = len(want)
            assert idx[s, h, :m].tolist() == want and (idx[s, h, m:] == -1).all()
            assert torch.equal(k2[s, :m, h].cpu(), k[s, want, h]) and torch.equal(v2[s, :m, h].cpu(), v[s, want, h])
            assert not k2[s, m:, h].any() and not v2[s, m:, h].any() and not w2[s, h, m:].any()
            assert torch.equal(w2[s, h, :m].cpu().view(torch.int32), w[s, h, want].view(torch.int32))


def test_evict_into_buffers_and_views():
    from long_vita_amd import ops
    b, rows, hkv, d, keep = 2, 600, 2, 64, 200
    lens = [600, 150]
    g = torch.Generator().manual_seed(9)
    k, v = (torch.randn(b, rows, hkv, d, generator=g).to(torch.bfloat16) for _ in range(2))
    w = torch.rand(b, hkv, rows, generator=g)
    L = torch.tensor(lens, dtype=torch.int32, device="cuda")
    want = ops.evict_cache(k.cuda(), v.cuda(), w.cuda(), L, keep, 2, 30)
    kv = torch.empty(rows, b, 2 * hkv, d, dtype=torch.bfloat16, device="cuda")
    kv[:, :, :hkv], kv[:, :, hkv:] = k.cuda().transpose(0, 1), v.cuda().transpose(0, 1)
    bufs = [torch.full((b, keep + 50, hkv, d + 8), 7.0, dtype=torch.bfloat16, device="cuda")[..., :d] for _ in range(2)]
    wb = torch.full((b, hkv, keep + 3), 7.0, device="cuda")
    wide = torch.zeros(b, hkv + 1, rows + 5, device="cuda")[:, :hkv, :rows]
    wide.copy_(w)
    got = ops.evict_cache(kv[:, :, :hkv].transpose(0, 1), kv[:, :, hkv:].transpose(0, 1), wide, L, keep, 2, 30, out=(bufs[0], bufs[1], wb))
    assert got[0] is bufs[0] and torch.equal(got[4], want[4]) and torch.equal(got[3], want[3])
    for s, m in enumerate((200, 150)):
        for a, c in zip(got[:2], want[:2]):
            assert torch.equal(a[s, :m], c[s, :m]) and (a[s, m:] == 7).all()
        assert torch.equal(wb[s, :, :m], want[2][s, :, :m]) and (wb[s, :, m:] == 7).all()


def test_run_together():
    """A serving loop: a prompt, its weights, drafted trees with an accepted path, an eviction, and decode on what is left: at
    every step against the float64 definition on the same cache."""
    from long_vita_amd import ops
    hq, hkv, d, rows, prompt, n = 10, 2, 128, 400, 230, 12
    g = torch.Generator().manual_seed(77)

    def draw(*shape, std=1.0):
        return (torch.randn(*shape, generator=g) * std).to(torch.bfloat16)
    k, v = torch.full((1, rows, hkv, d), float("nan"), dtype=torch.bfloat16), torch.full((1, rows, hkv, d), float("nan"), dtype=torch.bfloat16)
    k[:, :prompt], v[:, :prompt] = draw(1, prompt, hkv, d), draw(1, prompt, hkv, d)
    q = draw(1, prompt, hq, d, std=2.0)
    kc, vc = k.cuda(), v.cuda()
    # prompt: causal attention with a cap, its log-sum-exps feed the weights
    out, lse = ops.score_attention(q[0].cuda(), kc[0, :prompt], vc[0, :prompt], [0, prompt], softcap=30.0)
    zero = torch.zeros(1, dtype=torch.int32, device="cuda")
    w = ops.key_weights(q.cuda(), kc, lse.t().contiguous()[None], torch.zeros(1, hkv, rows, device="cuda"), zero, softcap=30.0)
    want_w = ref_weights(q, k, [0], d ** -0.5, lse.t().cpu()[None], torch.zeros(1, hkv, rows), cap=30.0)
    assert float((w.double().cpu() - want_w).abs().max()) <= W_TOL * float(want_w.max())
    L = torch.full((1,), prompt, dtype=torch.int32, device="cuda")
    host_len = prompt
    for step in range(3):
        par = random_parents(1, n, 100 + step)
        kd, vd, qd = draw(1, n, hkv, d), draw(1, n, hkv, d), draw(1, n, hq, d, std=2.0)
        kc[:, host_len:host_len + n], vc[:, host_len:host_len + n] = kd.cuda(), vd.cuda()
        o, ls = ops.tree_attention(qd.cuda(), kc, vc, L, parents=par.cuda(), softcap=30.0, return_lse=True)
        wo, wl = ref(qd, kc.cpu(), vc.cpu(), [host_len], d ** -0.5, par.tolist(), 30.0)
        assert float((o.double().cpu() - wo).abs().max()) <= 2.0 ** -7 * float(wo.abs().max())
        leaf = n - 1 - step                       # the path to one leaf is accepted
        path = []
        while leaf >= 0:
            path.insert(0, leaf)
            leaf = int(par[0, leaf])
        m = len(path)
        rho = torch.zeros(1, n, device="cuda")
        rho[0, path] = 1.0
        ops.key_weights(qd.cuda(), kc, ls, w, L, parents=par.cuda(), softcap=30.0, row_weight=rho, out=w)
        want_w = ref_weights(qd, kc.cpu(), [host_len], d ** -0.5, ls.cpu(), want_w.float(), par.tolist(), 30.0, rho=rho.cpu())
        pt = torch.zeros(1, n, dtype=torch.int32, device="cuda")
        pt[0, :m] = torch.tensor(path, dtype=torch.int32)
        L = ops.tree_accept(kc, vc, L, pt, torch.tensor([m], dtype=torch.int32, device="cuda"), w)
        want_w[:, :, host_len:host_len + m] = want_w[:, :, [host_len + x for x in path]]
        assert torch.equal(kc[0, host_len:host_len + m].cpu(), kd[0, path])
        host_len += m
        assert L.tolist() == [host_len]
        assert float((w.double().cpu() - want_w)[:, :, :host_len].abs().max()) <= 2 * W_TOL * float(want_w.max())
    bufs = (torch.zeros_like(kc), torch.zeros_like(vc), torch.zeros_like(w))
    k2, v2, w2, L2, idx = ops.evict_cache(kc, vc, w, L, 128, sink=4, recent=32, out=bufs)
    assert L2.tolist() == [128]
    for h in range(hkv):
        rows_kept = kept_ref(w[0, h].cpu(), host_len, 128, 4, 32)
        assert idx[0, h].tolist() == rows_kept and torch.equal(k2[0, :128, h], kc[0, rows_kept, h])
    qn, kn, vn = draw(1, 1, hq, d, std=2.0), draw(1, 1, hkv, d), draw(1, 1, hkv, d)
    k2[:, 128], v2[:, 128] = kn[:, 0].cuda(), vn[:, 0].cuda()
    o = ops.tree_attention(qn.cuda(), k2, v2, L2, softcap=30.0)
    wo, _ = ref(qn, k2.cpu(), v2.cpu(), [128], d ** -0.5, cap=30.0)
    assert float((o.double().cpu() - wo).abs().max()) <= 2.0 ** -7 * float(wo.abs().max())


@pytest.mark.parametrize("n", [1, 70])
def test_long_cache_past_32_bit_offsets(n):
    """A cache of more than 2^32 bytes and 2^31 elements: weights and eviction at both of its ends."""
    from long_vita_amd import ops
    rows, hq, hkv, d = (1 << 21) + 5000, 8, 8, 128
    length = rows - n
    g = torch.Generator(device="cuda").manual_seed(3)
    k = torch.randn(1, rows, hkv, d, generator=g, device="cuda", dtype=torch.bfloat16)
    q = torch.randn(1, n, hq, d, generator=g, device="cuda", dtype=torch.bfloat16)
    assert k.numel() > 2 ** 31
    L = torch.tensor([length], dtype=torch.int32, device="cuda")
    lse = torch.full((1, n, hq), 15.0, device="cuda")
    wide = 5 if n == 70 else 1             # heads of one KV head side by side: 70 tokens x 5 heads take the kernel for many rows
    qw = q.repeat_interleave(wide, 2)
    w0 = torch.zeros(1, hkv, rows, device="cuda")
    w = ops.key_weights(qw, k, lse.repeat_interleave(wide, 2), w0, L)
    for j in (0, 127, 1 << 20, length - 1, length, rows - 1):
        x = (q[0].double() * k[0, j].double()).sum(-1) * d ** -0.5                         # [n, heads]
        see = torch.arange(n, device="cuda")[:, None] >= j - length
        want = wide * (torch.exp(x - 15.0) * see).sum(0)
        assert float((w[0, :, j].double() - want).abs().max()) <= W_TOL * float(want.max())
    # the heaviest are planted, two of them behind the offsets
    top = torch.tensor([5, 1 << 20, length - 3], device="cuda")
    w[0, :, top] = w.max() * 2 + 1
    k2, v2, w2, L2, idx = ops.evict_cache(k, k, w, L, 40, sink=2, recent=1)
    keep = idx[0].long()
    assert int(L2[0]) == 40 and all(bool((keep == t).any(1).all()) for t in top.tolist()) and bool((keep[:, -1] == length - 1).all())
    for h in range(hkv):
        assert torch.equal(k2[0, :, h], k[0, keep[h], h]) and torch.equal(v2[0, :, h], k2[0, :, h]) and torch.equal(w2[0, h], w[0, h, keep[h]])


def test_two_streams_at_once():
    """Calls of different batches on two streams, interleaved without a wait, give what each gives alone."""
    from long_vita_amd import ops
    sets = []
    for seed, lens, n in ((1, [700, 20000, 90], 5), (2, [3000, 40, 18000, 256], 30)):
        b, rows = len(lens), max(lens) + n
        q, k, v = (t.cuda() for t in make(b, n, rows, 10, 2, 128, seed, lens))
        par = random_parents(b, n, seed, 0).cuda()
        sets.append((q, k, v, torch.tensor(lens, dtype=torch.int32, device="cuda"), par, torch.rand(b, 2, rows, device="cuda")))

    def step(q, k, v, L, par, w):
        out, lse = ops.tree_attention(q, k, v, L, parents=par, return_lse=True)
        w2 = ops.key_weights(q, k, lse, w, L, parents=par)
        return (out, lse, w2, *ops.evict_cache(k, v, w2, L, 500, sink=4, recent=50))
    alone = [[t.clone() for t in step(*x)] for x in sets]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in sets]
    got = []
    for _ in range(4):
        for st, x in zip(streams, sets):
            with torch.cuda.stream(st):
                got.append(step(*x))
    torch.cuda.synchronize()
    for i, res in enumerate(got):
        assert all(torch.equal(a, b) for a, b in zip(res, alone[i % 2]))


def test_graph_replay():
    from long_vita_amd import ops
    b, rows, hkv, d = 2, 20000, 2, 64
    g = torch.Generator(device="cuda").manual_seed(4)
    k, v = (torch.randn(b, rows, hkv, d, generator=g, device="cuda").to(torch.bfloat16) for _ in range(2))
    q = torch.randn(b, 9, 8, d, generator=g, device="cuda").to(torch.bfloat16)
    lse = torch.full((b, 9, 8), 9.0, device="cuda")
    w = torch.rand(b, hkv, rows, generator=g, device="cuda")
    L = torch.tensor([rows - 9, 5000], dtype=torch.int32, device="cuda")

    def step():
        x = ops.key_weights(q, k, lse, w, L)
        return (x, *ops.evict_cache(k, v, x, L, 3000, 4, 500))
    step()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        captured = step()
    for it in range(3):
        w.copy_(torch.rand(b, hkv, rows, generator=g, device="cuda"))
        L.copy_(torch.tensor([rows - 9 - 100 * it, 1000 * (it + 1)], dtype=torch.int32))
        for t in captured:
            t.zero_()
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, c) for a, c in zip(captured, step()))


def test_refusals():
    from long_vita_amd import ops
    q, k, v = (t.cuda() for t in make(2, 3, 20, 4, 2, 64, 1, [5, 9]))
    L = torch.tensor([5, 9], dtype=torch.int32, device="cuda")
    w, lse = torch.zeros(2, 2, 20, device="cuda"), torch.zeros(2, 3, 4, device="cuda")
    weights = [
        ((q, k, lse[:1], w, L), {}), ((q, k, lse.double(), w, L), {}), ((q, k, lse, w[..., :19], L), {}), ((q, k, lse, w.half(), L), {}),
        ((q.float(), k, lse, w, L), {}), ((q, k, lse, w, L.long()), {}), ((q, k, lse, w, L), dict(row_weight=torch.zeros(2, 4, device="cuda"))),
        ((q, k, lse, w, L), dict(parents=torch.zeros(2, dtype=torch.int32, device="cuda"))), ((q, k, lse, w, L), dict(softcap=0.0)),
        ((q, k, lse, w, L), dict(out=torch.zeros(2, 2, 21, device="cuda"))), ((q, k, lse, w.cpu(), L), {}),
        ((q, k, lse, torch.zeros(3, 2, 20, device="cuda")[:2], L), dict(out=None, scale=float("inf"))),
        ((q, k, lse, w.expand(2, 2, 20), L), dict(out=torch.zeros(1, 1, 20, device="cuda").expand(2, 2, 20))),
        ((q.clone().requires_grad_(True), k, lse, w, L), {}),
    ]
    buf = torch.zeros(2 * 2 * 20 + 4, device="cuda")
    weights.append(((q, k, lse, buf[:80].view(2, 2, 20), L), dict(out=buf[4:].view(2, 2, 20))))
    for args, kw in weights:
        with pytest.raises(_lib.LvAttnError):
            ops.key_weights(*args, **kw)
    fine = [torch.zeros(2, 8, 2, 64, dtype=torch.bfloat16, device="cuda") for _ in range(2)] + [torch.zeros(2, 2, 8, device="cuda")]
    evicts = [
        ((k, v, w, L, 0), {}), ((k, v, w, L, 21), {}), ((k, v, w, L, 8, 5, 4), {}), ((k, v, w, L, 8, -1, 0), {}), ((k, v, w, L, 8, 0, -1), {}),
        ((k, v[:, :19], w, L, 8), {}), ((k, v, w[..., :19], L, 8), {}), ((k, v, w, L[:1], 8), {}), ((k, v, w, L.long(), 8), {}),
        ((k.float(), v, w, L, 8), {}), ((k, v, w.cpu(), L, 8), {}), ((k, v, w, L, 8), dict(out=(k, fine[1], fine[2]))),
        ((k, v, w, L, 9), dict(out=tuple(fine))), ((k, v, w, L, 8), dict(out=(fine[0], fine[1], fine[2].half()))),
        ((k, v, w, L, 8), dict(out=(fine[0][:1].expand(2, 8, 2, 64), fine[1], fine[2]))),
        ((k, v, w.clone().requires_grad_(True), L, 8), {}), ((k, v, w, L, 8), dict(out=(fine[0], fine[0], fine[2]))),
    ]
    for args, kw in evicts:
        with pytest.raises(_lib.LvAttnError):
            ops.evict_cache(*args, **kw)
