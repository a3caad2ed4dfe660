"""tree_accept with lengths and counts outside their range: what it returns is what it moved."""
import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("rows,n", [(40, 6), (6, 6)])
def test_lengths_returned_are_those_moved(rows, n):
    from long_vita_amd import ops
    lens, counts = [7, -3, rows, rows - n + 1, 2 ** 31 - 1, 0], [n + 5, 2, 3, -4, 2 ** 31 - 1, -2 ** 31]
    b, hkv, d = len(lens), 2, 64
    g = torch.Generator().manual_seed(1)
    k, v = (torch.randn(b, rows, hkv, d, generator=g).to(torch.bfloat16) for _ in range(2))
    w = torch.rand(b, hkv, rows, generator=g)
    path = torch.tensor([[0, 2, 3, 4, 5, 5]] * b, dtype=torch.int32)
    kc, vc, wc = k.cuda(), v.cuda(), w.cuda()
    new = ops.tree_accept(kc, vc, torch.tensor(lens, dtype=torch.int32, device="cuda"), path.cuda(), torch.tensor(counts, dtype=torch.int32, device="cuda"), wc)
    clamp = [(min(max(x, 0), rows - n), min(max(c, 0), n)) for x, c in zip(lens, counts)]
    assert new.tolist() == [x + c for x, c in clamp] and max(new.tolist()) <= rows
    for s, (x, c) in enumerate(clamp):
        src = torch.arange(rows)
        src[x:x + c] = x + path[s, :c].long()
        assert torch.equal(kc[s].cpu(), k[s][src]) and torch.equal(vc[s].cpu(), v[s][src]) and torch.equal(wc[s].cpu(), w[s][:, src])


def test_graph_replay():
    from long_vita_amd import ops
    b, rows, n, hkv, d = 3, 64, 8, 2, 128
    g = torch.Generator().manual_seed(2)
    k0, v0 = (torch.randn(b, rows, hkv, d, generator=g).to(torch.bfloat16).cuda() for _ in range(2))
    k, v = k0.clone(), v0.clone()
    lens, path, cnt = torch.tensor([5, 0, 56], dtype=torch.int32).cuda(), torch.arange(n, dtype=torch.int32).expand(b, n).contiguous().cuda(), torch.zeros(b, dtype=torch.int32).cuda()
    ops.tree_accept(k, v, lens, path, cnt)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        new = ops.tree_accept(k, v, lens, path, cnt)
    for it in range(3):
        k.copy_(k0), v.copy_(v0), cnt.copy_(torch.tensor([it, 3, 20 * it], dtype=torch.int32)), new.zero_()
        path[:, 1:] = torch.arange(2, n + 1, dtype=torch.int32).clamp(max=n - 1).cuda()
        graph.replay()
        torch.cuda.synchronize()
        k1, v1 = k0.clone(), v0.clone()
        assert torch.equal(new, ops.tree_accept(k1, v1, lens, path, cnt)) and torch.equal(k, k1) and torch.equal(v, v1)
