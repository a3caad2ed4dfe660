"""Graphs of score_attention: each keeps its work-item tables for as long as it lives and no longer."""
import gc

import pytest
import torch

from long_vita_amd import _lib
from tests.test_gpu_score import make

pytestmark = pytest.mark.gpu


def test_tables_live_as_long_as_their_graphs():
    from long_vita_amd import ops
    q, k, v, do = (t.cuda() for t in make(500, 4, 2, 64, 43))
    leaves = [t.clone().requires_grad_(True) for t in (q, k, v)]
    cu = [0, 222, 500]

    def step():
        out, lse = ops.score_attention(*leaves, cu, softcap=30.0)
        return (out, lse, *torch.autograd.grad(out, leaves, do))

    def mine():
        return [t for key, t in ops._captured_tables.items() if key[1][1][0] == tuple(cu)]
    want = [t.detach().clone() for t in step()]
    side = torch.cuda.Stream()
    graphs = []
    for _ in range(2):
        with torch.cuda.stream(side):
            step()
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            captured = step()
        graphs.append((graph, captured))
        del captured
        for n in range(ops._blocks.capacity + 1):       # the tables' turn in the cache is over
            ops._blocks.get(("other", n), lambda: None)
    per_graph = len(mine()) // 2
    assert per_graph >= 2 and len({id(t) for t in mine()}) == 2 * per_graph
    junk = [torch.full((64,), -1, dtype=torch.int32, device="cuda") for _ in range(2000)]
    for _ in range(3):
        for graph, captured in graphs:
            for t in captured:
                t.detach().zero_()
            graph.replay()
            torch.cuda.synchronize()
            assert all(torch.equal(a, b) for a, b in zip(captured, want))
    del junk, graph, captured
    graphs.pop(0)
    gc.collect()
    torch.cuda.synchronize()
    ops.score_attention(q, k, v, [0, 9, 500])           # builds a table, which is when ended graphs are looked for
    assert len(mine()) == per_graph
    graph, captured = graphs[0]
    graph.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(captured, want))
    del graph, captured
    graphs.clear()
    gc.collect()
    torch.cuda.synchronize()
    ops.score_attention(q, k, v, [0, 10, 500])
    assert not mine()


def test_capture_entry_points():
    import ctypes as C
    L = _lib.lib()
    n = C.c_ulonglong(77)
    assert L.lv_capture_id(None, C.byref(n)) == 0 and L.lv_capture_id(None, None) == -1
    assert L.lv_capture_watch(None) == -1 and b"not being captured" in L.lvattn_last_error()
    assert L.lv_capture_ended(None, 1) == -1
